"""Attention: forms of a call that the formulas' tests leave out."""
import pytest
import torch

from tdgs_amd import decoder
from test_gpu_attention import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mask", ["none", "lengths", "keys"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
def test_no_queries_of_shared_states(gpu, dtype, mask):
    """Sums over no batches: the states' gradients are zeros."""
    c = Case(dtype, 0, 1, 7, 600, 4, 2, 40, mask=mask)
    c.run()
    assert not c.dk.any() and not c.dv.any()
    k = torch.randn((1, 600, 2, 40), device="cuda", requires_grad=True)
    out = decoder.cross_attention(torch.randn((0, 7, 4, 40), device="cuda", requires_grad=True), k, k)
    assert out.shape == (0, 7, 4, 40)
    torch.full((4096, 600), 7.0, device="cuda")   # (left where new tensors are taken from)
    out.sum().backward()
    assert not k.grad.any()


@pytest.mark.parametrize("mask", ["none", "both"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_queries_gradient_alone(gpu, dtype, mask):
    """Without dk and dv the call writes the same dq, and no other."""
    c = Case(dtype, 2, 1, 70, 600, 4, 2, 40, mask=mask)
    c.run()
    want = c.dq.clone()
    c.dq.zero_()
    decoder.cross_attention_grad_(c.dq, None, None, c.dout, c.out, c.lse, c.q, c.k, c.v, **c.args)
    assert torch.equal(c.dq, want)
    for dk, dv in ((c.dk, None), (None, c.dv)):
        with pytest.raises(ValueError):
            decoder.cross_attention_grad_(c.dq, dk, dv, c.dout, c.out, c.lse, c.q, c.k, c.v, **c.args)


@pytest.mark.parametrize("size", [
    # b, lq, lk, h, hk, d: rows go on by whole batches, by queries and heads with and without carries
    (150, 1, 40, 2, 2, 16), (150, 1, 600, 3, 1, 40), (67, 3, 520, 6, 2, 16), (40, 7, 90, 5, 1, 33), (9, 32, 70, 2, 2, 64),
    (9, 33, 530, 4, 2, 64), (3, 40, 70, 40, 1, 8), (5, 64, 20, 1, 1, 32), (2, 100, 33, 70, 1, 8),
], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_shared_states_of_batches_of_few_queries(gpu, dtype, size):
    b, lq, lk, h, hk, d = size
    c = Case(dtype, b, 1, lq, lk, h, hk, d, "bhld", seed=b)
    c.run()
    c.check()


def test_no_batches_of_many_queries(gpu):
    """Queries times shared heads do not fit 32 bits, but there are no batches of them."""
    q = torch.empty((0, 1 << 30, 4, 8), device="cuda")
    k = torch.randn((1, 5, 1, 8), device="cuda")
    dk, dv = torch.full_like(k, 7.0), torch.full_like(k, 7.0)
    decoder.cross_attention_(q, q, k, k)
    decoder.cross_attention_grad_(q, dk, dv, q, q, torch.empty((0, 4, 1 << 30), device="cuda"), q, k, k)
    assert not dk.any() and not dv.any()
