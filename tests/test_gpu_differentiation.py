"""The differentiable decoder operators on the GPU: what torch's differentiation may ask of them."""
import pytest
import torch

from tdgs_amd import appearance, decoder

pytestmark = pytest.mark.gpu


def test_gradient_penalty_raises(gpu):
    """The image reaches the corrected one by the operators and past them: a penalty on its gradient would lack the operators'
    part. The first derivative is the same with and without a graph."""
    dec = appearance.AppearanceDecoder(2, channels=32, groups=4)
    rgb = torch.rand((17, 9, 3), generator=torch.Generator().manual_seed(0)).cuda().requires_grad_(True)
    want, = torch.autograd.grad((dec(rgb, 1) ** 2).sum(), rgb)
    got, = torch.autograd.grad((dec(rgb, 1) ** 2).sum(), rgb, create_graph=True)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="differentiated again"):
        got.pow(2).sum().backward()


def test_empty_gradients(gpu):
    """The gradient of a sum over no elements comes with strides of zero."""
    q, k = torch.randn((2, 0, 4, 8), device="cuda"), torch.randn((2, 5, 2, 8), device="cuda")
    x, w, table = torch.randn((2, 0, 8), device="cuda"), torch.ones(8, device="cuda"), torch.randn((6, 8), device="cuda")
    for t in (q, k, x, w, table):
        t.requires_grad_(True)
    tokens = torch.empty((3, 0), dtype=torch.int64, device="cuda")
    for f in (lambda: decoder.cross_attention(q, k, k), lambda: decoder.group_norm(x, 2, w, w),
              lambda: decoder.embedding(table, tokens)):
        f().sum().backward()
    for t in (q, k, x, w, table):
        assert t.grad.shape == t.shape and not t.grad.any()
