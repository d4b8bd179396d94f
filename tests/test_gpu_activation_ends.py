"""Gradients of linear layers where z has left the type's range on its way to pre: infinities have the slopes of an
activation's ends, and nothing of their rows and columns is lost."""
import pytest
import torch

from tdgs_amd import decoder

pytestmark = pytest.mark.gpu

SLOPES = {"identity": (1.0, 1.0), "silu": (0.0, 1.0), "gelu": (0.0, 1.0), "relu": (0.0, 1.0)}


def rand(*shape, seed=0, t=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(t).cuda()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", SLOPES)
@pytest.mark.parametrize("rows", [40, 3000])
def test_infinite_pre(gpu, t, act, rows):
    """pre of +-infinity and at the ends of the range, next to zeros (slopes of a half, but relu's)."""
    n = 48
    pre = torch.zeros((rows, n), dtype=t, device="cuda")
    ends = [float("-inf"), float("inf"), torch.finfo(t).min, torch.finfo(t).max]
    for i, end in enumerate(ends):
        pre[3 + i::9, i::4] = end
    low, high = SLOPES[act]
    middle = {"identity": 1.0, "relu": 0.0}.get(act, 0.5)
    slope = torch.where(pre < 0, low, torch.where(pre > 0, high, middle)).double()
    x, w, dout = rand(rows, 32, t=t), rand(32, n, seed=1, t=t) / 8, rand(rows, n, seed=2, t=t)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(n, dtype=t, device="cuda")
    decoder.linear_grad_(dx, dw, db, dout, x, w, activation=act, pre=pre)
    dz = dout.double() * slope
    # dz rounded for its products, results rounded: two half steps, and sums in 32 bits of up to 3000 terms
    for got, want in ((dx, dz @ w.double().T), (dw, x.double().T @ dz), (db, dz.sum(0))):
        assert torch.isfinite(got).all()
        assert (got.double() - want).norm() <= (torch.finfo(t).eps + 4 * rows ** 0.5 * 2.0 ** -24 + 2.0 ** -20) * want.norm()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_half_past_its_range_forward_and_backward(gpu, act):
    """A column of features whose z is below -65504 in some rows: out is zero there, pre minus infinity, and the gradients are
    those of the rows that are left."""
    t = torch.float16
    x, w, dout = rand(200, 16, t=t), rand(16, 24, seed=1, t=t) / 4, rand(200, 24, seed=2, t=t)
    x[::5, 0], w[0, 5] = -300.0, 300.0
    leaves = [v.clone().requires_grad_(True) for v in (x, w)]
    out = decoder.linear(*leaves, activation=act)
    assert (out[::5, 5] == 0).all() and torch.isfinite(out).all()
    out.backward(dout)
    z = (x.double() @ w.double()).requires_grad_(True)
    y = z * torch.sigmoid(z) if act == "silu" else 0.5 * z * torch.erfc(-z * 0.5 ** 0.5)
    dz, = torch.autograd.grad(y, z, dout.double())
    for got, want in ((leaves[0].grad, dz @ w.double().T), (leaves[1].grad, x.double().T @ dz)):
        assert torch.isfinite(got).all()
        # pre rounded (act'' below 1, z of about 1 where the slope is not an end's), dz and the result rounded
        assert (got.double() - want).norm() <= 4 * torch.finfo(t).eps / 2 * want.norm()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_nan_pre_stays_nan(gpu, act):
    pre, dout, w = rand(30, 16), rand(30, 16, seed=1), rand(8, 16, seed=2)
    pre[7, 3] = float("nan")
    dx = torch.empty((30, 8), device="cuda")
    decoder.linear_grad_(dx, None, None, dout, rand(30, 8, seed=3), w, activation=act, pre=pre)
    rows = torch.arange(30, device="cuda") != 7
    assert torch.isnan(dx[7]).all() and torch.isfinite(dx[rows]).all()
