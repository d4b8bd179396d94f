"""Linear layers with bias, activation and residual, and their gradients, against the formulas in 64 bits."""
import pytest
import torch

from tdgs_amd import decoder

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = {"identity": lambda z: z, "silu": lambda z: z * torch.sigmoid(z),
        "gelu": lambda z: 0.5 * z * torch.erfc(-z * 0.5 ** 0.5), "relu": lambda z: z.clamp(min=0)}


def half_step(t):
    return torch.finfo(t).eps / 2


def inputs(rows, k, n, t, layout="in_out", bias=True, residual=True, pad=0, scale=1.0, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def matrix(r, c):
        return torch.randn((r, c + pad), generator=gen).to(t).cuda()[:, :c]

    x = matrix(rows, k)
    w = (k ** -0.5 * torch.randn((k, n) if layout == "in_out" else (n, k), generator=gen)).to(t).cuda()
    w = w if layout == "in_out" else w.T
    return (x, w, torch.randn(n, generator=gen).to(t).cuda() if bias else None, matrix(rows, n) if residual else None,
            (scale * matrix(rows, n).float()).to(t))


def exact(x, w, b, r, dout, act):
    leaves = [x.double().requires_grad_(True), w.double().requires_grad_(True)]
    if b is not None:
        leaves.append(b.double().requires_grad_(True))
    z = leaves[0] @ leaves[1] + (leaves[2] if b is not None else 0.0)
    y = ACTS[act](z)
    grads = torch.autograd.grad(y, leaves, dout.double())
    return (y.detach() + r.double() if r is not None else y.detach(), *grads, *([None] if b is None else []))


def close(got, want, t, steps, extra=0.0):
    """Relative error over the tensor: `steps` roundings to the type, each half a step at most, and `extra`."""
    assert got.dtype is t
    norm = want.norm()
    error = (got.double() - want).norm()
    assert torch.isfinite(got).all()
    assert error <= (steps * half_step(t) + extra) * norm + 1e-30, (error / norm).item()


def run(x, w, b, r, dout, act):
    n = w.shape[1]
    out = torch.full((x.shape[0], n), float("nan"), dtype=x.dtype, device="cuda")
    pre = None if act == "identity" else torch.full_like(out, float("nan"))
    temp = decoder.linear_temp(x, w, grad=True)
    decoder.linear_(out, x, w, b, residual=r, activation=act, pre=pre, temp=temp)
    temp.fill_(255)
    dx = torch.full(x.shape, float("nan"), dtype=x.dtype, device="cuda")
    dw = torch.full_like(w, float("nan"))
    db = None if b is None else torch.full_like(b, float("nan"))
    decoder.linear_grad_(dx, dw, db, dout, x, w, activation=act, pre=pre, temp=temp)
    return out, dx, dw, db


def check(case, act, t):
    got, want = run(*case, act), exact(*case, act)
    rows, k, n = *case[0].shape, case[1].shape[1]
    # out: rounded once; sums of `depth` products of 32 bits, of which up to sqrt(depth) half steps of 2^-24 remain on
    # average, taken four times over. Gradients: pre rounded (act'' is below 1, z on average below 2), dz
    # rounded, the result rounded.
    def sums(depth):
        return 4 * max(depth, 16) ** 0.5 * 2.0 ** -24
    close(got[0], want[0], t, 1, sums(k))
    close(got[1], want[1], t, 1 if act == "identity" else 4, sums(n) + sums(k))
    close(got[2], want[2], t, 1 if act == "identity" else 4, sums(rows) + sums(k))
    if case[2] is not None:
        close(got[3], want[3], t, 1 if act == "identity" else 4, 4 * sums(rows) + sums(k))


SIZES = [(1, 1, 1), (1, 512, 64), (3, 7, 5), (2, 16, 2048), (31, 8, 6), (33, 48, 64), (64, 65, 127), (65, 129, 33), (130, 32, 128),
         (200, 3, 300), (257, 515, 130), (513, 100, 1), (700, 1, 40), (16, 4096, 24), (2049, 6, 9), (4099, 72, 80)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", ["in_out", "out_in"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(gpu, t, layout, size):
    check(inputs(*size, TYPES[t], layout), "identity", TYPES[t])
    check(inputs(*size, TYPES[t], layout, bias=False, residual=False, pad=3, seed=1), "silu", TYPES[t])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activations(gpu, t, act):
    check(inputs(1000, 96, 264, TYPES[t], seed=2), act, TYPES[t])


@pytest.mark.parametrize("t", TYPES)
def test_large_tiles(gpu, t):
    """More than 256 tiles of the forward product, and a long depth of the weight's gradient that is split."""
    check(inputs(16400, 136, 392, TYPES[t], pad=8, seed=3), "gelu", TYPES[t])
    check(inputs(16385, 131, 257, TYPES[t], "out_in", seed=4), "silu", TYPES[t])


@pytest.mark.parametrize("t", TYPES)
def test_relu_slope_follows_pre(gpu, t):
    """ReLU's gradient is cut where the kept z is not positive, whatever sum made it."""
    t = TYPES[t]
    x, w, b, r, dout = inputs(300, 40, 72, t, seed=5)
    pre, out = torch.empty_like(dout), torch.empty_like(dout)
    decoder.linear_(out, x, w, b, activation="relu", pre=pre)
    assert torch.equal(out, pre.clamp(min=0))
    dx, dw, db = (torch.empty_like(v) for v in (x.contiguous(), w, b))
    decoder.linear_grad_(dx, dw, db, dout, x, w, activation="relu", pre=pre)
    dz = torch.where(pre > 0, dout, 0).double()
    close(dx, dz @ w.double().T, t, 1, 1e-5)
    close(dw, x.double().T @ dz, t, 1, 1e-5)
    close(db, dz.sum(0), t, 1, 1e-5)
