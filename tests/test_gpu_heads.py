"""Norms of queries and keys for each head, their rotation by position, and the gradients, against the formulas in
64 bits."""
import pytest
import torch

from tdgs_amd import decoder

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# Angles are rounded to 2^-26 turns (2^-23 radians) and their sines to 2^-23, the norm's sum and root to a few 2^-24.
EXTRA = 8 * 2.0 ** -23


def half_step(t):
    return torch.finfo(t).eps / 2


def rotate(y, rotary, positions, sign=1):
    n = rotary.pairs
    axis = [a for a, s in enumerate(rotary.sections) for _ in range(s)]
    at = positions.double()
    at = at[None] if at.dim() == 2 else at
    angle = sign * (at[..., axis] * rotary.turns * 2 * torch.pi)[:, :, None]
    if rotary.layout == "halves":
        a, b = y[..., :n], y[..., n:2 * n]
    else:
        a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
    c, s = angle.cos(), angle.sin()
    a, b = a * c - b * s, a * s + b * c
    turned = torch.cat([a, b], -1) if rotary.layout == "halves" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, y[..., 2 * n:]], -1)


def exact(x, w, eps, rotary, positions, dout, norm=True):
    leaves = [x.double().requires_grad_(True)] + ([w.double().requires_grad_(True)] if w is not None else [])
    y = leaves[0]
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        y = y * leaves[1] if w is not None else y
    if rotary is not None:
        y = rotate(y, rotary, positions)
    return (y.detach(), *torch.autograd.grad(y, leaves, dout.double()))


def close(got, want, t, steps=1, extra=EXTRA):
    assert got.dtype is t and torch.isfinite(got).all()
    error = (got.double() - want).norm()
    assert error <= (steps * half_step(t) + extra) * want.norm() + 1e-30, (error / want.norm()).item()


def tensors(t, b, l, h, hk, d, layout, gen):
    if layout == "fused":
        both = torch.randn((b, l, h + 2 * hk, d), generator=gen).to(t).cuda()
        return both[:, :, :h], both[:, :, h:h + hk]
    shape = (lambda n: (b, n, l, d)) if layout == "bhld" else (lambda n: (b, l, n, d + (3 if layout == "odd" else 0)))
    q, k = (torch.randn(shape(n), generator=gen).to(t).cuda() for n in (h, hk))
    return (q.transpose(1, 2), k.transpose(1, 2)) if layout == "bhld" else (q[..., :d], k[..., :d])


def check(t, b, l, h, hk, d, sections, pairs, layout="blhd", kind="int", batched=False, param=torch.float32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q, k = tensors(t, b, l, h, hk, d, layout, gen)
    dq_out, dk_out = tensors(t, b, l, h, hk, d, layout, gen)
    wq, wk = (1 + 0.3 * torch.randn(d, generator=gen).to(param).cuda() for _ in range(2))
    rotary = positions = None
    if sections:
        rotary = decoder.Rotary(sections, pairs=pairs)
        shape = (b, l, len(sections)) if batched else (l, len(sections))
        positions = torch.randint(0, 100000, shape, generator=gen).cuda()
        positions = positions.float() / 16 if kind == "float" else positions.to(torch.int32 if kind == "int" else torch.int64)
    q_out, k_out, dq, dk = (torch.full(x.shape, float("nan"), dtype=t, device="cuda") for x in (q, k, q, k))
    dwq, dwk = torch.full_like(wq, float("nan")), torch.full_like(wk, float("nan"))
    decoder.head_norm_(q_out, k_out, q, k, wq, wk, eps=1e-5, rotary=rotary, positions=positions)
    temp = decoder.head_norm_temp(q, k).fill_(255)
    decoder.head_norm_grad_(dq, dk, dwq, dwk, dq_out, dk_out, q, k, wq, wk, eps=1e-5, rotary=rotary, positions=positions,
                            temp=temp)
    for x, w, dout, out, dx, dw in ((q, wq, dq_out, q_out, dq, dwq), (k, wk, dk_out, k_out, dk, dwk)):
        want = exact(x, w, 1e-5, rotary, positions, dout)
        close(out, want[0], t)
        # a gradient across xhat may cancel: for heads of two it is what is left of the difference, so its error is
        # taken relative to what it is the difference of
        r = 1 / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-5)
        size = (dout.double() * w.double().abs().max() * r).norm()
        assert (dx.double() - want[1]).norm() <= half_step(t) * want[1].norm() + EXTRA * size
        rows = b * l * x.shape[2]
        terms = ((dout.double() * x.double() * r) ** 2).sum().sqrt()
        assert (dw.double() - want[2]).norm() <= half_step(param) * want[2].norm() + (EXTRA + rows ** 0.5 * 2.0 ** -24) * terms
    if rotary is not None:
        close(decoder.rotate(q, None, rotary, positions), rotate(q.double(), rotary, positions), t)
        a, c = decoder.rotate(q, k, rotary, positions, inverse=True)
        close(a, rotate(q.double(), rotary, positions, -1), t)
        close(c, rotate(k.double(), rotary, positions, -1), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("pairs", ["halves", "interleaved"])
@pytest.mark.parametrize("d,sections", [(2, (1,)), (16, (8,)), (40, (10, 10)), (64, (16, 16)), (64, (8, 10, 10)), (80, (8, 8, 8)),
                                        (96, (48,)), (127, (20, 30)), (128, (64,)), (250, (41, 42, 42)), (256, (32, 32, 32, 32)),
                                        (33, ()), (48, ()), (1, ())], ids=str)
def test_head_sizes(gpu, t, pairs, d, sections):
    check(TYPES[t], 2, 9, 3, 2, d, sections, pairs)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", ["blhd", "bhld", "fused", "odd"])
@pytest.mark.parametrize("kind", ["int", "long", "float"])
def test_layouts_and_positions(gpu, t, layout, kind):
    check(TYPES[t], 3, 50, 8, 2, 64, (12, 20), "halves", layout, kind, batched=kind != "float")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 16, 4), (8, 1, 1, 1), (1, 4000, 1, 1), (2, 5003, 4, 4), (1, 3, 70, 5)], ids=str)
def test_lengths(gpu, t, shape):
    check(TYPES[t], *shape, 32, (8, 8), "interleaved", param=TYPES[t])


@pytest.mark.parametrize("t", TYPES)
def test_far_positions(gpu, t):
    """A billion steps out, angles are as exact as at the start."""
    t = TYPES[t]
    q = torch.randn((1, 64, 2, 64), generator=torch.Generator().manual_seed(1)).to(t).cuda()
    positions = (2 ** 30 + 12345677 * torch.arange(64, device="cuda"))[:, None]
    rotary = decoder.Rotary((32,))
    close(decoder.rotate(q, None, rotary, positions), rotate(q.double(), rotary, positions), t)


def test_in_place_and_one_tensor(gpu):
    gen = torch.Generator().manual_seed(3)
    q = torch.randn((2, 30, 4, 64), generator=gen).bfloat16().cuda()
    rotary, positions = decoder.Rotary((16, 16)), torch.randint(0, 500, (30, 2), generator=gen).cuda()
    want = decoder.head_norm(q, rotary=rotary, positions=positions)
    dout = torch.randn(q.shape, generator=gen).bfloat16().cuda()
    dq = torch.empty_like(q)
    decoder.head_norm_grad_(dq, None, None, None, dout, None, q, rotary=rotary, positions=positions)
    decoder.head_norm_grad_(dout, None, None, None, dout, None, q, rotary=rotary, positions=positions)
    assert torch.equal(dq, dout)
    decoder.head_norm_(q, None, q, rotary=rotary, positions=positions)
    assert torch.equal(q, want)
