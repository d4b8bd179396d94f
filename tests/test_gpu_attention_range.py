"""The gradients of float16 attention over the range of its type: dP and dS are no results, and what they are must not
depend on what half holds. Small upstream gradients (a mean over many pixels), large ones (a scaled loss), and keys
that every query gives little weight."""
import pytest
import torch

from test_gpu_attention import U32, Case

pytestmark = pytest.mark.gpu

U = 2.0 ** -11          # half's unit roundoff
LEAST = 2.0 ** -25      # and what rounding a subnormal half loses


def _check(c):
    """dq, dk and dv of every element. p is off by ep of itself, dP by edp, as for normal values (rounding of out, which
    delta comes from, included); dS for its products by one rounding of half of itself, and by 2^-31 of the largest
    of its row (dq) or key (dk), far below which nothing of it is kept; the results by their own rounding."""
    d, group = c.q.shape[3], c.q.shape[2] // c.k.shape[2]
    scale = d ** -0.5
    for h in range(c.k.shape[2]):
        k, v = c.k[0, :, h].double().cpu(), c.v[0, :, h].double().cpu()
        want = {"k": torch.zeros_like(k), "v": torch.zeros_like(k)}
        err = {"k": torch.zeros_like(k), "v": torch.zeros_like(k)}
        top, rows = 0, []
        for g in range(h * group, (h + 1) * group):
            q, do = c.q[0, :, g].double().cpu(), c.dout[0, :, g].double().cpu()
            s = q @ k.T * scale
            lse = torch.logsumexp(s, dim=1, keepdim=True)
            p = torch.exp(s - lse)
            o = p @ v
            e = U32 * ((d + 8) * scale * (q.abs() @ k.abs().T) + 4 * s.abs()).amax(dim=1, keepdim=True)
            n = k.shape[0]
            ep = 2 * e + (n + 16) * U32 + 4 * U32 * lse.abs()
            eo = (ep + U) * (p @ v.abs()) + 1.01 * U * o.abs() + LEAST
            dp, delta = do @ v.T, (do * o).sum(dim=1, keepdim=True)
            ds = p * (dp - delta)
            edp = U32 * (d + 2) * (do.abs() @ v.abs().T + (do.abs() * o.abs()).sum(dim=1, keepdim=True)) \
                + (do.abs() * eo).sum(dim=1, keepdim=True)
            eds = p * edp * (1 + ep) + ds.abs() * (ep + 4 * U32 + U)
            dq = scale * ds @ k
            edq = scale * ((eds + 2.0 ** -31 * ds.abs().amax(dim=1, keepdim=True) + U32 * (n + 4) * ds.abs()) @ k.abs()) \
                + 1.01 * U * dq.abs() + LEAST
            got = c.dq[0, :, g].double().cpu()
            held = dq.abs() < 65000
            assert torch.isfinite(got[held]).all() and held.any()
            assert ((got - dq).abs() <= edq)[held].all(), ((got - dq).abs() / edq)[held].max()
            want["k"] += scale * ds.T @ q
            want["v"] += p.T @ do
            m = q.shape[0] * group
            err["k"] += scale * ((eds + U32 * (m + 4) * ds.abs()).T @ q.abs())
            err["v"] += ((ep + U + U32 * (m + 4)) * p).T @ do.abs() + 2.0 ** -38 * do.abs().sum(dim=0)
            rows.append(q)
            top = torch.maximum(torch.as_tensor(top), ds.abs().amax(dim=0)[:, None])
        for q in rows:
            err["k"] += scale * 2.0 ** -31 * top * q.abs().sum(dim=0)
        for name, t in (("k", c.dk), ("v", c.dv)):
            got = t[0, :, h].double().cpu()
            bound = err[name] + 1.01 * U * want[name].abs() + LEAST
            held = want[name].abs() < 65000
            assert torch.isfinite(got[held]).all() and held.any()
            assert ((got - want[name]).abs() <= bound)[held].all(), (name, ((got - want[name]).abs() / bound)[held].max())


@pytest.mark.parametrize("size", [
    # lq, lk, h, hk, d, layout
    (40, 4, 2, 2, 64, "blhd"), (700, 300, 4, 2, 64, "blhd"), (130, 1500, 2, 2, 24, "odd"), (300, 520, 2, 1, 128, "bhld"),
    (1500, 1100, 2, 2, 64, "blhd"),   # dK, dV by one operand, wide workgroups
    (900, 4, 4, 1, 128, "blhd"), (2000, 4096, 1, 1, 64, "blhd"),
], ids=str)
@pytest.mark.parametrize("power", [-13, -10, 0, 10, 13])
def test_upstream_gradients_of_any_size(gpu, size, power):
    lq, lk, h, hk, d, layout = size
    c = Case(torch.float16, 1, 1, lq, lk, h, hk, d, layout, seed=lq)
    c.dout.copy_(c.dout.clamp(-3, 3) * 2.0 ** power)
    c.run()
    _check(c)


def test_rows_of_very_different_size(gpu):
    """Rows, and values of keys, from 2^-12 to 2^12 of each other, in an order that rises and one that falls."""
    for flip in (False, True):
        c = Case(torch.float16, 1, 1, 320, 400, 2, 2, 64, seed=5)
        rise = 2.0 ** torch.linspace(-12, 12, 320, device="cuda")
        c.dout.mul_((rise.flip(0) if flip else rise)[None, :, None, None])
        rise = 2.0 ** torch.linspace(-8, 2, 400, device="cuda")
        c.v.mul_((rise.flip(0) if flip else rise)[None, :, None, None])
        c.run()
        _check(c)


def test_keys_of_little_weight(gpu):
    """Every query gives half of the keys a weight of 2^-16 to 2^-24, and all of them together move dv."""
    c = Case(torch.float16, 1, 1, 1000, 3000, 2, 2, 32, seed=7)
    c.q.copy_(0.2 * c.q + 1)
    c.k.copy_(0.2 * c.k - 1.0 * (torch.arange(3000, device="cuda") % 2)[None, :, None, None])
    c.dout.copy_(0.1 * c.dout + 1)
    c.run()
    _check(c)


def test_zero_and_infinite_rows(gpu):
    """A gradient of zeros is zero; an infinite row spoils its own dq only."""
    c = Case(torch.float16, 1, 1, 100, 200, 2, 2, 64, seed=8)
    c.dout.zero_()
    c.run()
    assert not c.dq.any() and not c.dk.any() and not c.dv.any()
    c.dout.normal_()
    c.run()
    want = c.dq.clone()
    c.dout[0, 17] = float("inf")
    c.run()
    assert not torch.isfinite(c.dq[0, 17]).any()
    c.dq[0, 17] = want[0, 17]
    assert torch.equal(c.dq, want)


@pytest.mark.parametrize("lq,h", [(20, 2), (16384, 8)])   # P by two operands; by one, every workgroup taking all keys
def test_one_key_far_above_the_others(gpu, lq, h):
    """A key that takes nearly all of every query's weight and has no value: the output is the others' small weights, which
    are alike, so that what half loses of one it loses of all."""
    c = Case(torch.float16, 1, 1, lq, 128, h, h, 32, seed=9)
    c.q.copy_(0.1 * c.q + 1)
    c.k.zero_()
    c.k[:, 0] = 2.0
    c.v.copy_(0.1 * c.v + 1)
    c.v[:, 0] = 0
    c.run(grad=False)
    c.check(grad=False)
