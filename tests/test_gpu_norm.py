"""Group norm with an activation and its gradients against the formulas in 64 bits, element by element
within the rounding errors that the computation may make, at the sizes, strides and values where it can
go wrong; against differences of the forward pass; and what the calls refuse."""
import math

import pytest
import torch

from tdgs_amd import core, decoder

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24}


def _act(z, act):
    """act(z) and its derivative in 64 bits."""
    if act == "identity":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    cdf = 0.5 * torch.erfc(-z * math.sqrt(0.5))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _image(shape, dtype, layout, gen):
    n, p, c = shape
    if layout == "sliced":   # some channels of a wider image, every other pixel
        return torch.randn((n, 2 * p, c + 16), generator=gen).to(dtype).cuda()[:, ::2, 8:c + 8]
    if layout == "odd":      # rows that start off 16 bytes
        return torch.randn((n, p, c + 3), generator=gen).to(dtype).cuda()[..., 1:c + 1]
    return torch.randn(shape, generator=gen).to(dtype).cuda()


class Case:
    def __init__(self, dtype, n, p, c, groups, act, layout="plain", params="f32", mean=0.0, spread=1.0, seed=0, eps=1e-5):
        gen = torch.Generator().manual_seed(seed)
        self.groups, self.act, self.eps = groups, act, eps
        self.x, self.dout, self.out, self.dx = (_image((n, p, c), dtype, layout, gen) for _ in range(4))
        self.x.mul_(spread).add_(mean)
        self.x.mul_(torch.exp(0.5 * torch.randn((c,), generator=gen)).to(dtype).cuda())
        ptype = torch.float32 if params != "same" else dtype
        self.w = (1 + 0.3 * torch.randn((c,), generator=gen)).to(ptype).cuda() if params != "none" else None
        self.b = (0.3 * torch.randn((c,), generator=gen)).to(ptype).cuda() if params != "none" else None
        self.dw, self.db = (torch.full((c,), 7.0, dtype=ptype, device="cuda") for _ in range(2))
        self.stats = torch.zeros((n, groups, 2), device="cuda")

    def run(self):
        decoder.group_norm_(self.out, self.x, self.groups, self.w, self.b, eps=self.eps, activation=self.act,
                            stats=self.stats)
        decoder.group_norm_grad_(self.dx, self.dw, self.db, self.dout, self.x, self.stats, self.groups, self.w, self.b,
                                 activation=self.act)
        torch.cuda.synchronize()

    def check(self):
        """k: the additions that one sum goes through one after another, at most as many as a group's
        pixels and a few joins. The mean is off by em = k w max |x| (w: a rounding in 32 bits), the variance by
        2 k w and (em / deviation)^2 of itself, 1 / deviation by half that; z, act (whose derivative stays below
        1.13 in size and changes by at most 0.8 per unit) and the sums of the backward pass follow from the
        formulas."""
        x, do = self.x.double().cpu(), self.dout.double().cpu()
        n, p, c = x.shape
        gs = c // self.groups
        u, tiny = torch.finfo(self.x.dtype).eps / 2, TINY[self.x.dtype]
        k = p + 64 + gs
        w = (self.w.double().cpu() if self.w is not None else torch.ones(c, dtype=torch.float64))
        b = (self.b.double().cpu() if self.b is not None else torch.zeros(c, dtype=torch.float64))

        def group(f, y):   # over pixels and the group's channels, at full shape
            return f(y.reshape(n, p, self.groups, gs).permute(0, 2, 1, 3).reshape(n, self.groups, -1)) \
                .repeat_interleave(gs, dim=1)[:, None, :]
        avg = lambda y: group(lambda t: t.mean(dim=2), y)
        mean, top = avg(x), group(lambda t: t.abs().amax(dim=2), x)
        var = avg((x - mean) ** 2)
        r = 1 / torch.sqrt(var + self.eps)
        em = k * U32 * top
        er = k * U32 + 0.5 * (em * r) ** 2 + 8 * U32
        xhat = (x - mean) * r
        exhat = em * r + xhat.abs() * (er + 3 * U32)
        z = xhat * w + b
        ez = exhat * w.abs() + 3 * U32 * (xhat * w).abs() + U32 * z.abs()
        y, slope = _act(z, self.act)
        flip = (z.abs() <= ez).double() if self.act == "relu" else torch.zeros_like(z)
        eact = 3e-7 * (1 + z.abs())
        ey = 1.13 * ez + eact + 1.01 * u * y.abs() + tiny
        out = self.out.double().cpu()
        assert ((out - y).abs() <= ey).all(), ((out - y).abs() / ey).max()
        stats = self.stats.double().cpu()
        assert ((stats[..., 0] - mean[:, 0, ::gs]).abs() <= em[:, 0, ::gs] + U32 * mean[:, 0, ::gs].abs()).all()
        assert ((stats[..., 1] - r[:, 0, ::gs]).abs() <= (er * r)[:, 0, ::gs]).all()
        e = do * slope
        ee = do.abs() * (0.8 * ez + eact * 2 + flip) + 2 * U32 * e.abs()
        kk = n * p + 64
        db, dw = e.sum(dim=(0, 1)), (e * xhat).sum(dim=(0, 1))
        up = torch.finfo(self.dw.dtype).eps / 2
        edb = ee.sum(dim=(0, 1)) + kk * U32 * e.abs().sum(dim=(0, 1)) + 1.01 * up * db.abs() + TINY[self.dw.dtype]
        edw = (ee * xhat.abs() + e.abs() * exhat).sum(dim=(0, 1)) + kk * U32 * (e * xhat).abs().sum(dim=(0, 1)) \
            + 1.01 * up * dw.abs() + TINY[self.dw.dtype]
        assert ((self.db.double().cpu() - db).abs() <= edb).all()
        assert ((self.dw.double().cpu() - dw).abs() <= edw).all()
        we = w * e
        m1, m2 = avg(we), avg(we * xhat)
        em1 = avg(w.abs() * ee) + k * U32 * avg(we.abs())
        em2 = avg(w.abs() * ee * xhat.abs() + we.abs() * exhat) + k * U32 * avg((we * xhat).abs())
        inner = we - m1 - xhat * m2
        edx = r * (w.abs() * ee + em1 + xhat.abs() * em2 + exhat * m2.abs()
                   + 4 * U32 * (we.abs() + m1.abs() + (xhat * m2).abs())) + (er + 4 * U32) * r * inner.abs()
        dx = r * inner
        edx = edx + 1.01 * u * dx.abs() + tiny
        got = self.dx.double().cpu()
        assert ((got - dx).abs() <= edx).all(), ((got - dx).abs() / edx).max()


DTYPES = [torch.float32, torch.bfloat16, torch.float16]

SIZES = [
    # n, pixels, channels, groups, act, layout, params
    (1, 1, 8, 1, "silu", "plain", "f32"),
    (1, 64, 128, 32, "silu", "plain", "f32"),
    (2, 1, 32, 32, "identity", "plain", "same"),      # one value per group: variance 0
    (3, 77, 24, 3, "gelu", "plain", "same"),
    (2, 1000, 30, 5, "relu", "plain", "none"),
    (1, 513, 27, 9, "silu", "odd", "f32"),
    (2, 300, 64, 8, "gelu", "sliced", "f32"),
    (1, 40, 2064, 16, "silu", "plain", "f32"),        # more channels than one workgroup holds
    (1, 33, 517, 11, "identity", "plain", "f32"),
    (5, 2, 3, 1, "relu", "plain", "f32"),
    (1, 20000, 8, 4, "silu", "plain", "f32"),
    (9, 129, 96, 8, "gelu", "plain", "f32"),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=["-".join(map(str, s)) for s in SIZES])
def test_against_formulas(gpu, dtype, size):
    c = Case(dtype, *size)
    c.run()
    c.check()


@pytest.mark.parametrize("n,p", [(1, 60), (2, 3000)])
def test_large_mean(gpu, n, p):
    """A mean of thousands of deviations, which a sum of squares less the squared mean would lose."""
    c = Case(torch.float32, n, p, 32, 4, "identity", mean=3000.0, spread=0.5)
    c.x.copy_(c.x / c.x.mean(dim=(0, 1)) * 3000.0)
    c.run()
    c.check()


def test_constant_image(gpu):
    """Variance zero: 1 / sqrt(eps) and outputs of the bias alone."""
    c = Case(torch.float32, 1, 100, 16, 4, "identity", params="f32")
    c.x.fill_(5.0)
    c.run()
    c.check()


def test_whole_images(gpu):
    """(n, width, height, channels) images, in place."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((2, 9, 7, 16), generator=gen).cuda()
    out = torch.empty_like(x)
    decoder.group_norm_(out, x, 4)
    flat = torch.empty((2, 63, 16), device="cuda")
    decoder.group_norm_(flat, x.reshape(2, 63, 16), 4)
    assert torch.equal(out.reshape(2, 63, 16), flat)
    decoder.group_norm_(x, x, 4)
    assert torch.equal(x, out)


def test_empty(gpu):
    x = torch.empty((2, 0, 16), device="cuda")
    stats = torch.zeros((2, 4, 2), device="cuda")
    dw, db = torch.full((16,), 3.0, device="cuda"), torch.full((16,), 3.0, device="cuda")
    decoder.group_norm_(torch.empty_like(x), x, 4, stats=stats)
    decoder.group_norm_grad_(torch.empty_like(x), dw, db, torch.empty_like(x), x, stats, 4)
    assert not dw.any() and not db.any()


def test_gradient_against_differences(gpu):
    """d/dt of sum(dout * out) along random directions, from central differences of the forward pass with
    step 2^-6 along unit directions: the third derivative's share stays below 1e-3 of the gradient's norm."""
    for act in ("silu", "gelu", "identity"):
        c = Case(torch.float32, 2, 50, 24, 3, act, seed=8)
        c.run()
        gen = torch.Generator().manual_seed(2)
        step = 2.0 ** -6
        for t, g in ((c.x, c.dx), (c.w, c.dw), (c.b, c.db)):
            t0 = t.clone()
            for _ in range(3):
                d = torch.randn(t.shape, generator=gen).cuda()
                d /= d.norm()
                f = []
                for sign in (1, -1):
                    t.copy_(t0 + sign * step * d)
                    decoder.group_norm_(c.out, c.x, c.groups, c.w, c.b, activation=act)
                    f.append((c.out.double() * c.dout.double()).sum())
                want = (f[0] - f[1]) / (2 * step)
                assert abs((g.double() * d.double()).sum() - want) <= 2e-3 * g.double().norm()
            t.copy_(t0)


def test_repeatable_and_on_another_stream(gpu):
    c = Case(torch.bfloat16, 2, 5000, 64, 8, "silu")
    c.run()
    first = [t.clone() for t in (c.out, c.stats, c.dx, c.dw, c.db)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        temp = decoder.group_norm_temp(c.x, c.groups, grad=True)
        temp.fill_(0xff)
        decoder.group_norm_(c.out, c.x, c.groups, c.w, c.b, stats=c.stats, temp=temp)
        decoder.group_norm_grad_(c.dx, c.dw, c.db, c.dout, c.x, c.stats, c.groups, c.w, c.b, temp=temp)
        # dx in dout's place
        decoder.group_norm_grad_(c.dout, None, None, c.dout, c.x, c.stats, c.groups, c.w, c.b, temp=temp)
    side.synchronize()
    for a, b in zip(first, (c.out, c.stats, c.dx, c.dw, c.db)):
        assert torch.equal(a, b)
    assert torch.equal(c.dout, c.dx)


def test_offsets_past_32_bits(gpu):
    """Images more than 2^32 bytes and 2^31 elements apart."""
    far = (1 << 31) + 64
    flat = torch.zeros(far + 100 * 16, dtype=torch.bfloat16, device="cuda")
    c = Case(torch.bfloat16, 2, 100, 16, 4, "silu")
    x = torch.as_strided(flat, (2, 100, 16), (far, 16, 1))
    x.copy_(c.x)
    c.x = x
    c.run()
    c.check()


def test_graph_replays(gpu):
    c = Case(torch.float16, 1, 700, 32, 4, "gelu")
    c.run()
    first = [t.clone() for t in (c.out, c.dx, c.dw, c.db)]
    temp = decoder.group_norm_temp(c.x, c.groups, grad=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decoder.group_norm_(c.out, c.x, c.groups, c.w, c.b, activation="gelu", stats=c.stats, temp=temp)
        decoder.group_norm_grad_(c.dx, c.dw, c.db, c.dout, c.x, c.stats, c.groups, c.w, c.b, activation="gelu", temp=temp)
    for _ in range(3):
        for t in (c.out, c.dx, c.dw, c.db):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(first, (c.out, c.dx, c.dw, c.db)):
            assert torch.equal(a, b)


def test_refusals(gpu):
    x = torch.zeros((2, 10, 16), device="cuda")
    out, stats, w = torch.empty_like(x), torch.zeros((2, 4, 2), device="cuda"), torch.zeros(16, device="cuda")
    large = torch.zeros((2, 100000, 16), device="cuda")
    decoder.group_norm_(out, x, 4, w, w, stats=stats)
    for bad in (
        lambda: decoder.group_norm_(out[:, :5], x, 4),
        lambda: decoder.group_norm_(out.half(), x, 4),
        lambda: decoder.group_norm_(out, x.transpose(1, 2), 4),
        lambda: decoder.group_norm_(out.cpu(), x, 4),
        lambda: decoder.group_norm_(out, x, 4, w[:8], w),
        lambda: decoder.group_norm_(out, x, 4, w.half(), w.half()),
        lambda: decoder.group_norm_(out, x, 4, w, w.double()),
        lambda: decoder.group_norm_(out, x, 4, activation="tanh"),
        lambda: decoder.group_norm_(out, x, 4, stats=stats[:1]),
        lambda: decoder.group_norm_(out.double(), x.double(), 4),
        lambda: decoder.group_norm_grad_(out, None, None, x, x, None, 4),
        lambda: decoder.group_norm_grad_(out, w.half(), None, x, x, stats, 4, w, w),
    ):
        with pytest.raises(ValueError):
            bad()
    for bad in (
        lambda: decoder.group_norm_(out, x, 5),
        lambda: decoder.group_norm_(out, x, 0),
        lambda: decoder.group_norm_(out, x, 4, eps=-1.0),
        lambda: decoder.group_norm_(out, x, 4, eps=math.nan),
        lambda: decoder.group_norm_(out[:1].expand(2, 10, 16), x, 4),
        lambda: decoder.group_norm_(torch.empty_like(large), large, 4, temp=torch.empty(8, dtype=torch.uint8, device="cuda")),
    ):
        with pytest.raises(core.TdgsError):
            bad()
