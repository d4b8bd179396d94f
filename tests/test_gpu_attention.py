"""Cross attention and its gradients against the formulas in 64 bits, element by element within the
rounding errors that the computation may make, at the sizes, strides and masks where it can go wrong;
against differences of the forward pass; and what the calls refuse."""
import math

import pytest
import torch

from tdgs_amd import core, decoder

pytestmark = pytest.mark.gpu

U = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}   # the unit roundoffs
U32 = 2.0 ** -24


def _view(shape, dtype, layout, gen):
    """A (batch, length, heads, d) tensor of normal values: contiguous, heads before length, every
    other row of a longer one, or rows of an odd pitch."""
    b, n, h, d = shape
    if layout == "bhld":
        x = torch.randn((b, h, n, d), generator=gen).to(dtype).cuda().transpose(1, 2)
    elif layout == "sliced":
        x = torch.randn((b, 2 * n + 1, h + 1, d), generator=gen).to(dtype).cuda()[:, 1::2, 1:]
    elif layout == "odd":
        x = torch.randn((b, n, h, d + 3), generator=gen).to(dtype).cuda()[..., 1:d + 1]
    else:
        x = torch.randn(shape, generator=gen).to(dtype).cuda()
    assert tuple(x.shape) == tuple(shape)
    return x


class Case:
    def __init__(self, dtype, b, kvb, lq, lk, h, hk, d, layout="blhd", mask="none", seed=0, spread=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.q = _view((b, lq, h, d), dtype, layout, gen)
        self.q.mul_(spread)
        self.k, self.v = (_view((kvb, lk, hk, d), dtype, layout, gen) for _ in range(2))
        self.dout = _view((b, lq, h, d), dtype, layout, gen)
        self.out, self.dq = (_view((b, lq, h, d), dtype, layout, gen) for _ in range(2))
        self.dk, self.dv = (_view((kvb, lk, hk, d), dtype, layout, gen) for _ in range(2))
        self.lse = torch.full((b, h, lq), 7.0, device="cuda")
        self.lengths = self.mask = None
        self.keep = torch.ones((kvb, lk), dtype=torch.bool)
        if mask in ("lengths", "both"):
            lengths = torch.randint(0, lk + 1, (kvb,), generator=gen)
            lengths[0] = 0 if kvb > 1 else max(lk - 1, 0)
            self.keep &= torch.arange(lk)[None] < lengths[:, None]
            self.lengths = lengths.to(torch.int32).cuda()
        if mask in ("keys", "both", "blocks"):
            m = torch.rand((kvb, lk), generator=gen) < 0.6
            if mask == "blocks":   # whole tiles without an allowed key, between others
                m = (torch.arange(lk)[None] // 70 % 2 == 1) & m
            if kvb > 1:
                m[-1] = False
            self.keep &= m
            self.mask = m.cuda()
        if mask == "nothing":
            self.keep[:] = False
            self.mask = self.keep.cuda()
        hidden = ~self.keep[:, :, None, None].cuda()
        self.k.masked_fill_(hidden, float("nan"))
        self.v.masked_fill_(hidden, float("inf"))
        self.args = dict(kv_lengths=self.lengths, kv_mask=self.mask)

    def run(self, grad=True):
        decoder.cross_attention_(self.out, self.q, self.k, self.v, lse=self.lse, **self.args)
        if grad:
            decoder.cross_attention_grad_(self.dq, self.dk, self.dv, self.dout, self.out, self.lse, self.q, self.k,
                                          self.v, **self.args)
        torch.cuda.synchronize()

    def check(self, grad=True):
        """Every output within its error bound. Per row, with u the rounding of the type and w that
        of 32 bits: a score is off by e = w ((d + 8) scale sum |q||k| + 4 |s|) at most, p by 2 e + (keys + 16) w
        + u of itself, out by that times sum p |v| and its own rounding; and so on by the chain of
        the formulas (delta = dout . out of the rounded out)."""
        dtype = self.q.dtype
        u, d = U[dtype], self.q.shape[3]
        scale, group = d ** -0.5, self.q.shape[2] // self.k.shape[2]
        q, do, out = (x.double().cpu().permute(0, 2, 1, 3) for x in (self.q, self.dout, self.out))
        # the rounding of subnormal results
        tiny = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24}[dtype]
        b_all = q.shape[0]
        acc = {n: torch.zeros(self.k.shape, dtype=torch.float64) for n in ("dk", "dv", "ek", "ev")}
        for b in range(b_all):
            kb = b if self.k.shape[0] > 1 else 0
            at = torch.nonzero(self.keep[kb]).flatten()
            for h in range(q.shape[1]):
                hk = h // group
                k, v = (x[kb].double().cpu()[at, hk] for x in (self.k, self.v))
                qq, dd = q[b, h], do[b, h]
                if at.numel() == 0:
                    assert not out[b, h].any()
                    assert torch.isneginf(self.lse[b, h]).all()
                    if grad:
                        assert not self.dq[b, :, h].any()
                    continue
                s = qq @ k.T * scale
                lse = torch.logsumexp(s, dim=1)
                p = torch.exp(s - lse[:, None])
                o = p @ v
                e = U32 * ((d + 8) * scale * (qq.abs() @ k.abs().T) + 4 * s.abs()).amax(dim=1, keepdim=True)
                ep = 2 * e + (at.numel() + 16) * U32 + u
                eo = ep * (p @ v.abs()) + 1.01 * u * o.abs() + tiny
                assert ((out[b, h] - o).abs() <= eo).all(), (b, h, ((out[b, h] - o).abs() / eo).max())
                el = (e + U32 * (at.numel() + 8 + 4 * lse.abs()[:, None]))[:, 0]
                assert ((self.lse[b, h].double().cpu() - lse).abs() <= el).all()
                if not grad:
                    continue
                ep = ep + 4 * U32 * lse.abs()[:, None] + tiny * at.numel()
                dp = dd @ v.T
                delta = (dd * o).sum(dim=1, keepdim=True)
                ds = p * (dp - delta)
                edp = U32 * (d + 2) * (dd.abs() @ v.abs().T) + (dd.abs() * eo).sum(dim=1, keepdim=True) \
                    + U32 * (d + 2) * (dd.abs() * o.abs()).sum(dim=1, keepdim=True)
                eds = p * edp * (1 + ep) + ds.abs() * (ep + 4 * U32) + tiny
                n = qq.shape[0]
                dq = scale * ds @ k
                edq = scale * (eds @ k.abs() + U32 * (at.numel() + 4) * (ds.abs() @ k.abs())) + 1.01 * u * dq.abs() + tiny
                got = self.dq[b, :, h].double().cpu()
                assert ((got - dq).abs() <= edq).all(), (b, h, ((got - dq).abs() / edq).max())
                acc["dk"][kb, at, hk] += scale * ds.T @ qq
                acc["dv"][kb, at, hk] += p.T @ dd
                acc["ek"][kb, at, hk] += scale * (eds.T @ qq.abs() + U32 * (n * b_all * group + 4) * (ds.abs().T @ qq.abs()))
                acc["ev"][kb, at, hk] += ((ep + U32 * (n * b_all * group + 4)) * p + tiny).T @ dd.abs()
        if grad:
            for name, got in (("k", self.dk), ("v", self.dv)):
                want, err = acc["d" + name], acc["e" + name]
                got = got.double().cpu()
                err = err + 1.01 * u * want.abs() + tiny
                assert ((got - want).abs() <= err).all(), (name, ((got - want).abs() / err).max())
                assert not got[~self.keep].any()


DTYPES = [torch.float32, torch.bfloat16, torch.float16]

SIZES = [
    # b, kvb, lq, lk, h, hk, d, layout, mask
    (1, 1, 1, 1, 1, 1, 1, "blhd", "none"),
    (1, 1, 1, 64, 4, 4, 64, "blhd", "none"),
    (2, 2, 31, 33, 2, 1, 7, "odd", "none"),
    (2, 2, 33, 65, 2, 2, 16, "bhld", "lengths"),
    (1, 1, 130, 63, 4, 2, 40, "sliced", "keys"),
    (3, 3, 65, 130, 3, 1, 64, "blhd", "both"),
    (3, 1, 70, 129, 4, 2, 65, "blhd", "both"),
    (2, 1, 257, 200, 2, 2, 32, "bhld", "none"),
    (2, 2, 40, 300, 2, 1, 80, "bhld", "blocks"),
    (1, 1, 129, 257, 2, 2, 96, "sliced", "none"),
    (2, 2, 33, 97, 4, 1, 128, "blhd", "keys"),
    (1, 1, 5, 31, 1, 1, 127, "odd", "lengths"),
    (2, 2, 9, 40, 2, 2, 64, "blhd", "nothing"),
    (1, 1, 2, 5000, 4, 1, 64, "bhld", "keys"),
    (2, 2, 1, 3001, 8, 2, 128, "blhd", "lengths"),
    (1, 1, 1500, 3, 1, 1, 24, "blhd", "none"),
    (2, 1, 150, 700, 4, 2, 64, "blhd", "both"),
    (1, 1, 200, 600, 3, 3, 40, "sliced", "none"),
    (2, 2, 90, 515, 2, 1, 33, "odd", "lengths"),
    (3, 1, 7, 520, 6, 1, 16, "bhld", "keys"),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=["-".join(map(str, s)) for s in SIZES])
def test_against_formulas(gpu, dtype, size):
    c = Case(dtype, *size)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_peaked_rows(gpu, dtype):
    """Scores of hundreds: one key takes all of a row, the others' weights underflow."""
    c = Case(dtype, 1, 1, 100, 200, 2, 2, 64, spread=30.0, seed=3)
    c.run(grad=False)
    c.check(grad=False)


@pytest.mark.parametrize("rise", [1.0, -1.0], ids=["rising", "falling"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_scores_that_rise_along_the_keys(gpu, dtype, rise):
    """The largest score of a row comes late, and every tile's is far above (or below) the one before."""
    c = Case(dtype, 1, 1, 70, 700, 2, 1, 64, seed=8)
    along = torch.linspace(0, 1, 700, device="cuda")[None, :, None, None]
    c.q.copy_(c.q.abs() + 0.5)
    c.k.copy_(0.05 * c.k + rise * 8 * along)
    c.run()
    c.check()


@pytest.mark.parametrize("lq,lk", [(0, 5), (5, 0), (0, 0)])
def test_empty_lengths(gpu, lq, lk):
    c = Case(torch.bfloat16, 2, 2, lq, lk, 2, 1, 32)
    c.run()
    assert not c.out.any() and not c.dq.any() and not c.dk.any() and not c.dv.any()
    assert torch.isneginf(c.lse).all()


@pytest.mark.parametrize("lq", [5, 3000])
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_single_key(gpu, dtype, lq):
    """The softmax of one key is constant: the output is its value, and no gradient reaches q or k."""
    for kw in (dict(lk=1), dict(lk=700, mask="single")):
        c = Case(dtype, 1, 1, lq, kw["lk"], 4, 2, 40, mask="none", seed=6)
        if "mask" in kw:
            c.keep[:] = False
            c.keep[0, 77] = True
            c.args = dict(kv_lengths=None, kv_mask=c.keep.cuda())
        c.run()
        c.check()
        assert not c.dq.any() and not c.dk.any()


def test_gradient_against_differences(gpu):
    """d/dt of sum(dout * out) along random directions, from central differences of the forward pass
    with step 2^-5 along unit directions: their error is the third derivative's, below 1e-3 of the
    gradient's norm here, and the forward pass's noise of a few 1e-6 over the step."""
    c = Case(torch.float32, 2, 1, 37, 45, 4, 2, 24, mask="keys", seed=5)
    c.run()
    gen = torch.Generator().manual_seed(11)
    step = 2.0 ** -5
    for name, g in (("q", c.dq), ("k", c.dk), ("v", c.dv)):
        x = getattr(c, name)
        x0 = x.clone()
        for _ in range(3):
            t = torch.randn(x.shape, generator=gen).cuda()
            t /= t.norm()
            f = []
            for sign in (1, -1):
                x.copy_(x0 + sign * step * t)
                decoder.cross_attention_(c.out, c.q, c.k, c.v, **c.args)
                f.append((c.out.double() * c.dout.double()).sum())
            want = (f[0] - f[1]) / (2 * step)
            got = (g.double() * t.double()).sum()
            assert abs(got - want) <= 2e-3 * g.double().norm(), (name, got, want)
        x.copy_(x0)


def test_repeatable_and_on_another_stream(gpu):
    """The same bits every time, on another stream too, with scratch of the caller's that held something else."""
    c = Case(torch.bfloat16, 2, 1, 300, 500, 4, 2, 64, mask="keys", seed=9)
    c.run()
    first = [x.clone() for x in (c.out, c.lse, c.dq, c.dk, c.dv)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        temp = decoder.cross_attention_temp(c.q, c.k, grad=True)
        temp.fill_(0xff)
        decoder.cross_attention_(c.out, c.q, c.k, c.v, lse=c.lse, temp=temp, **c.args)
        decoder.cross_attention_grad_(c.dq, c.dk, c.dv, c.dout, c.out, c.lse, c.q, c.k, c.v, temp=temp, **c.args)
    side.synchronize()
    for a, b in zip(first, (c.out, c.lse, c.dq, c.dk, c.dv)):
        assert torch.equal(a, b)


def test_offsets_past_32_bits(gpu):
    """Batches of keys more than 2^32 bytes and 2^31 elements apart."""
    far = (1 << 31) + 64
    flat = torch.zeros(far + 64 * 2 * 32, dtype=torch.bfloat16, device="cuda")
    c = Case(torch.bfloat16, 2, 2, 20, 64, 2, 2, 32, seed=4)
    k = torch.as_strided(flat, (2, 64, 2, 32), (far, 64, 32, 1))
    k.copy_(c.k)
    c.k = k
    c.run()
    c.check()


def test_graph_replays(gpu):
    """A captured pass gives the eager result on every replay."""
    c = Case(torch.float16, 1, 1, 40, 900, 4, 4, 64, seed=6)
    c.run()
    first = [x.clone() for x in (c.out, c.dq, c.dk, c.dv)]
    temp = decoder.cross_attention_temp(c.q, c.k, grad=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decoder.cross_attention_(c.out, c.q, c.k, c.v, lse=c.lse, temp=temp)
        decoder.cross_attention_grad_(c.dq, c.dk, c.dv, c.dout, c.out, c.lse, c.q, c.k, c.v, temp=temp)
    for _ in range(3):
        for x in (c.out, c.dq, c.dk, c.dv):
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(first, (c.out, c.dq, c.dk, c.dv)):
            assert torch.equal(a, b)


def test_refusals(gpu):
    c = Case(torch.bfloat16, 2, 2, 8, 9, 4, 2, 32)

    def call(q=c.q, k=c.k, v=c.v, out=c.out, **kw):
        decoder.cross_attention_(out, q, k, v, **kw)

    def grad(**kw):
        args = dict(dq=c.dq, dk=c.dk, dv=c.dv, dout=c.dout, out=c.out, lse=c.lse, q=c.q, k=c.k, v=c.v)
        args.update(kw)
        decoder.cross_attention_grad_(**args)

    call(lse=c.lse)
    grad()
    wide = torch.zeros((2, 8, 4, 136), dtype=torch.bfloat16, device="cuda")
    keys = torch.zeros((2, 9, 2, 136), dtype=torch.bfloat16, device="cuda")
    for bad in (
        lambda: call(q=c.q.float()),
        lambda: call(k=c.k[:, :, :, :16]),
        lambda: call(v=c.v[:, :5]),
        lambda: call(out=c.out.cpu()),
        lambda: call(q=c.q.transpose(2, 3), out=c.out.transpose(2, 3)),
        lambda: call(kv_lengths=torch.zeros(3, dtype=torch.int32, device="cuda")),
        lambda: call(kv_lengths=torch.zeros(2, dtype=torch.int64, device="cuda")),
        lambda: call(kv_mask=torch.zeros((2, 9), device="cuda")),
        lambda: call(kv_mask=torch.zeros((2, 8), dtype=torch.bool, device="cuda")),
        lambda: call(lse=torch.zeros((2, 4, 8), dtype=torch.float64, device="cuda")),
        lambda: call(q=c.q.to(torch.int32)),
        lambda: grad(lse=None),
        lambda: grad(dk=c.dk[:1]),
    ):
        with pytest.raises(ValueError):
            bad()
    for bad in (
        lambda: call(scale=0.0),
        lambda: call(scale=-1.0),
        lambda: call(scale=math.inf),
        lambda: call(scale=math.nan),
        lambda: call(q=wide, out=torch.empty_like(wide), k=keys, v=keys),
        lambda: call(q=c.q[:, :, :3], out=c.out[:, :, :3]),
        lambda: call(k=torch.cat([c.k, c.k[:1]]), v=torch.cat([c.v, c.v[:1]])),
        lambda: call(out=c.out[:, :1].expand(2, 8, 4, 32)),
        lambda: grad(dk=c.dk[:1].expand(2, 9, 2, 32)),
        lambda: grad(temp=torch.empty(16, dtype=torch.uint8, device="cuda")),
    ):
        with pytest.raises(core.TdgsError):
            bad()
