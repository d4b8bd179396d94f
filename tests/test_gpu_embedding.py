"""Embedding lookup with scaling, bit for bit, and its gradient by sorted tokens against the sums in 64
bits within their rounding errors, at the sizes, tokens and strides where it can go wrong."""
import pytest
import torch

from tdgs_amd import core, decoder

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _tokens(kind, n, vocab, gen, dtype):
    if kind == "one":
        t = torch.full((n,), vocab // 2)
    elif kind == "skewed":
        t = torch.clamp((torch.rand((n,), generator=gen).double().pow(6) * vocab).long(), max=vocab - 1)
    elif kind == "ends":
        t = torch.where(torch.rand((n,), generator=gen) < 0.5, 0, vocab - 1)
    else:
        t = torch.randint(0, vocab, (n,), generator=gen)
    return t.to(dtype).cuda()


SIZES = [
    # n, vocab, dim, tokens
    (1, 1, 1, "any"),
    (1, 5, 64, "any"),
    (77, 1000, 64, "any"),
    (31, 2, 48, "any"),
    (32, 3, 48, "one"),
    (33, 3, 48, "one"),
    (64, 256, 3, "ends"),
    (1000, 10, 27, "skewed"),
    (5000, 300, 16, "skewed"),
    (20000, 7, 8, "one"),
    (300, 65536, 40, "any"),
    (4097, 255, 512, "skewed"),
    (700, 50, 1000, "skewed"),
    (9000, 5000, 130, "any"),
    (4096, 9, 4, "skewed"),        # the most that one launch takes, of one token nearly
    (4096, 100000, 16, "any"),
    (3000, 5000000, 1, "any"),     # more rows than 2^12 for each of 1024 workgroups
    (100000, 3, 5, "skewed"),
    (2688, 20000, 48, "skewed"),   # the most that one launch takes of rows of 12 vectors, and one more
    (2689, 20000, 48, "skewed"),
    (4096, 300000, 8, "one"),      # one workgroup has all tokens, and rows of two sorting steps
    (4095, 300000, 8, "ends"),
    (513, 700000, 24, "any"),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("size", SIZES, ids=["-".join(map(str, s)) for s in SIZES])
def test_against_sums(gpu, dtype, index, size):
    """A token's sum over its n rows is off by (n + 2) roundings of the sum of their sizes at most."""
    n, vocab, dim, kind = size
    gen = torch.Generator().manual_seed(n + vocab)
    tokens = _tokens(kind, n, vocab, gen, index)
    table = torch.randn((vocab, dim), generator=gen).to(dtype).cuda()
    scale = dim ** 0.5
    out = torch.empty((n, dim), dtype=dtype, device="cuda")
    decoder.embedding_lookup_(out, table, tokens, scale=scale)
    assert torch.equal(out, (table[tokens.long()].float() * scale).to(dtype))
    dout = torch.randn((n, dim), generator=gen).to(dtype).cuda()
    padding = int(tokens[0]) if n > 1 and kind != "one" else None
    dtable = torch.full((vocab, dim), 7.0, dtype=dtype, device="cuda")
    decoder.embedding_grad_(dtable, dout, tokens, scale=scale, padding=padding)
    t, d = tokens.long().cpu(), dout.double().cpu()
    if padding is not None:
        d = d * (t != padding)[:, None]
    want = torch.zeros((vocab, dim), dtype=torch.float64).index_add_(0, t, d) * scale
    size_ = torch.zeros((vocab, dim), dtype=torch.float64).index_add_(0, t, d.abs()) * scale
    count = torch.bincount(t, minlength=vocab)[:, None]
    err = (count + 2) * U32 * size_ + 1.01 * torch.finfo(dtype).eps / 2 * want.abs() + TINY[dtype]
    got = dtable.double().cpu()
    assert ((got - want).abs() <= err).all()
    assert not got[count[:, 0] == 0].any()
    core.ctx_check(0)


def test_gradient_against_differences(gpu):
    """The lookup is linear: differences of sum(dout * out) give the gradient up to rounding."""
    gen = torch.Generator().manual_seed(3)
    tokens = _tokens("skewed", 500, 40, gen, torch.int32)
    table, dout = torch.randn((40, 12), generator=gen).cuda(), torch.randn((500, 12), generator=gen).cuda()
    out, dtable = torch.empty((500, 12), device="cuda"), torch.empty((40, 12), device="cuda")
    decoder.embedding_grad_(dtable, dout, tokens, scale=2.0)
    for _ in range(3):
        d = torch.randn((40, 12), generator=gen).cuda()
        f = []
        for sign in (1, -1):
            decoder.embedding_lookup_(out, table + sign * d, tokens, scale=2.0)
            f.append((out.double() * dout.double()).sum())
        # 500 * 12 products of values up to ~30, each rounded once or twice
        assert abs((f[0] - f[1]) / 2 - (dtable.double() * d.double()).sum()) <= 6000 * 30 * 4 * U32


def test_strided_rows_and_shapes(gpu):
    gen = torch.Generator().manual_seed(5)
    wide = torch.randn((50, 3, 32), generator=gen).cuda()
    tokens = torch.randint(0, 50, (4, 9), generator=gen).cuda()
    out = torch.empty((4, 9, 32), device="cuda")
    decoder.embedding_lookup_(out, wide[:, 1], tokens)
    assert torch.equal(out, wide[:, 1][tokens])
    dwide = torch.zeros((50, 3, 32), device="cuda")
    decoder.embedding_grad_(dwide[:, 1], out, tokens)
    want = torch.zeros((50, 32), dtype=torch.float64, device="cuda").index_add_(0, tokens.flatten(), out.reshape(36, 32).double())
    assert (dwide[:, 1].double() - want).abs().max() <= 40 * U32 * want.abs().max()
    assert not dwide[:, 0].any() and not dwide[:, 2].any()


def test_no_tokens(gpu):
    table = torch.randn((20, 8), device="cuda")
    tokens = torch.empty((0,), dtype=torch.int64, device="cuda")
    decoder.embedding_lookup_(torch.empty((0, 8), device="cuda"), table, tokens)
    dtable = torch.full((20, 8), 3.0, device="cuda")
    decoder.embedding_grad_(dtable, torch.empty((0, 8), device="cuda"), tokens)
    assert not dtable.any()


@pytest.mark.parametrize("bad", [-1, 20, 1 << 31, -(1 << 40)])
def test_token_outside_the_table(gpu, bad):
    """A row of zeros, no gradient, and an error on the context given; the next calls are clean again."""
    ctx = core.Context(0)
    table = torch.randn((20, 8), device="cuda")
    tokens = torch.tensor([3, bad, 19], device="cuda")
    out, dtable = torch.empty((3, 8), device="cuda"), torch.empty((20, 8), device="cuda")
    decoder.embedding_lookup_(out, table, tokens, ctx=ctx)
    assert not out[1].any() and torch.equal(out[0], table[3]) and torch.equal(out[2], table[19])
    with pytest.raises(core.TdgsError, match="outside its table"):
        core.ctx_check(0, ctx)
    core.ctx_check(0, ctx)
    decoder.embedding_grad_(dtable, torch.ones((3, 8), device="cuda"), tokens, ctx=ctx)
    assert dtable.sum() == 16 and (dtable[3] == 1).all() and (dtable[19] == 1).all()
    with pytest.raises(core.TdgsError, match="outside its table"):
        core.ctx_check(0, ctx)
    core.ctx_check(0)


def test_offsets_past_32_bits(gpu):
    """Rows more than 2^32 bytes into a table, and of a gradient."""
    vocab, dim = (1 << 20) + 8, 2112
    table = torch.empty((vocab, dim), dtype=torch.bfloat16, device="cuda")
    table[-8:] = torch.randn((8, dim), device="cuda").bfloat16()
    tokens = vocab - 1 - torch.arange(8, dtype=torch.int32, device="cuda")
    out = torch.empty((8, dim), dtype=torch.bfloat16, device="cuda")
    decoder.embedding_lookup_(out, table, tokens)
    assert torch.equal(out, table[-8:].flip(0))
    want = table[-8:].clone()
    table.fill_(3.0)
    decoder.embedding_grad_(table, out, tokens)
    assert torch.equal(table[-8:], want) and not table[:-8].any()


def test_repeatable_and_on_another_stream(gpu):
    gen = torch.Generator().manual_seed(6)
    tokens = _tokens("skewed", 50000, 400, gen, torch.int32)
    dout = torch.randn((50000, 48), generator=gen).cuda()
    first, second = (torch.empty((400, 48), device="cuda") for _ in range(2))
    decoder.embedding_grad_(first, dout, tokens)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        temp = decoder.embedding_temp(first, tokens)
        temp.fill_(0xff)
        decoder.embedding_grad_(second, dout, tokens, temp=temp)
    side.synchronize()
    assert torch.equal(first, second)


def test_graph_replays(gpu):
    gen = torch.Generator().manual_seed(7)
    tokens = _tokens("skewed", 3000, 100, gen, torch.int64)
    dout = torch.randn((3000, 20), generator=gen).cuda()
    want, got = (torch.empty((100, 20), device="cuda") for _ in range(2))
    decoder.embedding_grad_(want, dout, tokens)
    temp = decoder.embedding_temp(got, tokens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decoder.embedding_grad_(got, dout, tokens, temp=temp)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_refusals(gpu):
    table = torch.zeros((20, 8), device="cuda")
    tokens = torch.zeros((5,), dtype=torch.int64, device="cuda")
    out = torch.empty((5, 8), device="cuda")
    many = torch.zeros((5000,), dtype=torch.int64, device="cuda")
    decoder.embedding_lookup_(out, table, tokens)
    for bad in (
        lambda: decoder.embedding_lookup_(out[:4], table, tokens),
        lambda: decoder.embedding_lookup_(out.half(), table, tokens),
        lambda: decoder.embedding_lookup_(out, table, tokens.float()),
        lambda: decoder.embedding_lookup_(out, table, tokens.cpu()),
        lambda: decoder.embedding_lookup_(out, table.t(), tokens),
        lambda: decoder.embedding_lookup_(out, table, torch.zeros((10,), dtype=torch.int64, device="cuda")[::2]),
        lambda: decoder.embedding_lookup_(out.double(), table.double(), tokens),
        lambda: decoder.embedding_grad_(table, out[:, :4], tokens),
        lambda: decoder.embedding_grad_(table, out, tokens, temp=torch.empty(5, device="cuda")),
    ):
        with pytest.raises(ValueError):
            bad()
    for bad in (
        lambda: decoder.embedding_lookup_(out[:1].expand(5, 8), table, tokens),
        lambda: decoder.embedding_grad_(table[:1].expand(20, 8), out, tokens),
        lambda: decoder.embedding_grad_(table, torch.zeros((5000, 8), device="cuda"), many,
                                        temp=torch.empty(5, dtype=torch.uint8, device="cuda")),
    ):
        with pytest.raises(core.TdgsError):
            bad()
