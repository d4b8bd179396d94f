"""Results that share memory with what a call of a linear layer, head norm or dropout reads or writes besides: refused before
anything is launched. Columns of one buffer that lie between each other share none, and in place means the same tensor."""
import ctypes as C
import os

import pytest
import torch

from tdgs_amd import abi, core, decoder

KB = 1 << 10


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(core.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return core.lib()


def fill(s, **kw):
    for k, v in kw.items():
        if isinstance(v, tuple) and isinstance(getattr(s, k), C.Structure):
            for (f, _), x in zip(getattr(s, k)._fields_, v):
                setattr(getattr(s, k), f, x)
        elif isinstance(v, tuple):
            for i, x in enumerate(v):
                getattr(s, k)[i] = x
        else:
            setattr(s, k, v)
    return s


def linear(**kw):
    """8 x 16 -> 24 of 16 bits, every tensor in a kilobyte or two of its own (none of these addresses is ever used)."""
    given = dict(dtype=abi.TDGS_BF16, activation=abi.TDGS_ACT_SILU, rows=8, in_features=16, out_features=24, x=(64 * KB, 16),
                 weight=(66 * KB, 24), out=(68 * KB, 24), pre=(70 * KB, 24), residual=(72 * KB, 24), bias=74 * KB, temp=1 << 30,
                 temp_bytes=1 << 30)
    return fill(abi.LinearC(), **{**given, **kw})


@pytest.mark.parametrize("kw,text", [
    ({"out": (64 * KB + 16, 24)}, b"out overlaps x"), ({"out": (66 * KB - 2, 24)}, b"out overlaps the weight"),
    ({"out": (66 * KB + 766, 24)}, b"out overlaps the weight"), ({"out": (74 * KB + 46, 24)}, b"out overlaps the bias"),
    ({"out": (72 * KB + 2, 24)}, b"out overlaps the residual"), ({"out": (72 * KB, 48)}, b"out overlaps the residual"),
    ({"out": (72 * KB, 24), "residual": (72 * KB, 0)}, b"out overlaps the residual"),   # its first row for all of them
    ({"out": (72 * KB + 48, 24), "residual": (72 * KB, 48)}, b"out overlaps the residual"),
    ({"pre": (68 * KB + 32, 24)}, b"pre overlaps out"), ({"pre": (72 * KB - 32, 24)}, b"pre overlaps the residual"),
    ({"pre": (64 * KB + 16, 40), "x": (64 * KB, 40)}, b"pre overlaps x"),               # rows of 24 behind 16, eight too early
    ({"x": (64 * KB, 64), "out": (64 * KB + 30, 64)}, b"out overlaps x"),
    ({"x": (64 * KB, 64), "out": (64 * KB + 90, 64)}, b"out overlaps x"),               # its rows end behind x's next
])
def test_linear(lib, kw, text):
    assert lib.tdgs_linear_forward(None, C.byref(linear(**kw))) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error(), lib.tdgs_last_error()


@pytest.mark.parametrize("kw,grads,text", [
    ({}, {"dx": (80 * KB + 2, 16)}, b"dx overlaps dout"), ({}, {"dx": (70 * KB + 2, 16)}, b"dx overlaps pre"),
    ({}, {"dx": (64 * KB + 2, 16)}, b"dx overlaps x"), ({}, {"dx": (66 * KB + 2, 16)}, b"dx overlaps the weight"),
    ({}, {"dx": (84 * KB + 2, 16)}, b"dx overlaps dweight"), ({}, {"dweight": (80 * KB - 2, 24)}, b"dweight overlaps dout"),
    ({}, {"dweight": (64 * KB + 2, 24)}, b"dweight overlaps x"), ({}, {"dweight": (66 * KB + 2, 16), "dweight_layout": 1},
                                                                  b"dweight overlaps the weight"),
    ({}, {"dbias": 80 * KB + 4}, b"dbias overlaps dout"), ({}, {"dbias": 84 * KB + 4}, b"dbias overlaps dweight"),
    ({}, {"dbias": 82 * KB + 4}, b"dbias overlaps dx"), ({}, {"dbias": 64 * KB + 4}, b"dbias overlaps x"),
])
def test_linear_gradient(lib, kw, grads, text):
    given = dict(dout=(80 * KB, 24), dx=(82 * KB, 16), dweight=(84 * KB, 24), dbias=86 * KB)
    g = fill(abi.LinearGradsC(), **{**given, **grads})
    assert lib.tdgs_linear_grad(None, C.byref(linear(**kw)), C.byref(g)) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error(), lib.tdgs_last_error()


@pytest.mark.parametrize("kw,text", [
    ({"out": (64 * KB + 4, 5)}, b"out overlaps x"), ({"out": (64 * KB, 6)}, b"out overlaps x"), ({"x": (64 * KB, 0), "out": (64 * KB, 5)},
                                                                                                b"out overlaps x"),
    ({"residual": (66 * KB, 5), "out": (66 * KB - 4, 5)}, b"out overlaps the residual"),
    ({"residual": (66 * KB, 8), "out": (66 * KB + 16, 8)}, b"out overlaps the residual"),
])
def test_dropout(lib, kw, text):
    a = fill(abi.DropoutC(), **{**dict(dtype=0, rows=3, cols=5, p=0.5, x=(64 * KB, 5), out=(68 * KB, 5)), **kw})
    assert lib.tdgs_dropout_apply(None, C.byref(a)) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error(), lib.tdgs_last_error()


def head_norm(**kw):
    """Two batches of three tokens, four heads and two of 32 elements of 16 bits."""
    given = dict(dtype=abi.TDGS_BF16, param_dtype=abi.TDGS_F32, batch=2, length=3, heads=4, kv_heads=2, head_dim=32, norm=1, eps=1e-6,
                 q=(64 * KB, 384, 128, 32), q_out=(68 * KB, 384, 128, 32), k=(72 * KB, 192, 64, 32), k_out=(76 * KB, 192, 64, 32))
    return fill(abi.HeadNormC(), **{**given, **kw})


@pytest.mark.parametrize("kw,text", [
    ({"q_out": (64 * KB + 64, 384, 128, 32)}, b"q_out overlaps q"), ({"q_out": (64 * KB, 384, 32, 96)}, b"q_out overlaps q"),
    ({"q_out": (64 * KB, 768, 256, 32)}, b"q_out overlaps q"), ({"k_out": (64 * KB, 192, 64, 32)}, b"k_out overlaps q"),
    ({"q_out": (72 * KB, 384, 128, 32)}, b"q_out overlaps k"), ({"k_out": (68 * KB + 1024, 192, 64, 32)}, b"q_out overlaps k_out"),
    # two results in one buffer whose columns reach into each other
    ({"q_out": (68 * KB, 576, 192, 32), "k_out": (68 * KB + 192, 576, 192, 32)}, b"q_out overlaps k_out"),
    # one place for several rows of a result
    ({"q_out": (68 * KB, 384, 32, 32)}, b"rows of q_out overlap"), ({"q_out": (68 * KB, 128, 128, 32)}, b"rows of q_out overlap"),
    ({"k_out": (76 * KB, 96, 64, 32)}, b"rows of k_out overlap"), ({"k_out": (76 * KB, 32, 64, 64)}, b"rows of k_out overlap"),
])
def test_head_norm(lib, kw, text):
    assert lib.tdgs_head_norm_forward(None, C.byref(head_norm(**kw))) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error(), lib.tdgs_last_error()


def test_head_norm_transposed_in_place(lib):
    """Heads and tokens of equal number: q_out starts where q does, but is its transpose."""
    a = head_norm(length=4, q=(64 * KB, 512, 128, 32), q_out=(64 * KB, 512, 32, 128), k=(80 * KB, 256, 64, 32), k_out=(90 * KB, 256, 64, 32))
    assert lib.tdgs_head_norm_forward(None, C.byref(a)) == abi.TDGS_ERR_INVALID and b"q_out overlaps q" in lib.tdgs_last_error()


@pytest.mark.parametrize("grads,text", [
    ({"dq": (80 * KB + 64, 384, 128, 32)}, b"dq overlaps dq_out"), ({"dq": (64 * KB + 64, 384, 128, 32)}, b"dq overlaps q"),
    ({"dq": (88 * KB, 384, 128, 32)}, b"dq overlaps dk_out"), ({"dk": (84 * KB, 192, 64, 32)}, b"dq overlaps dk"),
    ({"dk": (64 * KB, 192, 64, 32)}, b"dk overlaps q"), ({"dk": (92 * KB, 64, 64, 32)}, b"rows of dk overlap"),
])
def test_head_norm_gradient(lib, grads, text):
    given = dict(dq_out=(80 * KB, 384, 128, 32), dq=(84 * KB, 384, 128, 32), dk_out=(88 * KB, 192, 64, 32), dk=(92 * KB, 192, 64, 32))
    g = fill(abi.HeadNormGradsC(), **{**given, **grads})
    assert lib.tdgs_head_norm_grad(None, C.byref(head_norm()), C.byref(g)) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error(), lib.tdgs_last_error()


def rand(*shape, seed=0, t=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(t).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_columns_of_one_buffer(gpu, t):
    """x, residual, out, pre and the gradients side by side in the rows of one buffer."""
    m, k, n = 300, 40, 24
    buffer = rand(m, 2 * k + 4 * n, t=t)
    x, res, out, pre, dout, dx = buffer.split([k, n, n, n, n, k], dim=1)
    w = rand(k, n, seed=1, t=t) / 6
    kept = [v.clone() for v in (x, res, dout)]
    wants = [torch.empty((m, n), dtype=t, device="cuda") for _ in range(2)] + [torch.empty((m, k), dtype=t, device="cuda")]
    dw, want_dw = torch.empty_like(w), torch.empty_like(w)
    decoder.linear_(wants[0], kept[0], w, residual=kept[1], activation="silu", pre=wants[1])
    decoder.linear_grad_(wants[2], want_dw, None, kept[2], kept[0], w, activation="silu", pre=wants[1])
    decoder.linear_(out, x, w, residual=res, activation="silu", pre=pre)
    decoder.linear_grad_(dx, dw, None, dout, x, w, activation="silu", pre=pre)
    for got, want in zip((out, pre, dx, dw, x, res, dout), (*wants, want_dw, *kept)):
        assert (got.double() - want.double()).norm() <= torch.finfo(t).eps * want.double().norm()
    # dropout between columns, and rows of x that are all one row
    a, b = rand(50, 24).split([16, 8], dim=1)
    want = decoder.dropout(a[:, :8].contiguous(), 0.4, 3, residual=b.contiguous())
    assert torch.equal(decoder.dropout_(b, a[:, :8], 0.4, 3, residual=b), want)
    row = rand(1, 16).expand(50, 16)
    assert torch.equal(decoder.dropout_(torch.empty((50, 16), device="cuda"), row, 0.4, 3), decoder.dropout(row.contiguous(), 0.4, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["fused", "heads_first", "padded", "every_second"])
def test_heads_in_place(gpu, layout):
    """Queries and keys of one buffer, in place, in several orders of its dimensions."""
    b, l, h, hk, d = 2, 5, 4, 2, 16
    make = {"fused": lambda s: rand(b, l, h + hk, d, seed=s), "heads_first": lambda s: rand(b, h + hk, l, d, seed=s).transpose(1, 2),
            "padded": lambda s: rand(b, l, h + hk, d + 4, seed=s)[..., :d], "every_second": lambda s: rand(b, 2 * l, h + hk, d, seed=s)[:, ::2]}[layout]
    q, k = make(1)[:, :, :h], make(1)[:, :, h:]
    both, dboth = make(1), make(2)
    rotary, places = decoder.Rotary((8,)), torch.arange(l, device="cuda")[:, None]
    wq = 1 + 0.1 * rand(d, seed=4)
    want = decoder.head_norm(q, k, wq, rotary=rotary, positions=places)
    dwant = [torch.empty((b, l, n, d), device="cuda") for n in (h, hk)]
    decoder.head_norm_grad_(*dwant, None, None, dboth[:, :, :h].clone(), dboth[:, :, h:].clone(), q, k, wq, rotary=rotary, positions=places)
    decoder.head_norm_grad_(dboth[:, :, :h], dboth[:, :, h:], None, None, dboth[:, :, :h], dboth[:, :, h:], q, k, wq, rotary=rotary,
                            positions=places)
    decoder.head_norm_(both[:, :, :h], both[:, :, h:], both[:, :, :h], both[:, :, h:], wq, rotary=rotary, positions=places)
    for got, w in zip((both, dboth), (want, dwant)):
        assert torch.equal(got[:, :, :h], w[0]) and torch.equal(got[:, :, h:], w[1])
