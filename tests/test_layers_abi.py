"""Linear layers, head norms and dropout without a GPU: struct mirrors, packed forms, the arguments that the C calls and the
Python functions refuse before they touch the device, and the device they are launched on."""
import contextlib
import ctypes as C
import os
import random
import subprocess

import pytest
import torch

from conftest import ROOT
from tdgs_amd import abi, core, decoder

HEADER = os.path.join(ROOT, "include", "tdgs.h")
STRUCTS = {"tdgs_rows": abi.RowsC, "tdgs_linear": abi.LinearC, "tdgs_linear_grads": abi.LinearGradsC,
           "tdgs_head_norm": abi.HeadNormC, "tdgs_head_norm_grads": abi.HeadNormGradsC, "tdgs_dropout": abi.DropoutC}


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(core.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return core.lib()


def test_mirrors_match_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, py in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True).stdout.split()]
    want = []
    for py in STRUCTS.values():
        want.append(C.sizeof(py))
        want += [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want


def flat(s):
    out = []
    for f, t in s._fields_:
        v = getattr(s, f)
        out += flat(v) if isinstance(v, C.Structure) else list(v) if isinstance(v, C.Array) else [v]
    return out


def test_packed_layouts():
    """The packed forms put every field where the structures have it."""
    for packer, py, values in (
            (decoder._LINEAR, abi.LinearC, range(1, 21)), (decoder._LINEAR_GRADS, abi.LinearGradsC, range(1, 10)),
            (decoder._HEAD_NORM, abi.HeadNormC, [*range(1, 9), 0.5, *range(10, 42)]),
            (decoder._HEAD_NORM_GRADS, abi.HeadNormGradsC, range(1, 19)),
            (decoder._DROPOUT, abi.DropoutC, [1, 2, 3, 4, 0.25, *range(6, 15)])):
        assert flat(py.from_buffer_copy(packer.pack(*values))) == list(values)


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
    given = dict(dtype=abi.TDGS_BF16, rows=8, in_features=16, out_features=24, x=(64, 16), weight=(128, 24), out=(192, 24), temp=64,
                 temp_bytes=1 << 30, pre=(256, 24))
    return fill(abi.LinearC(), **{**given, **kw})


@pytest.mark.parametrize("kw,text", [
    ({"dtype": 3}, b"element type"), ({"activation": 4}, b"activation"), ({"activation": -1}, b"activation"),
    ({"rows": -1}, b"rows"), ({"rows": 2 ** 31}, b"rows"), ({"in_features": 0}, b"weight matrix"),
    ({"out_features": 2 ** 21}, b"weight matrix"), ({"in_features": 2 ** 20, "out_features": 2 ** 20}, b"weight matrix"),
    ({"weight_layout": 2}, b"weight layout"), ({"x": (0, 16)}, b"x is null"), ({"x": (65, 16)}, b"x is not aligned"),
    ({"weight": (0, 24)}, b"the weight is null"), ({"out": (0, 24)}, b"out is null"), ({"out": (192, 23)}, b"rows of out overlap"),
    ({"out": (192, -24)}, b"negative stride"), ({"pre": (256, 5)}, b"rows of pre overlap"), ({"residual": (65, 24)}, b"residual"),
    ({"out": (64, 24)}, b"out is also an operand"), ({"out": (128, 24)}, b"out is also an operand"),
    ({"pre": (192, 24)}, b"pre is also"), ({"pre": (64, 24)}, b"pre is also"), ({"residual": (256, 24)}, b"pre is also"),
    ({"bias": 65}, b"bias"), ({"x": (64, 2 ** 24)}, b"too far apart"), ({"weight": (64, 2 ** 24)}, b"too far apart"),
    ({"rows": 64, "in_features": 4096, "weight": (64, 24), "x": (64, 4096), "temp_bytes": 0}, b"scratch"),
])
def test_linear_refusals(lib, kw, text):
    assert lib.tdgs_linear_forward(None, C.byref(linear(**kw))) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error(), lib.tdgs_last_error()
    assert lib.tdgs_linear_forward(None, None) == abi.TDGS_ERR_INVALID


@pytest.mark.parametrize("kw,grads,text", [
    ({}, {"dout": (0, 24)}, b"dout is null"), ({}, {"dx": (384, 15)}, b"rows of dx overlap"),
    ({}, {"dweight_layout": 5}, b"weight layout"), ({}, {"dweight": (448, 23)}, b"rows of dweight"),
    ({}, {"dbias": 65}, b"dbias"), ({"activation": 1, "pre": (0, 24)}, {}, b"pre is null"), ({"x": (0, 16)}, {"dx": (0, 0)}, b"x is null"),
    ({"temp_bytes": 16}, {}, b"scratch"), ({"temp": 8}, {}, b"scratch"), ({}, {"dout": (320, 2 ** 24)}, b"too far apart"),
    ({}, {"dx": (320, 24)}, b"dx is also"), ({}, {"dx": (64, 16)}, b"dx is also"), ({"activation": 1}, {"dx": (256, 24)}, b"dx is also"),
    ({}, {"dx": (448, 24)}, b"dx is also"), ({}, {"dweight": (320, 24)}, b"dweight is also"), ({}, {"dweight": (64, 24)}, b"dweight is also"),
    ({}, {"dweight": (128, 24)}, b"dweight is also"),
])
def test_linear_gradient_refusals(lib, kw, grads, text):
    g = fill(abi.LinearGradsC(), **{**dict(dout=(320, 24), dx=(384, 16), dweight=(448, 24), dbias=64), **grads})
    assert lib.tdgs_linear_grad(None, C.byref(linear(**kw)), C.byref(g)) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error(), lib.tdgs_last_error()
    assert lib.tdgs_linear_grad(None, C.byref(linear()), None) == abi.TDGS_ERR_INVALID


def test_linear_scratch_follows_sizes(lib):
    size = lib.tdgs_linear_temp_bytes
    assert size(C.byref(linear(dtype=9)), 1) == 0
    assert size(C.byref(linear(rows=0)), 1) >= 0
    r = random.Random(0)
    for _ in range(300):
        a = linear(dtype=r.randint(0, 2), activation=r.randint(0, 3), rows=int(2 ** r.uniform(0, 20)),
                   in_features=int(2 ** r.uniform(0, 13)), out_features=int(2 ** r.uniform(0, 13)))
        n, g = size(C.byref(a), 0), size(C.byref(a), 1)
        # partial sums take a few times the results, never a multiple of the operands' product
        results = a.rows * a.out_features + a.rows * a.in_features + a.in_features * a.out_features
        assert n <= g <= 16 * results + 4 * 2048 * (65536 + 8 * a.out_features) + 65536


def head_norm(**kw):
    given = dict(dtype=abi.TDGS_BF16, param_dtype=abi.TDGS_F32, batch=2, length=3, heads=4, kv_heads=2, head_dim=32, norm=1,
                 eps=1e-6, pairs=8, axes=2, sections=(4, 4, 0, 0), turns=64, positions=64, q=(64, 384, 128, 32),
                 q_out=(64, 384, 128, 32), k=(64, 192, 64, 32), k_out=(64, 192, 64, 32))
    return fill(abi.HeadNormC(), **{**given, **kw})


@pytest.mark.parametrize("kw,text", [
    ({"dtype": 5}, b"element type"), ({"param_dtype": abi.TDGS_F16}, b"weights"), ({"batch": -1}, b"negative"),
    ({"heads": 70000}, b"heads"), ({"batch": 65536, "length": 65536}, b"tokens"), ({"head_dim": 0}, b"head dimension"),
    ({"head_dim": 257}, b"head dimension"), ({"eps": -1.0}, b"eps"), ({"eps": float("nan")}, b"eps"), ({"pairs": 17}, b"rotated pairs"),
    ({"pairs": -1}, b"rotated pairs"), ({"axes": 5}, b"axes"), ({"axes": 0}, b"axes"), ({"sections": (8, 0, 0, 0)}, b"axis 1"),
    ({"sections": (4, 5, 0, 0)}, b"have 9 pairs"), ({"pair_layout": 2}, b"layout of pairs"), ({"position_type": 3}, b"positions"),
    ({"turns": 0}, b"frequencies"), ({"positions": 0}, b"positions are null"), ({"position_batch_stride": -1}, b"stride"),
    ({"q": (0, 1, 1, 1)}, b"q is null"), ({"q_out": (64, 384, 128, 31)}, b"rows of q_out overlap"),
    ({"k": (65, 192, 64, 32)}, b"k is not aligned"), ({"k_out": (64, 192, 64, -32)}, b"negative stride"),
])
def test_head_norm_refusals(lib, kw, text):
    assert lib.tdgs_head_norm_forward(None, C.byref(head_norm(**kw))) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error(), lib.tdgs_last_error()


def test_head_norm_gradient_refusals(lib):
    views = dict(dq_out=(64, 384, 128, 32), dq=(64, 384, 128, 32), dk_out=(64, 192, 64, 32), dk=(64, 192, 64, 32))
    for kw, grads, text in (({"norm": 0}, {}, b"inverse rotation"), ({}, {"dq_out": (0, 0, 0, 0)}, b"dq_out is null"),
                            ({}, {"dk": (64, 1, 64, 32)}, b"rows of dk overlap"), ({}, {"dq_weight": 64}, b"scratch"),
                            ({"temp": 64, "temp_bytes": 100}, {"dk_weight": 64}, b"scratch")):
        g = fill(abi.HeadNormGradsC(), **{**views, **grads})
        assert lib.tdgs_head_norm_grad(None, C.byref(head_norm(**kw)), C.byref(g)) == abi.TDGS_ERR_INVALID
        assert text in lib.tdgs_last_error(), lib.tdgs_last_error()
    assert lib.tdgs_head_norm_grad(None, C.byref(head_norm()), None) == abi.TDGS_ERR_INVALID
    assert lib.tdgs_head_norm_temp_bytes(C.byref(head_norm())) >= 6 * 2 * 32 * 4


@pytest.mark.parametrize("kw,text", [
    ({"dtype": 3}, b"element type"), ({"rows": -1}, b"rows"), ({"rows": 2 ** 40, "cols": 2 ** 40}, b"rows"), ({"p": -0.1}, b"probability"),
    ({"p": 1.5}, b"probability"), ({"p": float("nan")}, b"probability"), ({"x": (0, 5)}, b"x is null"), ({"out": (64, 4)}, b"rows of out"),
    ({"residual": (66, 5)}, b"residual"), ({"call_dev": 4}, b"calls"),
])
def test_dropout_refusals(lib, kw, text):
    a = fill(abi.DropoutC(), **{**dict(dtype=0, rows=3, cols=5, p=0.5, x=(64, 5), out=(64, 5)), **kw})
    assert lib.tdgs_dropout_apply(None, C.byref(a)) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error(), lib.tdgs_last_error()


class OnDevice(torch.Tensor):
    """A tensor that says it is on GPU 1."""
    is_cuda = True
    device = torch.device("cuda", 1)

    def get_device(self):
        return 1


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)


class Turns(decoder.Rotary):
    def __init__(self, *sections):
        self.sections, self.pairs, self.layout, self.axes = sections, sum(sections), "halves", len(sections)
        self.turns = t(self.pairs, dtype=torch.float64)
        self.device, self.pointer = 1, 64
        self._fields = (self.pairs, 0, self.axes, *sections, *(0,) * (4 - self.axes))


@pytest.fixture
def device(monkeypatch):
    """The library and the devices as stand-ins: the calls seen, with the device that was current."""
    now, seen = [0], []

    @contextlib.contextmanager
    def as_current(d):
        before, now[0] = now[0], d
        yield
        now[0] = before

    class Library:
        def __getattr__(self, entry):
            return lambda *args: 64 if entry.endswith("temp_bytes") else seen.append((entry, now[0])) or 0

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", as_current)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    monkeypatch.setattr(decoder, "lib", Library)
    return now, seen


@pytest.mark.parametrize("current", [0, 1])
def test_launched_on_the_tensors_device(device, current):
    now, seen = device
    now[0] = current
    x, w, o, q, temp = t(3, 4), t(4, 5), t(3, 5), t(1, 2, 3, 8), t(64, dtype=torch.uint8)
    places = t(2, 1, dtype=torch.int32)
    decoder.linear_(o, x, w, temp=temp)
    decoder.linear_grad_(x, w, None, o, x, w, temp=temp)
    decoder.head_norm_(q, None, q, rotary=Turns(4), positions=places)
    decoder.head_norm_grad_(q, None, None, None, q, None, q, temp=temp)
    decoder.rotate_(q, None, q, None, Turns(4), places)
    decoder.dropout_(x, x, 0.5, 1)
    assert [d for _, d in seen] == [1] * 6 and now == [current]


def test_python_refusals(device):
    x, w, o, b = t(3, 4), t(4, 5), t(3, 5), t(5)
    host = torch.zeros(3, 4)
    half = t(3, 4, dtype=torch.float16)
    q, k = t(2, 3, 4, 8), t(2, 3, 2, 8)
    r, places = Turns(2, 2), t(3, 2, dtype=torch.int64)
    temp = t(64, dtype=torch.uint8)
    calls = [
        lambda: decoder.linear_(o, host, w), lambda: decoder.linear_(o, x, torch.zeros(4, 5)), lambda: decoder.linear_(torch.zeros(3, 5), x, w),
        lambda: decoder.linear_(o, half, w), lambda: decoder.linear_(o, t(3, 6), w), lambda: decoder.linear_(t(3, 6), x, w),
        lambda: decoder.linear_(o, x, w, t(4)), lambda: decoder.linear_(o, x, w, b.half()), lambda: decoder.linear_(o, x, w, activation="tanh"),
        lambda: decoder.linear_(o, x, w, residual=t(3, 4)), lambda: decoder.linear_(o, x, w, pre=t(2, 5)),
        lambda: decoder.linear_(o, t(3, 8)[:, ::2], w), lambda: decoder.linear_(o, x, t(8, 10)[::2, ::2]), lambda: decoder.linear_(o, x, t(4)),
        lambda: decoder.linear_(t(2, 2, 3, 5), t(3, 2, 2, 4).transpose(0, 2), w), lambda: decoder.linear_(o, x, w, temp=t(4)),
        lambda: decoder.linear_grad_(x, w, b, o, x, w, activation="gelu"), lambda: decoder.linear_grad_(x, t(5, 4), b, o, x, w),
        lambda: decoder.linear_grad_(x, w, t(4), o, x, w), lambda: decoder.linear_grad_(o, w, b, o, x, w),
        lambda: decoder.head_norm_(q, None, t(3, 4, 8)), lambda: decoder.head_norm_(q, k, q), lambda: decoder.head_norm_(q, None, q, k),
        lambda: decoder.head_norm_(q, k, q, t(2, 4, 2, 8)), lambda: decoder.head_norm_(q, None, q, q_weight=t(7)),
        lambda: decoder.head_norm_(q, k, q, k, t(8), t(8).half()), lambda: decoder.head_norm_(q, None, q, None, t(8).bfloat16()),
        lambda: decoder.head_norm_(q, None, q, positions=places), lambda: decoder.head_norm_(q, None, q, rotary=r),
        lambda: decoder.head_norm_(q, None, q, rotary=r, positions=places.double()),
        lambda: decoder.head_norm_(q, None, q, rotary=r, positions=t(3, 1, dtype=torch.int64)),
        lambda: decoder.head_norm_(q, None, q, rotary=r, positions=t(2, 3, dtype=torch.int64).T),
        lambda: decoder.head_norm_(q, None, t(2, 3, 4, 16)[..., ::2]), lambda: decoder.rotate_(q, None, q, None, None, places),
        lambda: decoder.head_norm_grad_(q, None, t(7), None, q, None, q, temp=temp),
        lambda: decoder.head_norm_grad_(q, None, t(8).half(), None, q, None, q, temp=temp),
        lambda: decoder.dropout_(x, x, 1.1, 0), lambda: decoder.dropout_(x, x, float("nan"), 0), lambda: decoder.dropout_(x, host, 0.1, 0),
        lambda: decoder.dropout_(x, x, 0.1, 0, call=t(1)), lambda: decoder.dropout_(x, x, 0.1, 0, call=t(2, dtype=torch.int64)),
        lambda: decoder.dropout_(x, x, 0.1, 0, residual=o), lambda: decoder.dropout_(x, t(), 0.1, 0), lambda: decoder.dropout_(x, half, 0.1, 0),
        lambda: decoder.Rotary(()), lambda: decoder.Rotary((1, 0)), lambda: decoder.Rotary((1,) * 5), lambda: decoder.Rotary((2,), pairs="odd"),
        lambda: decoder.Rotary((2,), base=0.0), lambda: decoder.Rotary((2,), frequencies=[1.0]),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} went through")
    assert not device[1]


def test_weights_of_one_row_or_column(device):
    """Matrices whose strides say nothing: which way round they lie does not matter, but their row stride has to hold."""
    like = t(1, 1)
    for w in (t(4, 1), t(1, 4), t(1, 1), t(4, 1).T, t(4, 9)[:, :1], t(9, 4)[:1].T):
        layout, _, stride = decoder._weight(w, "w", like)
        rows, cols = w.shape if layout == abi.TDGS_WEIGHT_IN_OUT else w.shape[::-1]
        step, element = w.stride() if layout == abi.TDGS_WEIGHT_IN_OUT else w.stride()[::-1]
        assert (cols == 1 or element == 1) and (rows == 1 or stride == step >= cols)
