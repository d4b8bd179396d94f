"""The decoder operators' C-ABI without a GPU: struct mirrors, and the arguments that the calls refuse
before they touch the device."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import ROOT
from tdgs_amd import abi, core, decoder

HEADER = os.path.join(ROOT, "include", "tdgs.h")
STRUCTS = {"tdgs_heads": abi.HeadsC, "tdgs_attention": abi.AttentionC, "tdgs_attention_grads": abi.AttentionGradsC,
           "tdgs_pixels": abi.PixelsC, "tdgs_norm": abi.NormC, "tdgs_norm_grads": abi.NormGradsC}


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


def test_packed_layouts():
    """The packed forms put every field where the structures have it."""
    a = abi.AttentionC.from_buffer_copy(decoder._ATTENTION.pack(*range(1, 9), 0.5, 0, *range(100, 116), *range(200, 206)))
    assert (a.dtype, a.batch, a.kv_batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim) == tuple(range(1, 9))
    assert a.scale == 0.5
    assert [getattr(v, f) for v in (a.q, a.k, a.v, a.out) for f in ("data", "stride_b", "stride_l", "stride_h")] \
        == list(range(100, 116))
    assert [a.kv_lengths, a.kv_mask, a.kv_mask_stride, a.lse, a.temp, a.temp_bytes] == list(range(200, 206))
    g = abi.AttentionGradsC.from_buffer_copy(decoder._ATTENTION_GRADS.pack(*range(1, 17)))
    assert [getattr(v, f) for v in (g.dout, g.dq, g.dk, g.dv) for f in ("data", "stride_b", "stride_l", "stride_h")] \
        == list(range(1, 17))
    n = abi.NormC.from_buffer_copy(decoder._NORM.pack(*range(1, 7), 0.25, 0, 9, *range(20, 26), *range(30, 35)))
    assert (n.dtype, n.param_dtype, n.n, n.channels, n.groups, n.activation, n.eps, n.pixels) == (1, 2, 3, 4, 5, 6, 0.25, 9)
    assert [getattr(v, f) for v in (n.x, n.out) for f in ("data", "stride_n", "stride_p")] == list(range(20, 26))
    assert [n.weight, n.bias, n.stats, n.temp, n.temp_bytes] == list(range(30, 35))
    d = abi.NormGradsC.from_buffer_copy(decoder._NORM_GRADS.pack(*range(1, 9)))
    assert [d.dout.data, d.dout.stride_n, d.dout.stride_p, d.dx.data, d.dx.stride_n, d.dx.stride_p, d.dweight, d.dbias] \
        == list(range(1, 9))


def _attention(**kw):
    a = abi.AttentionC()
    a.dtype, a.batch, a.kv_batch, a.q_len, a.kv_len, a.heads, a.kv_heads, a.head_dim = abi.TDGS_BF16, 2, 2, 8, 9, 4, 2, 32
    a.scale = 0.1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,text", [
    ({"dtype": 7}, b"element type"), ({"heads": 3}, b"do not divide"), ({"kv_heads": 0}, b"do not divide"),
    ({"kv_batch": 3}, b"neither"), ({"head_dim": 0}, b"head dimension"), ({"head_dim": 129}, b"head dimension"),
    ({"scale": 0.0}, b"scale"), ({"scale": float("nan")}, b"scale"), ({"q_len": -1}, b"negative"),
    ({"q_len": 2 ** 31 - 1}, b"too many"), ({}, b"q is null"),
])
def test_attention_refusals(lib, kw, text):
    a = _attention(**kw)
    assert lib.tdgs_cross_attention(None, C.byref(a)) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error()
    assert lib.tdgs_cross_attention_grad(None, C.byref(a), C.byref(abi.AttentionGradsC())) == abi.TDGS_ERR_INVALID


def test_attention_scratch_follows_sizes(lib):
    size = lib.tdgs_cross_attention_temp_bytes
    assert size(C.byref(_attention(dtype=9)), 0) == 0
    small, long = size(C.byref(_attention(q_len=1)), 0), size(C.byref(_attention(q_len=1, kv_len=50000)), 0)
    assert long > small
    assert size(C.byref(_attention()), 1) >= size(C.byref(_attention()), 0)
    assert size(C.byref(_attention(q_len=0)), 1) >= 0 and size(C.byref(_attention(kv_len=0)), 1) >= 0


def _norm(**kw):
    a = abi.NormC()
    a.dtype, a.param_dtype, a.n, a.channels, a.groups, a.eps, a.pixels = abi.TDGS_F16, abi.TDGS_F32, 1, 32, 4, 1e-5, 10
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,text", [
    ({"dtype": -1}, b"element type"), ({"param_dtype": abi.TDGS_BF16}, b"weight and bias"), ({"groups": 5}, b"do not divide"),
    ({"groups": 0}, b"do not divide"), ({"channels": 0}, b"do not divide"), ({"activation": 4}, b"activation"),
    ({"eps": -1.0}, b"eps"), ({"eps": float("inf")}, b"eps"), ({"n": 70000}, b"images"), ({"pixels": -1}, b"pixels"),
    ({}, b"is null"),
])
def test_norm_refusals(lib, kw, text):
    a = _norm(stats=64, **kw)
    assert lib.tdgs_group_norm(None, C.byref(a)) == abi.TDGS_ERR_INVALID
    assert text in lib.tdgs_last_error()
    assert lib.tdgs_group_norm_grad(None, C.byref(a), C.byref(abi.NormGradsC())) == abi.TDGS_ERR_INVALID


def test_embedding_refusals(lib):
    def lookup(ctx=64, dtype=0, stride=8, vocab=20, dim=8, size=4, n=3, out=64):
        return lib.tdgs_embedding_lookup(ctx, None, dtype, 64, stride, vocab, dim, 64, size, n, 1.0, out, 8)

    for kw, text in (({"ctx": None}, b"context"), ({"dtype": 3}, b"element type"), ({"size": 2}, b"bytes"),
                     ({"dim": 0}, b"rows of 0"), ({"vocab": 2 ** 31}, b"table of"), ({"n": 2 ** 31}, b"tokens"),
                     ({"out": None}, b"out is null"), ({"out": 66}, b"aligned")):
        assert lookup(**kw) == abi.TDGS_ERR_INVALID, kw
        assert text in lib.tdgs_last_error()
    assert lib.tdgs_embedding_grad_temp_bytes(100000, 50, 8) > 100000 * 8
    assert lib.tdgs_embedding_grad_temp_bytes(-1, 50, 8) == 0
    assert lib.tdgs_embedding_grad(64, None, 0, 64, 8, 64, 4, 100000, -1, 1.0, 64, 8, 50, 8, 64, 16) == abi.TDGS_ERR_INVALID
    assert b"scratch" in lib.tdgs_last_error()
