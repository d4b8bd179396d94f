"""Head norms refuse weights, and gradients of weights, off their type's alignment, as they do every other tensor."""
import ctypes as C
import os

import pytest

from tdgs_amd import abi, core

KB = 1 << 10


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(core.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return core.lib()


def views(s, **at):
    for name, (data, heads) in at.items():
        v = getattr(s, name)
        v.data, v.stride_b, v.stride_l, v.stride_h = data, 3 * heads * 32, heads * 32, 32
    return s


@pytest.mark.parametrize("param,off", [(abi.TDGS_F32, 2), (abi.TDGS_BF16, 1)])
@pytest.mark.parametrize("name", ["q_weight", "k_weight", "dq_weight", "dk_weight"])
def test_weights(lib, param, off, name):
    a = abi.HeadNormC(dtype=abi.TDGS_BF16, param_dtype=param, batch=2, length=3, heads=4, kv_heads=2, head_dim=32, norm=1, eps=1e-6,
                      temp=1 << 30, temp_bytes=1 << 30)
    views(a, q=(64 * KB, 4), q_out=(68 * KB, 4), k=(72 * KB, 2), k_out=(76 * KB, 2))
    g = views(abi.HeadNormGradsC(), dq_out=(80 * KB, 4), dq=(84 * KB, 4), dk_out=(88 * KB, 2), dk=(92 * KB, 2))
    setattr(g if name.startswith("d") else a, name, 96 * KB + off)
    assert lib.tdgs_head_norm_grad(None, C.byref(a), C.byref(g)) == abi.TDGS_ERR_INVALID
    assert b"not aligned" in lib.tdgs_last_error(), lib.tdgs_last_error()
    if not name.startswith("d"):
        assert lib.tdgs_head_norm_forward(None, C.byref(a)) == abi.TDGS_ERR_INVALID
        assert b"not aligned" in lib.tdgs_last_error(), lib.tdgs_last_error()
