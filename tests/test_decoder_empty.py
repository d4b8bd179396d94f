"""The decoder operators' C-ABI without a GPU: calls with nothing to do."""
import ctypes as C

from tdgs_amd import abi
from test_decoder_abi import _attention, lib  # noqa: F401


def test_no_batches_of_shared_states(lib):  # noqa: F811
    """There are gradients of the states to write (zeros), so the call is checked as any other."""
    a = _attention(batch=0, kv_batch=1)
    assert lib.tdgs_cross_attention(None, C.byref(a)) == abi.TDGS_OK
    g = abi.AttentionGradsC()
    assert lib.tdgs_cross_attention_grad(None, C.byref(a), C.byref(g)) == abi.TDGS_OK   # (not wanted)
    g.dk.data = g.dv.data = 64
    assert lib.tdgs_cross_attention_grad(None, C.byref(a), C.byref(g)) == abi.TDGS_ERR_INVALID
    assert b"k is null" in lib.tdgs_last_error()
    a.kv_lengths = 64
    assert lib.tdgs_cross_attention_temp_bytes(C.byref(a), 1) >= 4 * (9 + 1)   # the list of keys


def test_nothing_at_all(lib):  # noqa: F811
    for kw in (dict(batch=0, kv_batch=0), dict(batch=0, kv_batch=1, kv_len=0), dict(q_len=0, kv_len=0)):
        a = _attention(**kw)
        assert lib.tdgs_cross_attention_grad(None, C.byref(a), C.byref(abi.AttentionGradsC())) == abi.TDGS_OK
