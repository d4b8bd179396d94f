"""Calls whose tokens or rows make more workgroups than one launch takes (2^32 threads): walked over, or refused by name."""
import ctypes as C
import os

import pytest
import torch

from tdgs_amd import abi, core, decoder


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(core.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return core.lib()


@pytest.mark.parametrize("features", [1, 2, 64])
def test_too_many_tiles(lib, features):
    """2^30 rows and more by tiles of 64 (addresses that are never used, each tensor in 2^45 bytes of its own)."""
    a = abi.LinearC(dtype=abi.TDGS_F32, rows=2 ** 31 - 2 ** 21, in_features=features, out_features=1, temp=64, temp_bytes=1 << 40)
    for i, name in enumerate(("x", "weight", "out")):
        getattr(a, name).data, getattr(a, name).stride = (i + 1) << 45, features if name == "x" else 1
    assert lib.tdgs_linear_forward(None, C.byref(a)) == abi.TDGS_ERR_INVALID
    assert b"too many tiles" in lib.tdgs_last_error(), lib.tdgs_last_error()


@pytest.mark.gpu
def test_heads_of_2_to_the_30_tokens(gpu):
    """More than 2^24 workgroups' worth of tokens, rotated in place: those in the middle and at the end are a small call's."""
    n = 2 ** 30 + 4097
    q = torch.zeros((1, n, 1, 2), dtype=torch.bfloat16, device="cuda")
    places = torch.zeros((n, 1), dtype=torch.int32, device="cuda")
    rotary = decoder.Rotary((1,))
    at = (slice(0, 100), slice(n // 2, n // 2 + 100), slice(n - 100, n))
    given = torch.randn((3, 1, 100, 1, 2), generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    steps = torch.arange(300, dtype=torch.int32, device="cuda").reshape(3, 100, 1)
    for i, s in enumerate(at):
        q[:, s], places[s] = given[i], steps[i]
    decoder.rotate_(q, None, q, None, rotary, places)
    for i, s in enumerate(at):
        assert torch.equal(q[:, s], decoder.rotate(given[i], None, rotary, steps[i]))
    assert int((q[:, :, 0].view(torch.int32) != 0).sum()) <= 300   # (the rest stays zero)


@pytest.mark.gpu
def test_no_rows_and_a_weight_of_more_than_2_to_the_32(gpu):
    """The weight's gradient is zero in every element, also behind what 2^32 threads would reach."""
    t = torch.float16
    k, n = 2 ** 17, 2 ** 15 + 8
    x, dout = torch.empty((0, k), dtype=t, device="cuda"), torch.empty((0, n), dtype=t, device="cuda")
    dw = torch.full((k, n), 5.0, dtype=t, device="cuda")
    decoder.linear_grad_(None, dw, None, dout, x, dw)
    assert not dw[-1].any() and not dw[::4099].any() and int(torch.count_nonzero(dw[k // 2:])) == 0
