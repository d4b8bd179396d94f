"""Rotations of no tokens: their positions are an empty tensor, which has no address."""
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


@pytest.mark.parametrize("batch,length", [(0, 3), (2, 0), (0, 0)])
def test_no_tokens(lib, batch, length):
    turns = (C.c_double * 4)()
    a = abi.HeadNormC(dtype=abi.TDGS_F32, batch=batch, length=length, heads=2, head_dim=8, norm=1, eps=1e-6, pairs=4, axes=1,
                      turns=C.addressof(turns))
    a.sections[0] = 4
    assert lib.tdgs_head_norm_forward(None, C.byref(a)) == abi.TDGS_OK, lib.tdgs_last_error()
    a.batch, a.length = 2, 3
    assert lib.tdgs_head_norm_forward(None, C.byref(a)) == abi.TDGS_ERR_INVALID and b"positions are null" in lib.tdgs_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 0, 4, 8), (0, 3, 4, 8), (2, 3, 0, 8)], ids=str)
@pytest.mark.parametrize("batched", [False, True])
def test_python(gpu, shape, batched):
    b, l, h, d = shape
    rotary = decoder.Rotary((2, 2))
    places = torch.zeros((b, l, 2) if batched else (l, 2), dtype=torch.int64, device="cuda")
    q, w = torch.zeros(shape, device="cuda").requires_grad_(True), torch.ones(d, device="cuda").requires_grad_(True)
    y = decoder.rotate(decoder.head_norm(q, None, w, rotary=rotary, positions=places), None, rotary, places)
    assert y.shape == shape
    y.sum().backward()
    assert q.grad.shape == shape and not w.grad.any()
