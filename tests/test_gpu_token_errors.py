"""A token outside an embedding's table is an error of the embedding call, and of no other on its context."""
import ctypes as C

import numpy as np
import pytest
import torch

from tdgs_amd import appearance, core, decoder, host, synthetic

pytestmark = pytest.mark.gpu


def _bad_lookup(ctx=None):
    table = torch.randn((20, 8), device="cuda")
    decoder.embedding_lookup_(torch.empty((2, 8), device="cuda"), table, torch.tensor([3, 20], device="cuda"), ctx=ctx)


@pytest.mark.parametrize("grad", [False, True], ids=["lookup", "grad"])
def test_renders_and_scans_go_on(gpu, grad):
    ctx = core.Context(0)
    if grad:
        n = 100000   # the tokens are sorted
        tokens = torch.full((n,), -5, device="cuda")
        decoder.embedding_grad_(torch.empty((20, 8), device="cuda"), torch.ones((n, 8), device="cuda"), tokens, ctx=ctx)
    else:
        _bad_lookup(ctx)
    w = synthetic.config(0, n=500)
    cam = w.cameras[0]
    t = host.Tiling.for_camera(cam, 16, 16)
    g = gpu.TrainableGaussiansVector.from_host(w.gaussians, 0)
    options = host.RenderOptions.for_camera(cam, w.gaussians.sh_degree)
    for device_counts in (False, True):
        out = gpu.RenderOutputs.for_camera(cam, 0)
        gpu.render_(out, g, cam, t, options, gpu.RenderBuffers(len(g), t, 0, 100_000), device_counts=device_counts, ctx=ctx)
    torch.cuda.synchronize()
    monitor = C.POINTER(C.c_int64)()
    core.check(core.lib().tdgs_ctx_frame_monitor(ctx.handle, C.byref(monitor)))
    assert (monitor[0], monitor[4]) == (1, 0)   # no error of the frame with its counts on the device
    with pytest.raises(core.TdgsError, match="outside its table"):
        core.ctx_check(0, ctx)
    core.ctx_check(0, ctx)


@pytest.mark.parametrize("image", [-1, 3, np.int64(5)])
def test_photographs_outside_the_collection(gpu, image):
    """Refused on the host, before any token is looked up."""
    dec = appearance.AppearanceDecoder(3, channels=32, groups=4)
    with pytest.raises(ValueError, match="of a collection of 3"):
        dec(torch.rand((8, 8, 3), device="cuda"), image)
    dec(torch.rand((8, 8, 3), device="cuda"), 2)
    core.ctx_check(0)
