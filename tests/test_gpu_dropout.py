"""Dropout by a counter-based generator, against the generator in numpy's integers."""
import numpy as np
import pytest
import torch

from tdgs_amd import decoder

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def words(n, seed, call):
    low, by = np.uint64(2 ** 32 - 1), np.uint64(32)
    c = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [c & low, c >> by, np.full_like(c, call & 0xFFFFFFFF), np.full_like(c, call >> 32)]
    for r in range(10):
        k = [np.uint64((seed + 0x9E3779B9 * r) & 0xFFFFFFFF), np.uint64(((seed >> 32) + 0xBB67AE85 * r) & 0xFFFFFFFF)]
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> by) ^ c[1] ^ k[0], b & low, (a >> by) ^ c[3] ^ k[1], a & low]
    return np.stack(c, 1).reshape(-1)[:n]


def test_generator():
    """The published vectors of Philox4x32-10: counter and key of zeros, of ones."""
    assert [int(w) for w in words(4, 0, 0)] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


def want(x, p, seed, call, residual=None):
    keep = torch.from_numpy(words(x.numel(), seed, call) >= np.uint64(int(p * 2.0 ** 32))).reshape(x.shape).cuda()
    y = torch.where(keep, x.double() / (1 - p) if p < 1 else 0.0, 0.0)
    return keep, y if residual is None else y + residual.double()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", [(1,), (3,), (5, 1), (1, 7), (96, 64), (7, 33), (3, 5, 8), (1000, 257), (4, 8192)], ids=str)
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_masks_and_values(gpu, t, shape, p):
    t = TYPES[t]
    gen = torch.Generator().manual_seed(1)
    x, r = (torch.randn(shape, generator=gen).to(t).cuda() for _ in range(2))
    seed, call = 0xFEDCBA9876543210, 2 ** 40 + 17
    out = torch.full_like(x, float("nan"))
    decoder.dropout_(out, x, p, seed, call=call)
    keep, y = want(x, p, seed, call)
    assert torch.equal(out != 0, keep & (x != 0))
    # the factor and the product are rounded to 32 bits, the result to its type
    step = torch.finfo(t).eps / 2 + 2 * 2.0 ** -24
    assert ((out.double() - y).abs() <= step * y.abs() + torch.finfo(t).tiny).all()
    decoder.dropout_(out, x, p, seed, call=torch.tensor([call], device="cuda"), residual=r)
    y = want(x, p, seed, call, r)[1]
    size = y.abs() + x.double().abs() / (1 - p) + r.double().abs()
    assert ((out.double() - y).abs() <= step * y.abs() + 3 * 2.0 ** -24 * size + torch.finfo(t).tiny).all()


@pytest.mark.parametrize("t", TYPES)
def test_strides_do_not_change_the_mask(gpu, t):
    t = TYPES[t]
    for rows, cols, pad in ((50, 24, 8), (50, 24, 1), (33, 12, 4), (20, 7, 2), (3, 3000, 16)):
        x = torch.ones((rows, cols + pad), dtype=t, device="cuda")[:, :cols]
        out = torch.full((rows, cols + pad), 7.0, dtype=t, device="cuda")
        decoder.dropout_(out[:, :cols], x, 0.3, 5)
        assert torch.equal(out[:, :cols], decoder.dropout(x.contiguous(), 0.3, 5))
        assert (out[:, cols:] == 7).all()


def test_edges(gpu):
    x = torch.tensor([float("nan"), float("inf"), -2.0, 1.0], device="cuda").repeat(100)
    assert torch.equal(torch.nan_to_num(decoder.dropout(x, 0.0, 1)), torch.nan_to_num(x))
    assert (decoder.dropout(x, 1.0, 1) == 0).all()
    r = torch.arange(400.0, device="cuda")
    assert torch.equal(decoder.dropout(x, 1.0, 1, residual=r), r)
    y = decoder.dropout(x, 0.5, 1)
    keep = want(x, 0.5, 1, 0)[0]
    assert (y[~keep] == 0).all()   # whatever was dropped
    a = torch.ones(5000, device="cuda")
    masks = [decoder.dropout(a, 0.5, s, call=c) != 0 for s, c in ((1, 0), (1, 1), (2, 0), (2 ** 32 + 1, 0), (1, 2 ** 32))]
    for i in range(5):
        for j in range(i):   # independent masks agree in half of the places, 5 deviations of 35 either way
            assert abs(int((masks[i] == masks[j]).sum()) - 2500) < 180
    for out in (x, r):   # in place
        expected = decoder.dropout(x, 1.0, 9, residual=r)
    decoder.dropout_(r, x, 1.0, 9, residual=r)
    assert torch.equal(r, expected)


def test_replays_take_the_calls_masks(gpu):
    """A captured call reads its number on the device: each replay has the mask that an eager call of its number has."""
    x = torch.randn((64, 100), device="cuda")
    call = torch.zeros(1, dtype=torch.int64, device="cuda")
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        decoder.dropout_(out, x, 0.4, 11, call=call)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decoder.dropout_(out, x, 0.4, 11, call=call)
        call.add_(1)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, decoder.dropout(x, 0.4, 11, call=i)), i


def test_gradient_takes_the_same_mask(gpu):
    x = torch.randn((30, 40), device="cuda", requires_grad=True)
    r = torch.randn((30, 40), device="cuda", requires_grad=True)
    call = torch.tensor([3], device="cuda")
    y = decoder.dropout(x, 0.25, 8, call=call, residual=r)
    call.add_(1)   # (the program goes on before the backward pass)
    dout = torch.randn_like(y)
    y.backward(dout)
    assert torch.equal(x.grad, decoder.dropout(dout, 0.25, 8, call=3)) and torch.equal(r.grad, dout)
