"""Dropout's generator against its published vectors, its masks at the ends of seed and call, and dropout in place against the
call with a result of its own."""
import numpy as np
import pytest
import torch

from tdgs_amd import decoder

LOW, BY = np.uint64(2 ** 32 - 1), np.uint64(32)


def philox(counter, key):
    """Philox4x32-10 of arrays of four 32-bit counter words and two key words."""
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    for r in range(10):
        k = [np.uint64((key[0] + 0x9E3779B9 * r) & 0xFFFFFFFF), np.uint64((key[1] + 0xBB67AE85 * r) & 0xFFFFFFFF)]
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> BY) ^ c[1] ^ k[0], b & LOW, (a >> BY) ^ c[3] ^ k[1], a & LOW]
    return c


def test_published_vectors():
    """Counter and key of zeros, of ones, and of the digits of pi (Salmon, Moraes, Dror & Shaw 2011)."""
    ones = 0xFFFFFFFF
    for counter, key, want in (
            ((0,) * 4, (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
            ((ones,) * 4, (ones, ones), (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
            ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0), (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
        assert tuple(int(w) for w in philox(counter, key)) == want


def kept(n, p, seed, call):
    i = np.arange((n + 3) // 4, dtype=np.uint64)
    words = philox((i & LOW, i >> BY, np.full_like(i, call & 0xFFFFFFFF), np.full_like(i, call >> 32)), (seed & 0xFFFFFFFF, seed >> 32))
    return torch.from_numpy(np.stack(words, 1).reshape(-1)[:n] >= np.uint64(int(p * 2.0 ** 32))).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [0, 2 ** 32 - 1, 2 ** 32, 2 ** 64 - 1])
@pytest.mark.parametrize("call", [0, 2 ** 32 - 1, 2 ** 63, 2 ** 64 - 1])
def test_ends_of_seed_and_call(gpu, seed, call):
    x = torch.ones(4099, device="cuda")
    want = kept(4099, 0.3, seed, call)
    assert torch.equal(decoder.dropout(x, 0.3, seed, call=call) != 0, want)
    signed = call - 2 ** 64 if call >= 2 ** 63 else call
    assert torch.equal(decoder.dropout(x, 0.3, seed, call=torch.tensor([signed], device="cuda")) != 0, want)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad", [0, 8], ids=["dense", "padded"])
@pytest.mark.parametrize("shape", [(1, 5), (33, 7), (33, 12), (33, 64), (300, 1024), (7, 3001)], ids=str)
def test_in_place(gpu, t, pad, shape):
    """By single elements (rows apart whose columns do not divide by four), vectors of four and of eight."""
    gen = torch.Generator().manual_seed(2)

    def rows():
        return torch.randn((shape[0], shape[1] + pad), generator=gen).to(t).cuda()[:, :shape[1]]

    x, r = rows(), rows()
    mask = kept(x.numel(), 0.4, 9, 6).reshape(shape)
    want = decoder.dropout_(torch.full(shape, float("nan"), dtype=t, device="cuda"), x, 0.4, 9, call=6, residual=r)
    # factor and product rounded to 32 bits, the sum once more and to its type
    y = torch.where(mask, x.double() / 0.6, 0) + r.double()
    size = y.abs() + x.double().abs() / 0.6 + r.double().abs()
    assert ((want.double() - y).abs() <= torch.finfo(t).eps / 2 * y.abs() + 3 * 2.0 ** -24 * size + torch.finfo(t).tiny).all()
    alone = decoder.dropout_(torch.full(shape, float("nan"), dtype=t, device="cuda"), x, 0.4, 9, call=6)
    for name in ("x", "residual", "x alone", "both"):
        a, b = (v.clone() if pad == 0 else torch.empty_strided(v.shape, v.stride(), dtype=t, device="cuda").copy_(v) for v in (x, r))
        out = b if name == "residual" else a
        if name == "both":
            b = a
        decoder.dropout_(out, a, 0.4, 9, call=6, residual=None if name == "x alone" else b)
        if name == "both":
            assert torch.equal(out, decoder.dropout_(torch.empty_like(alone), x, 0.4, 9, call=6, residual=x))
        else:
            assert torch.equal(out, alone if name == "x alone" else want), name
            assert torch.equal(a if name == "residual" else b, x if name == "residual" else r)
    assert not torch.equal(want, r)


@pytest.mark.gpu
def test_replays_take_the_calls_masks(gpu):
    """Captured on inputs that the capture's stream has waited for: each replay has the mask that an eager call of its number has."""
    x = torch.randn((64, 100), device="cuda")
    call = torch.zeros(1, dtype=torch.int64, device="cuda")
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decoder.dropout_(out, x, 0.4, 11, call=call)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decoder.dropout_(out, x, 0.4, 11, call=call)
        call.add_(1)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, decoder.dropout(x, 0.4, 11, call=i)), i
