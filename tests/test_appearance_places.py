"""The patches' positions of the appearance decoder belong to the call that makes them: a tensor kept for later calls would be
read on streams, and before replays, that do not wait for what fills it."""
import pytest
import torch

from tdgs_amd import appearance, decoder


@pytest.mark.parametrize("size", [(1, 1), (3, 5), (7, 2)])
def test_made_in_every_call(size):
    dec = object.__new__(appearance.AppearanceDecoder)   # (without a GPU)
    dec.device, dec._places = torch.device("cpu"), {}
    first, second = dec._patch_places(*size), dec._patch_places(*size)
    assert first.data_ptr() != second.data_ptr() and not dec._places
    assert first.dtype is torch.int32 and first.is_contiguous()
    assert torch.equal(first, torch.cartesian_prod(*(torch.arange(n, dtype=torch.int32) for n in size)).reshape(-1, 2))
    assert torch.equal(first, second)


@pytest.mark.gpu
def test_first_use_of_a_size_in_a_graph(gpu):
    """Positions and rotation captured before any eager call of the size: eager calls before the first replay, and replays
    between them."""
    dec, other = (appearance.AppearanceDecoder(2, channels=32, heads=2, groups=4, rotary=True, seed=1) for _ in range(2))
    gen = torch.Generator().manual_seed(2)
    rgb, q = torch.rand((30, 26, 3), generator=gen).cuda(), torch.randn((1, 8 * 7, 2, 16), generator=gen).cuda()

    def turned(d):
        return decoder.head_norm(q, None, d.parameters["query_norm"], rotary=d.rotary, positions=d._patch_places(8, 7))

    with torch.no_grad():
        want, want_q = other(rgb, 1), turned(other)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = turned(dec)
        assert torch.equal(dec(rgb, 1), want) and torch.equal(turned(dec), want_q)
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want_q)
            assert torch.equal(dec(rgb, 1), want)


@pytest.mark.gpu
def test_two_streams(gpu):
    dec = appearance.AppearanceDecoder(2, channels=32, heads=2, groups=4, rotary=True, seed=1)
    rgb = torch.rand((201, 130, 3), generator=torch.Generator().manual_seed(2)).cuda()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    with torch.no_grad():
        for stream in streams:
            with torch.cuda.stream(stream):
                outs.append(dec(rgb, 1))
        torch.cuda.synchronize()
        want = dec(rgb, 1)
    assert all(torch.equal(o, want) for o in outs)
