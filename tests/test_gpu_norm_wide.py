"""Group norm with as many groups as channels, and more channels than one workgroup takes: every channel block has
groups of its own."""
import pytest
import torch

from test_gpu_norm import Case

pytestmark = pytest.mark.gpu

SIZES = [
    # dtype, n, pixels, channels (and groups), layout
    (torch.float32, 1, 600, 259, "plain"),      # one element a vector
    (torch.float32, 2, 2100, 1028, "plain"),    # four
    (torch.bfloat16, 1, 2100, 2056, "plain"),   # eight
    (torch.float16, 2, 300, 515, "odd"),
    (torch.float32, 1, 2060, 1600, "plain"),    # more groups than a block has room for
]


@pytest.mark.parametrize("act", ["silu", "identity"])
@pytest.mark.parametrize("size", SIZES, ids=["-".join(map(str, s)) for s in SIZES])
def test_a_group_per_channel(gpu, size, act):
    dtype, n, p, c, layout = size
    case = Case(dtype, n, p, c, c, act, layout)
    case.run()
    case.check()


@pytest.mark.parametrize("size", SIZES, ids=["-".join(map(str, s)) for s in SIZES])
def test_a_group_of_two_channels_is_unchanged(gpu, size):
    """The neighbouring case, whose partial statistics come by channel."""
    dtype, n, p, c, layout = size
    case = Case(dtype, n, p, c + c % 2, (c + c % 2) // 2, "silu", layout)
    case.run()
    case.check()
