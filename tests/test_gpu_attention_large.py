"""The attention kernels that calls with many results take, against the formulas: 16-bit types with one operand for P and dS,
without a list of keys and with one, rows on 16 bytes and not, every padded head size, several tiles with a tail, the keys
in one part and in several."""
import pytest
import torch

from test_gpu_attention import DTYPES, Case

pytestmark = pytest.mark.gpu

SIZES = [
    # b, kvb, lq, lk, h, hk, d, layout, mask
    (1, 1, 1500, 600, 4, 4, 24, "blhd", "none"),
    (2, 2, 600, 500, 4, 4, 32, "blhd", "none"),
    (1, 1, 600, 700, 4, 4, 64, "blhd", "none"),
    (2, 2, 400, 400, 4, 4, 64, "bhld", "none"),
    (1, 1, 600, 333, 4, 2, 40, "sliced", "none"),
    (1, 1, 600, 700, 4, 2, 80, "blhd", "none"),
    (1, 1, 700, 200, 2, 2, 96, "blhd", "none"),
    (2, 2, 400, 400, 2, 2, 96, "bhld", "none"),
    (2, 2, 500, 300, 3, 3, 128, "blhd", "none"),
    (1, 1, 300, 1100, 2, 1, 128, "sliced", "none"),
    # rows off 16 bytes
    (1, 1, 1200, 600, 4, 4, 32, "odd", "none"),
    (1, 1, 600, 700, 4, 4, 63, "odd", "none"),
    (2, 2, 400, 400, 4, 4, 64, "odd", "none"),
    (2, 2, 300, 300, 2, 2, 90, "odd", "none"),
    (2, 2, 300, 300, 2, 2, 128, "odd", "none"),
    # lists of keys
    (2, 2, 700, 900, 4, 4, 64, "blhd", "both"),
    (2, 2, 1200, 900, 4, 2, 32, "bhld", "keys"),
    (2, 2, 500, 500, 2, 2, 96, "blhd", "keys"),
    (2, 1, 300, 700, 4, 2, 128, "blhd", "lengths"),
    # so many workgroups that each takes all keys, or all rows
    (1, 1, 9000, 130, 16, 16, 32, "blhd", "none"),
    (1, 1, 9000, 200, 16, 16, 64, "blhd", "none"),
    (1, 1, 5000, 150, 16, 16, 96, "blhd", "none"),
    (1, 1, 600, 17000, 4, 4, 32, "blhd", "none"),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=["-".join(map(str, s)) for s in SIZES])
def test_against_formulas(gpu, dtype, size):
    b, kvb, lq, lk, h, hk, d = size[:7]
    assert b * lq * h * d > 1 << 16
    c = Case(dtype, *size, seed=lq + lk)
    c.run()
    c.check()


@pytest.mark.parametrize("rise", [1.0, -1.0], ids=["rising", "falling"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("lq,h,d", [(700, 2, 64), (700, 2, 128), (9000, 16, 32)])
def test_scores_that_rise_along_the_keys(gpu, dtype, rise, lq, h, d):
    """Every tile's largest score is far above (or below) the one before; the last size in one part."""
    lk = 700 if h == 2 else 200
    c = Case(dtype, 1, 1, lq, lk, h, h, d, seed=8)
    along = torch.linspace(0, 1, lk, device="cuda")[None, :, None, None]
    c.q.copy_(c.q.abs() + 0.5)
    c.k.copy_(0.05 * c.k + rise * 8 * along)
    c.run()
    c.check()


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_peaked_rows(gpu, dtype):
    c = Case(dtype, 1, 1, 700, 300, 2, 2, 64, spread=30.0, seed=3)
    c.run(grad=False)
    c.check(grad=False)
