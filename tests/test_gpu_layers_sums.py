"""How exact the sums over rows are: bias gradients of linear layers and weight gradients of head norms in float32, as errors
relative to the root of the sum of squares, in 2^-24.

An addition rounds its result by 0.42 of 2^-24 of it (root mean square over a spread-out mantissa). For terms of random
signs the squares of all partial sums add up, relative to the whole's, to (r + 1) / 2 for r terms one after the other and
to 1 for every level of sums by halves."""
import pytest
import torch

from tdgs_amd import decoder

pytestmark = pytest.mark.gpu


def rms(errors):
    return torch.cat(errors).square().mean().sqrt().item() * 2.0 ** 24


@pytest.mark.parametrize("rows", [300, 3000, 20000, 64800])
@pytest.mark.parametrize("n", [1, 3, 8, 17, 64])
def test_bias(gpu, rows, n):
    """Up to eight rows to a thread (4.5), 256 threads by halves (8), up to 254 workgroups, eight to a thread (4.5), and 32 by
    halves (5): 0.42 sqrt(22) = 2.0. A third more for the few values that this is taken over. One after the other, 256
    threads alone make 0.42 sqrt(128) = 4.8."""
    gen = torch.Generator(device="cuda").manual_seed(rows + n)
    errors = []
    for _ in range(-(-128 // n)):
        dout = torch.randn((rows, n), generator=gen, device="cuda")
        db = torch.empty(n, device="cuda")
        decoder.linear_grad_(None, None, db, dout, torch.empty((rows, 4), device="cuda"), torch.empty((4, n), device="cuda"))
        want = dout.double()
        errors.append((db.double() - want.sum(0)) / want.square().sum(0).sqrt())
    assert rms(errors) <= 2.7


@pytest.mark.parametrize("size", [(1, 300, 4, 64), (3, 2501, 8, 64), (1, 64800, 4, 16), (1, 30000, 1, 10), (2, 9000, 4, 128)], ids=str)
def test_head_weights(gpu, size):
    """Up to four rows to a thread (2.5), eight threads to a thread (4.5), those in turn or by halves (5), 1024 workgroups, 32 to a
    thread (16.5), and 32 by halves (5): 0.42 sqrt(33) = 2.4; and each term's own error, of a root and three products
    (0.42 sqrt(4) of the root of their sum of squares): 2.6 together, a fifth more for few values. One after the other, 128 rows
    make 3.4 alone."""
    gen = torch.Generator(device="cuda").manual_seed(sum(size))
    errors = []
    for _ in range(-(-128 // size[-1])):
        q, dout = (torch.randn(size, generator=gen, device="cuda") for _ in range(2))
        dw = torch.empty(size[-1], device="cuda")
        decoder.head_norm_grad_(torch.empty_like(q), None, dw, None, dout, None, q)
        x = q.double()
        terms = dout.double() * x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        errors.append((dw.double() - terms.sum((0, 1, 2))) / terms.square().sum((0, 1, 2)).sqrt())
    assert rms(errors) <= 3.1
