"""The token that gives no gradient is a row of the table: other numbers are refused, not ignored (without a GPU)."""
import pytest
import torch

from tdgs_amd import abi, decoder
from test_decoder_abi import lib  # noqa: F401


@pytest.mark.parametrize("padding", [-2, 50, 1 << 40, -(1 << 40)])
def test_the_call_refuses(lib, padding):  # noqa: F811
    assert lib.tdgs_embedding_grad(64, None, 0, 64, 8, 64, 4, 100000, padding, 1.0, 64, 8, 50, 8, 64, 16) == abi.TDGS_ERR_INVALID
    assert b"padding" in lib.tdgs_last_error()


@pytest.mark.parametrize("padding", [-1, -2, 7])
def test_the_differentiable_function_refuses(padding):
    """-1 too, which is the last row to torch's own embedding."""
    with pytest.raises(ValueError, match="padding"):
        decoder.embedding(torch.zeros((7, 3)), torch.zeros(2, dtype=torch.long), padding=padding)
