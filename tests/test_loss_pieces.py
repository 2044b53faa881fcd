"""How large a piece of the vocabulary may be, by the workspace it takes, without a GPU: no larger than the kernels' offsets reach,
whatever is asked for."""
from __future__ import annotations

import pytest

from hffn_amd import _lib

F32, BF16 = 0, 1


def loss_bytes(value_type, n, d, vocab, piece):
    return _lib.query_bytes(_lib.load().hffn_loss_workspace, value_type, n, d, vocab, 1, 1, piece)


@pytest.mark.parametrize("value_type,n,rows", [(BF16, 256, 256), (BF16, 1000, 256), (F32, 256, 128), (F32, 300, 128)])
def test_rows_of_a_piece_lie_within_32_bits(value_type, n, rows):
    """A tile of ``rows`` tokens is read by 32-bit byte offsets: its last row starts below 2^32 bytes after the first. Asking for
    more gives the piece, and the workspace, of the largest row that does."""
    vocab, per_row = 1 << 24, (1 << 32) // (rows - 1)
    tokens = -(-n // 256) * 256
    assert loss_bytes(value_type, n, 8, vocab, 1 << 50) <= loss_bytes(value_type, n, 8, vocab, per_row * tokens)


@pytest.mark.parametrize("value_type,size", [(BF16, 2), (F32, 4)])
@pytest.mark.parametrize("n", (1 << 18, (1 << 18) - 1, 100_000))
def test_a_piece_fits_a_launch(value_type, size, n):
    """A launch of below 2^32 threads turns a piece's exponentials into D, 8 entries a thread."""
    assert loss_bytes(value_type, n, 8, 1 << 20, 1 << 50) <= loss_bytes(value_type, n, 8, 1 << 20, (1 << 35) * size)


def test_float32_calls_take_the_packed_weight_and_little_more():
    """x's three parts lie where the packed weight is not read; where the weight is smaller they have their own place."""
    lib, n, d, vocab = _lib.load(), 2048, 1024, 50304
    losses = lambda vocab: _lib.query_bytes(lib.hffn_loss_workspace, F32, n, d, vocab, 1, 0, 0)  # noqa: E731
    assert losses(vocab) < 4 * d * (vocab + n) + 8 * n * (vocab // 32 + 8) + (1 << 20)
    assert losses(1000) > 4 * d * (1000 + n) + 6 * d * n
