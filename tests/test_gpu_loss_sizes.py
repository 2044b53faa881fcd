"""``HeadLoss`` at sizes where its kernels take other ways than at those of ``test_gpu_loss``, whose oracle and bounds these tests
share."""
from __future__ import annotations

import math

import pytest
import torch

from hffn_amd.loss import HeadLoss

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("n,dtype", [(256, BF16), (128, F32)])
def test_a_piece_whose_rows_pass_32_bits(n, dtype):
    """8.5 million vocabulary rows asked for as one piece: the last tokens of a tile lie 4 GB after its first.

    gx against float64 at tokens at both ends of the tile. Its sum over the vocabulary is taken in 64 parts or more, so that
    (beside test_gpu_loss's terms) 2^-23 of vocab / 64 terms' magnitudes bound it."""
    vocab, d = 8_500_001, 16
    g = torch.Generator("cuda").manual_seed(n)
    x = torch.randn(n, d, generator=g, dtype=F32, device="cuda").to(dtype)
    weight = (torch.randn(vocab, d, generator=g, dtype=F32, device="cuda") / math.sqrt(d)).to(dtype)
    labels = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    head = HeadLoss(weight, piece_bytes=16 << 30)
    _, gx, gw = head.step(x, labels)
    rounding = 2.0 ** -8 if dtype == BF16 else 0.0
    rows, w = x.double(), weight.double()
    lse = torch.stack([torch.logsumexp(rows @ part.T, 1) for part in w.split(1 << 19)]).logsumexp(0)
    e = d * 2.0 ** -23 * max(float((rows.abs() @ part.abs().T).max()) for part in w.split(1 << 19))

    def within(got, want, size, terms):
        bound = (2 * e + 2.0 ** -19 + rounding + terms * 2.0 ** -23) * (1 + rounding) * size + (rounding + 2.0 ** -24) * want.abs()
        return bool(((got.double() - want).abs() <= bound).all())

    for t in (0, 1, n // 2 - 1, n // 2, n - 2, n - 1):
        D = torch.exp(w @ rows[t] - lse[t])
        D[labels[t]] -= 1.0
        D /= n
        assert within(gx[t], D @ w, D.abs() @ w.abs(), vocab / 64), t
    at = torch.cat([labels, torch.arange(0, vocab, 9973, device="cuda"), torch.tensor([vocab - 1], device="cuda")])
    D = (torch.exp(rows @ w[at].T - lse[:, None]) - (labels[:, None] == at).double()) / n
    assert within(gw[at], D.T @ rows, D.abs().T @ rows.abs(), n)
