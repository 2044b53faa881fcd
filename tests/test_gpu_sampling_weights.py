"""``sample`` where a row's weights come to the most they can: flat rows over large vocabularies, against the definition in float64.

Weights are whole multiples of 2^-b of the largest, b such that V 2^b is at most 2^62 (46 at 50304 entries, 42 at 2^20). Each is off by at
most half of one, the sum of V weights of at least a half by V / 2 of them, so by 2^-42 of itself, which is below what the comparison
of the probabilities allows (2^-24 and 2^-37 of theirs), and a number drawn lies that close to a border of two tokens once in 2^22 rows
of 2^20."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_sampling import BF16, F32, check, draw_logits, draw_uniform

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("vocab", (16383, 16384, 16385, 32768, 50257, 50304, 65536, 151936, 1 << 20))
def test_flat_rows(vocab, dtype):
    """Equal logits, an untrained head's, and a high temperature's: weights of V times the largest in all."""
    n = 2 if vocab < 100000 else 1
    uniform, untrained = draw_uniform(n, vocab), draw_logits(n, vocab, seed=vocab, std=1.0).sub_(draw_logits(n, vocab, seed=vocab, std=0.98)).to(dtype)
    peaked = draw_logits(n, vocab, dtype, seed=vocab)
    for logits, temperature in ((torch.full((n, vocab), 0.25, dtype=dtype, device="cuda"), 1.0), (untrained, 1.0), (peaked, 1e4), (peaked, math.inf)):
        for settings in (dict(), dict(top_p=0.9), dict(top_k=vocab - 5), dict(top_k=vocab // 2, top_p=0.8, min_p=0.001)):
            check(logits, uniform, temperature, **settings)


@pytest.mark.parametrize("dtype", (F32, BF16))
def test_min_p_at_a_zero(dtype):
    """The lowest logit of weight enough is a zero, of either sign: at a temperature that parts a zero from the largest negative number."""
    rows = torch.tensor([[0.0, -1.0, 0.0, -2.0], [-0.0, -1.0, -0.0, -3.0], [-1.0, 0.0, -0.0, -1e-38], [-5.0, -1.0, -1e-30, 0.0]], device="cuda").to(dtype)
    for u in (0.0, 0.4, 0.6, 0.999):
        for temperature in (1e-30, 1e-38):
            for settings in (dict(), dict(top_k=2), dict(top_k=3, top_p=0.9), dict(top_p=0.7)):
                check(rows, torch.full((4,), u, device="cuda"), temperature, min_p=1.0, **settings)
