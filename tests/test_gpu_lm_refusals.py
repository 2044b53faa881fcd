"""Calls of ``LMTrainer`` that mean nothing are refused by the host, before a kernel reads through what they hold."""
from __future__ import annotations

import pytest
import torch

from test_gpu_lm_operators import draw, trainer_of

pytestmark = pytest.mark.gpu

WIDE = torch.iinfo(torch.int64)


@pytest.mark.parametrize("kind", (None, "tied"))
def test_prompts_outside_the_tokens(kind):
    _, trainer = trainer_of(kind)
    ids = draw(50, 1)
    for bounds, match in (([0, 5, 100], "50 tokens"), ([0, 51], "50 tokens"), ([-1, 20, 50], "50 tokens"), ([-50, -1], "50 tokens"), ([0, WIDE.max, WIDE.min, -1, 50], "empty"),
                          ([0, 20, 10, 50], "empty"), ([0, 0, 50], "empty"), ([0], "bounds")):
        for dtype in (torch.int64, torch.int32):
            if dtype == torch.int32 and max(map(abs, bounds)) > 2 ** 31:
                continue
            at = torch.tensor(bounds, dtype=dtype, device="cuda")
            with pytest.raises(ValueError, match=match):
                trainer.generate(ids, torch.zeros(2, len(bounds) - 1, device="cuda"), at, temperature=0.0)
    tokens = trainer.generate(ids, torch.zeros(2, 2, device="cuda"), torch.tensor([3, 20, 50], dtype=torch.int32, device="cuda"), temperature=0.0)
    assert bool(((tokens >= 0) & (tokens < 300)).all())
