"""Calls of ``LMTrainer`` that mean nothing are refused by the host, before a kernel reads through what they hold."""
from __future__ import annotations

import pytest
import torch

from test_gpu_lm_operators import VOCAB, draw, trainer_of

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


@pytest.mark.parametrize("kind", (None, "tied"))
@pytest.mark.parametrize("bad", (VOCAB, -VOCAB - 1, WIDE.max, WIDE.min))
def test_ids_outside_the_table(kind, bad):
    """A step with one is refused and leaves parameters and moments alone, whatever call came before; generating is refused; losses are NaN from there on."""
    _, trainer = trainer_of(kind)
    ids, labels, uniform = draw(50, 1), draw(50, 2), torch.zeros(2, 1, device="cuda")
    trainer.step(ids, labels)
    state = lambda: [t.clone() for t in (*trainer.parameters(), *(m for pair in trainer._moments for m in pair), trainer.train.forward(0, torch.ones(1, 128, device="cuda")))]  # noqa: E731
    before, steps = state(), trainer.steps
    wrong = ids.clone()
    wrong[17] = bad
    for ids_of in ((lambda t: t), (lambda t: t.cpu())):
        for call in (lambda t: trainer.step(t, labels), lambda t: trainer.generate(t, uniform)):
            for _ in range(2):
                with pytest.raises(ValueError, match=f"{VOCAB} rows"):
                    call(ids_of(wrong))
    assert trainer.steps == steps and all(torch.equal(a, b) for a, b in zip(state(), before))
    losses = trainer.losses(wrong, labels).isfinite()
    assert not losses[17] and (losses.sum() == (49 if kind is None else 17))
    with pytest.raises(ValueError, match=f"{VOCAB} rows"):
        trainer.losses(wrong.cpu(), labels)
    with pytest.raises(ValueError):  # the lookup has run, nobody has asked about its ids
        trainer.step(wrong, labels[:3])
    loss, norm = trainer.step(ids, labels)
    assert bool(loss.isfinite()) and bool(norm.isfinite()) and trainer.steps == steps + 1
    trainer.step(ids.clamp(max=VOCAB - 1) - VOCAB, labels)
    assert all(bool(t.isfinite().all()) for t in trainer.parameters())
