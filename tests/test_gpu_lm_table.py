"""Another table assigned to an ``LMTrainer``: what its gradients and moments are then, and which tables are refused."""
from __future__ import annotations

import pytest
import torch

from test_gpu_lm_operators import VOCAB, draw, trainer_of

pytestmark = pytest.mark.gpu


def table(rows, width=128):
    return torch.randn(rows, width, generator=torch.Generator("cuda").manual_seed(rows), dtype=torch.float32, device="cuda")


def test_gradients_stay_until_the_next_backward():
    _, trainer = trainer_of("tied")
    ids, labels = draw(50, 1), draw(50, 2)
    trainer.step(ids, labels)
    before = [t.clone() for t in trainer.gradients()]
    trainer.embedding = table(VOCAB)
    after = trainer.gradients()
    assert len(after) == len(before) and all(torch.equal(a, b) for a, b in zip(after, before))
    assert [t.shape for t in after[:len(trainer.parameters())]] == [t.shape for t in trainer.parameters()]
    trainer.backward(ids, labels)
    assert not torch.equal(trainer.gradients()[0], before[0])
    trainer.step(ids, labels)


def test_another_vocabulary():
    _, trainer = trainer_of(None)
    ids, labels = draw(50, 1), draw(50, 2)
    trainer.backward(ids, labels)
    trainer.embedding = wider = table(VOCAB + 100)
    with pytest.raises(RuntimeError, match="before the first"):
        trainer.gradients()
    ids[7] = VOCAB + 99
    assert torch.equal(trainer.forward(ids)[0][0], wider[ids])
    trainer.step(ids, labels)
    assert [t.shape for t in trainer.gradients()[:2]] == [t.shape for t in trainer.parameters()[:2]]
    kept = trainer.embedding
    for other in (table(VOCAB), table(VOCAB + 101)):
        with pytest.raises(ValueError, match="moments"):
            trainer.embedding = other
    assert trainer.embedding is kept


def test_a_table_that_is_not_contiguous():
    _, trainer = trainer_of(None)
    ids = draw(50, 1)
    view = table(128, VOCAB).T
    trainer.embedding = view
    assert torch.equal(trainer.forward(ids)[0][0], view[ids])
    trainer.step(ids, draw(50, 2))
    assert not torch.equal(trainer.embedding, view)


def test_tables_that_are_refused():
    _, trainer = trainer_of(None)
    kept = trainer.embedding
    for bad in (table(VOCAB).bfloat16(), table(VOCAB).double(), table(VOCAB, 127), table(VOCAB)[0], table(VOCAB).cpu(), table(VOCAB)[:0]):
        with pytest.raises(ValueError):
            trainer.embedding = bad
    assert trainer.embedding is kept
