"""``hffn_amd.train_lm``: parameters that AdamW takes in parts are updated as whole ones are; there are no gradients before a backward."""
from __future__ import annotations

import pytest
import torch

from hffn_amd import train_lm
from hffn_amd.bench_train import make_cell
from hffn_amd.ffn import hip_layer

pytestmark = pytest.mark.gpu


def test_adamw_in_parts(monkeypatch):
    ids = torch.arange(50, device="cuda")

    def trained():
        trainer = train_lm.LMTrainer([hip_layer(make_cell("128_256_d020", 5))], 300, 50, seed=2)
        for _ in range(3):
            trainer.step(ids, ids + 7)
        return trainer.parameters()

    whole = trained()
    monkeypatch.setattr(train_lm, "_ADAM_ENTRIES", 100)
    assert all(torch.equal(a, b) for a, b in zip(trained(), whole))


def test_gradients_before_the_first_backward_are_refused():
    trainer = train_lm.LMTrainer([hip_layer(make_cell("128_256_d020", 5))], 300, 50, seed=2)
    ids = torch.arange(50, device="cuda")
    for _ in range(2):
        with pytest.raises(RuntimeError, match="before the first backward"):
            trainer.gradients()
        trainer.losses(ids, ids + 7)
    trainer.backward(ids, ids + 7)
    assert [g.shape for g in trainer.gradients()][:len(trainer.parameters())] == [p.shape for p in trainer.parameters()]
