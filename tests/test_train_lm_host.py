"""``hffn_amd.train_lm`` without a GPU: what the optimizer's launches are told."""
from __future__ import annotations

import pytest
import torch

from hffn_amd import _lib, train_lm


class Recorder:
    """Stands in for the library: notes the entry counts of every AdamW call."""

    def __init__(self):
        self.counts = []

    def hffn_adamw_arrays(self, arrays, p, g, m, v, counts, *rest):
        self.counts += list(counts)
        return _lib.OK


@pytest.mark.parametrize("sizes", [((1 << 32) + 5, 7, 3), (3 << 31, (1 << 32) - 1), (8, 4)])
def test_adamw_reaches_every_entry_of_parameters_of_2_32_entries_and_more(monkeypatch, sizes):
    class Train:
        lr, betas, eps, weight_decay, _lib = 1e-3, (0.9, 0.999), 1e-8, 0.01, Recorder()

    parameters = [torch.empty(size, dtype=torch.float32, device="meta") for size in sizes]
    trainer = object.__new__(train_lm.LMTrainer)
    trainer.train, trainer.steps, trainer._moments, trainer.boundaries, trainer.device = Train(), 0, [], [None], torch.device("cpu")
    monkeypatch.setattr(train_lm.LMTrainer, "parameters", lambda self: parameters)
    monkeypatch.setattr(train_lm.LMTrainer, "_gradients", lambda self: parameters)
    monkeypatch.setattr(train_lm, "current_stream", lambda device: 0)
    trainer._adamw()
    assert sum(Train._lib.counts) == sum(sizes)
