"""``hffn_amd.train_lm``: the head loss, the residual norms and the clipping together with the HFFN layers, against the same
model in float64 with autograd.

Bounds. Every operator's float32 gradient is within 1e-5 of its own formula's in the 2-norm (as their tests hold it); the
model below chains fewer than twenty of them, so the 2-norm of a gradient's error is held to 20 x 1e-5 of the gradient's, and
the gradients' common norm likewise."""
from __future__ import annotations

import json
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from hffn_amd.bench_train import make_cell
from hffn_amd.ffn import hip_layer
from hffn_amd.train_lm import IGNORE, LMTrainer, main

pytestmark = pytest.mark.gpu

BOUND = 20 * 1e-5
CELL, VOCAB = "128_256_d020", 300


def dense(layer):
    """(w_up, b_up, w_down, b_down) float64 and where the support lies."""
    rows = np.repeat(np.arange(layer.d_ff), np.diff(layer.up_offsets)), np.repeat(np.arange(layer.d_ff), np.diff(layer.down_offsets))
    w_up, w_down = torch.zeros(layer.d_ff, layer.d_model, dtype=torch.float64), torch.zeros(layer.d_model, layer.d_ff, dtype=torch.float64)
    w_up[rows[0], layer.up_idx.astype(np.int64)] = torch.from_numpy(layer.up_val).double()
    w_down[layer.down_idx.astype(np.int64), rows[1]] = torch.from_numpy(layer.down_val).double()
    return [t.cuda().requires_grad_() for t in (w_up, torch.from_numpy(layer.b_up).double(), w_down, torch.from_numpy(layer.b_down).double())]


def batch(n, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    ids, labels = (torch.randint(0, VOCAB, (n,), generator=g, device="cuda") for _ in range(2))
    return ids, labels.masked_fill(torch.rand(n, generator=g, device="cuda") < 0.2, IGNORE)


def reference(trainer, layers, ids, labels):
    """(loss, gradients of trainer.parameters() and of the layers' dense weights), float64."""
    params = [p.double().clone().requires_grad_() for p in trainer.parameters()]
    dense_layers = [dense(layer) for layer in layers]
    embedding, head, *norms = params
    x, d = embedding[ids], embedding.shape[1]
    weight, bias, *norms = norms
    h = F.layer_norm(x, (d,), weight, bias, 1e-5)
    for w_up, b_up, w_down, b_down in dense_layers:
        f = F.linear(F.gelu(F.linear(h, w_up, b_up)), w_down, b_down)
        weight, bias, gate, *norms = norms
        x = x + gate * f
        h = F.layer_norm(x, (d,), weight, bias, 1e-5)
    loss = F.cross_entropy(h @ head.T, labels, ignore_index=IGNORE)
    loss.backward()
    return float(loss.detach()), [p.grad for p in params], [[t.grad for t in layer] for layer in dense_layers]


@pytest.mark.parametrize("n", (1, 37, 300))
def test_gradients_of_the_model(n):
    cells = [make_cell(CELL, 7 + i) for i in range(2)]
    trainer = LMTrainer([hip_layer(c) for c in cells], VOCAB, n, seed=3)
    ids, labels = batch(n, n)
    labels[0] = 5  # one counted token at least
    loss, grads, layer_grads = reference(trainer, cells, ids, labels)
    assert abs(float(trainer.backward(ids, labels)) - loss) <= BOUND * abs(loss)
    for k, (got, want) in enumerate(zip(trainer._gradients(), grads)):
        assert float((got.double() - want).norm()) <= BOUND * float(want.norm()), k
    total = sum(float(g.norm()) ** 2 for g in grads)
    for i, (cell, (w_up, b_up, w_down, b_down)) in enumerate(zip(cells, layer_grads)):
        got = trainer.train.gradients(i)
        up_rows = torch.from_numpy(np.repeat(np.arange(cell.d_ff), np.diff(cell.up_offsets))).cuda()
        up = w_up[up_rows, torch.from_numpy(cell.up_idx.astype(np.int64)).cuda()]
        assert float((got["up_val"].double() - up).norm()) <= BOUND * float(up.norm())
        down_rows = np.repeat(np.arange(cell.d_ff), np.diff(cell.down_offsets))
        order = np.lexsort((down_rows, cell.down_idx))  # output-major, as the runtime holds the down values
        down = w_down[torch.from_numpy(cell.down_idx.astype(np.int64)[order]).cuda(), torch.from_numpy(down_rows[order]).cuda()]
        assert float((got["out_val"].double() - down).norm()) <= BOUND * float(down.norm())
        for name, want in (("b_up", b_up), ("b_down", b_down)):
            assert float((got[name].double() - want).norm()) <= BOUND * float(want.norm())
        total += sum(float(t.norm()) ** 2 for t in (up, down, b_up, b_down))
    trainer.max_norm = 0.5 * math.sqrt(total)
    before = [g.clone() for g in trainer.gradients()]
    _, norm = trainer.step(ids, labels)
    assert abs(float(norm) - math.sqrt(total)) <= BOUND * math.sqrt(total)
    for old, new in zip(before, trainer.gradients()):
        assert float((new - 0.5 * old).norm()) <= BOUND * float(old.norm())


def test_training_learns_the_successors():
    """A fixed successor of each of 300 tokens: from ln 300 the loss falls below a fifth of that."""
    trainer = LMTrainer([hip_layer(make_cell(CELL, i)) for i in range(2)], VOCAB, 256, lr=1e-2, seed=1)
    g = torch.Generator("cuda").manual_seed(2)
    successor = torch.randperm(VOCAB, generator=g, device="cuda")
    losses = []
    for _ in range(60):
        ids = torch.randint(0, VOCAB, (256,), generator=g, device="cuda")
        loss, norm = trainer.step(ids, successor[ids])
        assert math.isfinite(float(norm))
        losses.append(float(loss))
    assert abs(losses[0] - math.log(VOCAB)) < 1.0 and losses[-1] < math.log(VOCAB) / 5
    ids = torch.arange(VOCAB, device="cuda")
    assert float(trainer.losses(ids, successor).mean()) < math.log(VOCAB) / 4


def test_command(capsys):
    assert main(["--cell", CELL, "--layers", "1", "--vocab", "500", "--tokens", "33", "--steps", "3"]) == 0
    lines = [json.loads(line) for line in capsys.readouterr().out.splitlines()]
    assert [line["step"] for line in lines] == [0, 1, 2] and all(math.isfinite(line["loss"]) and line["grad_norm"] > 0 for line in lines)


def test_refusals():
    trainer = LMTrainer([hip_layer(make_cell(CELL, 0))], VOCAB)
    ids, labels = batch(4, 1)
    with pytest.raises(ValueError, match="no tokens"):
        trainer.step(ids[:0], labels[:0])
    with pytest.raises(ValueError, match="labels"):
        trainer.step(ids, labels[:3])
