"""A small language model around the HFFN layers, trained on the device: an embedding, a residual stack whose blocks are HFFN
layers and whose boundaries are ``ResidualNorm``s, a head whose loss and gradients come from ``HeadLoss``, and a step that
clips the gradients of all of them together (``clip_grad_norm_``) before AdamW.

    x = embedding[ids];  (x, h_0) = boundary_0(x);  f_i = layer_i(h_i);  (x, h_i+1) = boundary_i+1(x, f_i);  loss(h_L)

    python -m hffn_amd.train_lm [--cell 512_2048_d020] [--layers 2] [--vocab 50304] [--tokens 512] [--steps 20]

The command trains on a synthetic language, each token's successor fixed by a random permutation, a tenth of the positions
masked out of the loss, and prints one JSON line per step: loss, gradient norm before clipping and milliseconds.
Embedding, head, norms and gates are float32, drawn at random; layers are ``bench_train``'s synthetic cells.
"""
from __future__ import annotations

import argparse
import ctypes
import json
import math
import time

import torch

from . import _lib
from .bench_train import make_cell
from .clip import clip_grad_norm_
from .ffn import hip_layer
from .loss import HeadLoss
from .norm import ResidualNorm
from .runtime import HFFNLayer, HFFNRuntime, current_stream, leading_dim
from .train_runtime import HFFNTrainRuntime

IGNORE = -100
_ADAM_ARRAYS = 4  # arrays of one AdamW launch
_ADAM_ENTRIES = 1 << 30  # of one of them: the library counts in 32 bits


class LMTrainer:
    """The model above and its step. ``boundaries`` has one more entry than there are layers; the first is a norm alone, the others
    have a gate, a vector that starts at ``1 / sqrt(layers)``. Calls of one trainer belong on one stream."""

    def __init__(self, layers: list[HFFNLayer], vocab: int, max_tokens: int = 1, max_norm: float = 1.0, lr: float = 1e-3,
                 betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, seed: int = 0) -> None:
        self.train = HFFNTrainRuntime(HFFNRuntime(layers, "cuda"), lr, betas, eps, weight_decay, max_tokens)
        device, d = self.train.runtime.device, self.train.d_model
        self.device, self.max_norm, self.steps = device, float(max_norm), 0
        g = torch.Generator(device).manual_seed(seed)
        self.embedding = torch.randn(vocab, d, generator=g, dtype=torch.float32, device=device)
        self.head = HeadLoss(torch.randn(vocab, d, generator=g, dtype=torch.float32, device=device) / math.sqrt(d), max_tokens, IGNORE)
        vector = lambda value: torch.full((d,), value, dtype=torch.float32, device=device)  # noqa: E731
        self.boundaries = [ResidualNorm(vector(1.0), vector(0.0), gate=vector(1.0 / math.sqrt(len(layers))) if i else None)
                           for i in range(len(layers) + 1)]
        self._embedding_grad = torch.zeros_like(self.embedding)
        self._moments: list[tuple[torch.Tensor, torch.Tensor]] = []
        self._z: torch.Tensor | None = None

    def parameters(self) -> list[torch.Tensor]:
        """Embedding, head, boundaries: what AdamW updates beside the layers."""
        return [self.embedding, self.head.weight, *(t for b in self.boundaries for t in b.parameters().values())]

    def _gradients(self) -> list[torch.Tensor]:
        return [self._embedding_grad, self.head.grad, *(t for b in self.boundaries for t in b.gradients().values())]

    def gradients(self) -> list[torch.Tensor]:
        """Of ``parameters()``, then of every layer, by the last ``backward``. Raises ``RuntimeError`` before the first."""
        if self.head.grad is None:
            raise RuntimeError("no gradients before the first backward")
        layers = range(len(self.boundaries) - 1)
        return self._gradients() + [t for i in layers for t in self.train.gradients(i).values()]

    def forward(self, ids: torch.Tensor) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
        """The boundaries' (r, h), first to last, of tokens ids [N]."""
        r, h = self.boundaries[0].forward(self.embedding[ids])
        rs, hs = [r], [h]
        for i, boundary in enumerate(self.boundaries[1:]):
            r, h = boundary.forward(r, self.train.forward(i, h))
            rs.append(r)
            hs.append(h)
        return rs, hs

    def losses(self, ids: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        """float32 [N], of the labels given the tokens; a view that the next call overwrites."""
        return self.head.losses(self.forward(ids)[1][-1], labels)

    def backward(self, ids: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        """The mean loss (0-d, a view that the next call overwrites), with all gradients of it computed. A layer runs again with
        its pre-activations kept where its turn comes, so one layer's are in memory at a time."""
        n = ids.shape[0]
        if n == 0:
            raise ValueError("no tokens")
        entries = self.train.d_ff * leading_dim(n)
        if self._z is None or self._z.numel() < entries:
            self._z = torch.empty(entries, dtype=torch.float32, device=self.device)
        rs, hs = self.forward(ids)
        loss, gh, _ = self.head.step(hs[-1], labels)
        gr = None
        for i in reversed(range(len(self.boundaries) - 1)):
            f = self.train.forward(i, hs[i], self._z)
            gr, gf = self.boundaries[i + 1].backward(rs[i + 1], f, gr, gh)
            gh = self.train.backward(i, gf)
        gr, _ = self.boundaries[0].backward(rs[0], None, gr, gh)
        self._embedding_grad.zero_().index_put_((ids,), gr, accumulate=True)
        return loss

    def _adamw(self) -> None:
        train, (beta1, beta2) = self.train, self.train.betas
        parameters, gradients = self.parameters(), self._gradients()
        if not self._moments:
            self._moments = [(torch.zeros_like(p), torch.zeros_like(p)) for p in parameters]
        self.steps += 1
        scalars = (train.lr * train.weight_decay, beta1, 1.0 - beta1, beta2, 1.0 - beta2, train.lr / (1.0 - beta1 ** self.steps),
                   math.sqrt(1.0 - beta2 ** self.steps), train.eps)
        parts = [part for row in zip(parameters, gradients, *zip(*self._moments)) for part in zip(*(t.view(-1).split(_ADAM_ENTRIES) for t in row))]
        for first in range(0, len(parts), _ADAM_ARRAYS):
            rows = parts[first:first + _ADAM_ARRAYS]
            pointers = [(ctypes.c_void_p * len(rows))(*(t.data_ptr() for t in column)) for column in zip(*rows)]
            counts = (ctypes.c_uint32 * len(rows))(*(row[0].numel() for row in rows))
            _lib.check(train._lib.hffn_adamw_arrays(len(rows), *pointers, counts, *scalars, current_stream(self.device)), "AdamW")
        for i in range(len(self.boundaries) - 1):
            train.adamw(i)

    def step(self, ids: torch.Tensor, labels: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(loss, gradient norm before clipping), both 0-d on the device: gradients, clipping over all of them, AdamW."""
        loss = self.backward(ids, labels)
        norm = clip_grad_norm_(self.gradients(), self.max_norm)
        self._adamw()
        return loss, norm


def synthetic_batch(vocab: int, n: int, device, generator: torch.Generator, successor: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Uniform tokens and their successors, a tenth of them masked out."""
    ids = torch.randint(0, vocab, (n,), generator=generator, device=device)
    masked = torch.rand(n, generator=generator, device=device) < 0.1
    return ids, successor[ids].masked_fill(masked, IGNORE)


def main(argv: list[str] | None = None) -> int:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--cell", default="512_2048_d020", help="<d_model>_<d_ff>_d<density percent> of the layers")
    parser.add_argument("--layers", type=int, default=2)
    parser.add_argument("--vocab", type=int, default=50304)
    parser.add_argument("--tokens", type=int, default=512)
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--lr", type=float, default=1e-3)
    parser.add_argument("--max-norm", type=float, default=1.0)
    parser.add_argument("--seed", type=int, default=0)
    args = parser.parse_args(argv)
    layers = [hip_layer(make_cell(args.cell, args.seed + i)) for i in range(args.layers)]
    trainer = LMTrainer(layers, args.vocab, args.tokens, args.max_norm, args.lr, seed=args.seed)
    g = torch.Generator(trainer.device).manual_seed(args.seed + 1)
    successor = torch.randperm(args.vocab, generator=g, device=trainer.device)
    for k in range(args.steps):
        ids, labels = synthetic_batch(args.vocab, args.tokens, trainer.device, g, successor)
        torch.cuda.synchronize()
        start = time.perf_counter()
        loss, norm = trainer.step(ids, labels)
        torch.cuda.synchronize()
        print(json.dumps({"step": k, "loss": round(float(loss), 5), "grad_norm": round(float(norm), 5),
                          "ms": round((time.perf_counter() - start) * 1e3, 3)}), flush=True)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
