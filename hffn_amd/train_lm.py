"""A small language model around the HFFN layers, trained on the device: an embedding (``TokenEmbedding``), a residual stack whose
blocks are HFFN layers and whose boundaries are ``ResidualNorm``s, a head whose loss and gradients come from ``HeadLoss``, and a
step that clips the gradients of all of them together (``clip_grad_norm_``) before AdamW.

    x = embedding[ids];  (x, h_0) = boundary_0(x);  f_i = layer_i(h_i);  (x, h_i+1) = boundary_i+1(x, f_i);  loss(h_L)

With ``mixing`` a ``GatedRecurrence`` of that kind stands before every layer and lets tokens know of those before them in their
sequence: ``f_i = layer_i(mixer_i(h_i, h_i G_i^T))``, G_i a [d, d] matrix. ``generate`` goes on from prompts, one token of each
sequence at a time, drawn by ``sample``.

    python -m hffn_amd.train_lm [--cell 512_2048_d020] [--layers 2] [--vocab 50304] [--tokens 512] [--steps 20]
                                [--mixing tied] [--sequences 4] [--generate 16]

The command trains on a synthetic language, each token's successor fixed by a random permutation (with ``--mixing``, the successor
of the token before it), a tenth of the positions masked out of the loss, and prints one JSON line per step: loss, gradient norm
before clipping and milliseconds; then, with ``--generate``, one with the tokens that follow a prompt.
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
from .embedding import TokenEmbedding
from .ffn import hip_layer
from .loss import HeadLoss
from .norm import ResidualNorm
from .recurrence import KINDS, GatedRecurrence
from .runtime import HFFNLayer, HFFNRuntime, current_stream, leading_dim
from .sampling import sample
from .train_runtime import HFFNTrainRuntime

IGNORE = -100
_ADAM_ARRAYS = 4  # arrays of one AdamW launch
_ADAM_ENTRIES = 1 << 30  # of one of them: the library counts in 32 bits


class LMTrainer:
    """The model above and its step. ``boundaries`` has one more entry than there are layers; the first is a norm alone, the others
    have a gate, a vector that starts at ``1 / sqrt(layers)``. ``mixing`` (a kind of ``GatedRecurrence``; ``None``: tokens know of
    no others): ``gates`` and ``mixers`` have one entry per layer, the mixers' biases spread over -5 to 1. Ids count from the
    table's end where they are negative, as tensors are indexed; of those beyond it ``step`` and ``generate``, and on the host every call, raise
    ``ValueError``, the other calls give NaN. Calls of one trainer belong on one stream."""

    def __init__(self, layers: list[HFFNLayer], vocab: int, max_tokens: int = 1, max_norm: float = 1.0, lr: float = 1e-3,
                 betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, seed: int = 0,
                 mixing: str | None = None) -> None:
        self.train = HFFNTrainRuntime(HFFNRuntime(layers, "cuda"), lr, betas, eps, weight_decay, max_tokens)
        device, d = self.train.runtime.device, self.train.d_model
        self.device, self.max_norm, self.steps = device, float(max_norm), 0
        self._moments: list[tuple[torch.Tensor, torch.Tensor]] = []
        g = torch.Generator(device).manual_seed(seed)
        self.embedding = torch.randn(vocab, d, generator=g, dtype=torch.float32, device=device)
        self.head = HeadLoss(torch.randn(vocab, d, generator=g, dtype=torch.float32, device=device) / math.sqrt(d), max_tokens, IGNORE)
        vector = lambda value: torch.full((d,), value, dtype=torch.float32, device=device)  # noqa: E731
        self.boundaries = [ResidualNorm(vector(1.0), vector(0.0), gate=vector(1.0 / math.sqrt(len(layers))) if i else None)
                           for i in range(len(layers) + 1)]
        self.gates: list[torch.Tensor] = []
        self.mixers: list[GatedRecurrence] = []
        for _ in layers if mixing is not None else ():
            self.gates.append(torch.randn(d, d, generator=g, dtype=torch.float32, device=device) / math.sqrt(d))
            self.mixers.append(GatedRecurrence(torch.linspace(-5.0, 1.0, d, dtype=torch.float32, device=device), mixing))
        self._gate_grads = [torch.empty_like(t) for t in self.gates]
        self._z: torch.Tensor | None = None
        self._outside = torch.zeros(1, dtype=torch.int32, device=device)  # 1: an id had no row
        self._outside_host = torch.zeros(1, dtype=torch.int32, pin_memory=True)
        self._looked_up, self._unchecked = torch.cuda.Event(), False

    @property
    def embedding(self) -> torch.Tensor:
        """float32 [vocab, d], contiguous. Another may be assigned (a copy is taken where it is not contiguous): gradients and AdamW's
        moments stay as they are; one of another vocabulary has no gradients before its first ``backward``, and comes before the first
        ``step``, which makes the moments."""
        return self._table.weight

    @embedding.setter
    def embedding(self, weight: torch.Tensor) -> None:
        old = self.__dict__.get("_table")
        d = self.train.d_model
        if weight.dim() != 2 or weight.shape[1] != d or weight.dtype != torch.float32:
            raise ValueError(f"embedding: a float32 [vocab, {d}] tensor is required, not {weight.dtype} {list(weight.shape)}")
        same = old is not None and weight.shape == old.weight.shape
        if self._moments and not same:
            raise ValueError(f"embedding: a vocabulary of {weight.shape[0]} for AdamW's moments of {old.weight.shape[0]}")
        self._table = TokenEmbedding(weight.detach().contiguous())
        if same:
            self._table.grad = old.grad

    def parameters(self) -> list[torch.Tensor]:
        """Embedding, head, boundaries, with mixing the gates' matrices and the mixers' biases: what AdamW updates beside the layers."""
        return [self.embedding, self.head.weight, *(t for b in self.boundaries for t in b.parameters().values()), *self.gates,
                *(t for m in self.mixers for t in m.parameters().values())]

    def _gradients(self) -> list[torch.Tensor]:
        return [self._table.grad, self.head.grad, *(t for b in self.boundaries for t in b.gradients().values()), *self._gate_grads,
                *(t for m in self.mixers for t in m.gradients().values())]

    def gradients(self) -> list[torch.Tensor]:
        """Of ``parameters()``, then of every layer, by the last ``backward``. Raises ``RuntimeError`` before the first
        (of the table that is assigned, where its vocabulary is another)."""
        if self.head.grad is None or self._table.grad is None:
            raise RuntimeError("no gradients before the first backward")
        layers = range(len(self.boundaries) - 1)
        return self._gradients() + [t for i in layers for t in self.train.gradients(i).values()]

    def _tokens(self, ids: torch.Tensor) -> torch.Tensor:
        """Ids on the device; those on the host are checked there."""
        if ids.device.type == "cpu" and ids.numel():
            low, high = (int(v) for v in ids.aminmax())
            vocab = self._table.vocab
            if low < -vocab or high >= vocab:
                raise ValueError(f"ids from {low} to {high} outside the table's {vocab} rows")
        return ids.to(self.device)

    def _check_tokens(self) -> None:
        """Raises ``ValueError`` if an id of the last guarded ``_walk`` had no row. Waits for that lookup alone."""
        self._looked_up.synchronize()
        self._unchecked = bool(self._outside_host[0])
        if self._unchecked:
            raise ValueError(f"ids outside the table's {self._table.vocab} rows")

    def _mixed(self, i: int, h: torch.Tensor, mix) -> tuple[torch.Tensor, torch.Tensor | None]:
        """(what layer i reads, its gates) of hidden rows h; ``mix(i, h, gates)`` runs the mixer."""
        if not self.mixers:
            return h, None
        gates = h @ self.gates[i].T
        return mix(i, h, gates), gates

    def _walk(self, ids: torch.Tensor, mix, guarded: bool = False, from_end: bool = True) -> tuple[list, list, list, list]:
        """The boundaries' (r, h), first to last, of tokens ids [N], and the layers' inputs and gates. ``guarded``: ``_check_tokens`` follows."""
        if guarded and self._unchecked:  # the word may still be that of an earlier call
            self._outside.zero_()
        x = self._table.forward(ids, from_end=from_end, outside=self._outside if guarded else None)
        if guarded:
            self._unchecked = True
            self._outside_host.copy_(self._outside, non_blocking=True)
            self._looked_up.record()
        r, h = self.boundaries[0].forward(x)
        rs, hs, ms, gates = [r], [h], [], []
        for i, boundary in enumerate(self.boundaries[1:]):
            m, gate = self._mixed(i, h, mix)
            r, h = boundary.forward(r, self.train.forward(i, m))
            for kept, t in ((rs, r), (hs, h), (ms, m), (gates, gate)):
                kept.append(t)
        return rs, hs, ms, gates

    def _sequences(self, bounds: torch.Tensor | None, states: list[torch.Tensor] | None = None):
        """The mixers' run over sequences; ``states`` gets each layer's states behind them."""
        def mix(i: int, h: torch.Tensor, gates: torch.Tensor) -> torch.Tensor:
            m, last = self.mixers[i].forward(h, gates, bounds)
            if states is not None:
                states.append(last)
            return m
        return mix

    def forward(self, ids: torch.Tensor, bounds: torch.Tensor | None = None) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
        """The boundaries' (r, h), first to last, of tokens ids [N]; ``bounds`` [S + 1]: where the sequences that mixing knows of
        begin, and where the last ends (``None``: one sequence)."""
        return self._walk(self._tokens(ids), self._sequences(bounds))[:2]

    def losses(self, ids: torch.Tensor, labels: torch.Tensor, bounds: torch.Tensor | None = None) -> torch.Tensor:
        """float32 [N], of the labels given the tokens; a view that the next call overwrites."""
        return self.head.losses(self.forward(ids, bounds)[1][-1], labels)

    def backward(self, ids: torch.Tensor, labels: torch.Tensor, bounds: torch.Tensor | None = None) -> torch.Tensor:
        """The mean loss (0-d, a view that the next call overwrites), with all gradients of it computed. A layer runs again with
        its pre-activations kept where its turn comes, so one layer's are in memory at a time."""
        return self._backward(ids, labels, bounds, False)

    def _backward(self, ids: torch.Tensor, labels: torch.Tensor, bounds: torch.Tensor | None, guarded: bool) -> torch.Tensor:
        ids, n = self._tokens(ids), ids.shape[0]
        if n == 0:
            raise ValueError("no tokens")
        entries = self.train.d_ff * leading_dim(n)
        if self._z is None or self._z.numel() < entries:
            self._z = torch.empty(entries, dtype=torch.float32, device=self.device)
        rs, hs, ms, gates = self._walk(ids, self._sequences(bounds), guarded)
        loss, gh, _ = self.head.step(hs[-1], labels)
        gr = None
        for i in reversed(range(len(self.boundaries) - 1)):
            f = self.train.forward(i, ms[i], self._z)
            gr, gf = self.boundaries[i + 1].backward(rs[i + 1], f, gr, gh)
            gh = self.train.backward(i, gf)
            if self.mixers:
                gx, ggate, _ = self.mixers[i].backward(hs[i], gates[i], ms[i], gh, bounds)
                torch.mm(ggate.T, hs[i], out=self._gate_grads[i])
                gh = torch.addmm(gx, ggate, self.gates[i])
        gr, _ = self.boundaries[0].backward(rs[0], None, gr, gh)
        self._table.backward(ids, gr, from_end=True)
        return loss

    @torch.no_grad()
    def generate(self, ids: torch.Tensor, uniform: torch.Tensor, bounds: torch.Tensor | None = None, **settings) -> torch.Tensor:
        """int64 [K, S]: the tokens that follow each of the S prompts laid end to end in ids [N] (``bounds`` as in ``forward``, all of it in
        [0, N]; no prompt may be empty), drawn with the numbers ``uniform``, float32 [K, S]; ``settings`` are ``sample``'s."""
        if bounds is not None and (bounds.dim() != 1 or bounds.shape[0] < 2):
            raise ValueError(f"bounds: an [S + 1] tensor is required, not {list(bounds.shape)}")
        sequences = 1 if bounds is None else bounds.shape[0] - 1
        if uniform.dim() != 2 or uniform.shape[1] != sequences:
            raise ValueError(f"uniform: a [K, {sequences}] tensor is required, not {list(uniform.shape)}")
        if ids.shape[0] == 0:
            raise ValueError("an empty prompt")
        if bounds is not None:
            empty, begin, end = torch.stack([(bounds[1:] <= bounds[:-1]).any().long(), bounds[0].long(), bounds[-1].long()]).tolist()
            if empty:
                raise ValueError("an empty prompt")
            if begin < 0 or end > ids.shape[0]:
                raise ValueError(f"bounds: prompts from {begin} to {end} of {ids.shape[0]} tokens")
        ends = torch.tensor([ids.shape[0] - 1], device=self.device) if bounds is None else bounds[1:].long() - 1
        states: list[torch.Tensor] = []
        h = self._walk(self._tokens(ids), self._sequences(bounds, states), guarded=True)[1][-1][ends]
        self._check_tokens()
        tokens = torch.empty(uniform.shape, dtype=torch.int64, device=self.device)
        for k in range(uniform.shape[0]):
            if k:
                h = self._walk(tokens[k - 1], lambda i, h, gates: self.mixers[i].step(h, gates, states[i]), from_end=False)[1][-1]
            tokens[k] = sample(h @ self.head.weight.T, uniform[k], **settings)[0]
        return tokens

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

    def step(self, ids: torch.Tensor, labels: torch.Tensor, bounds: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(loss, gradient norm before clipping), both 0-d on the device: gradients, clipping over all of them, AdamW. Ids outside the
        table raise ``ValueError`` before any parameter is written (but not from a captured graph, which cannot)."""
        guarded = not torch.cuda.is_current_stream_capturing()
        loss = self._backward(ids, labels, bounds, guarded)
        if guarded:
            self._check_tokens()
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
    parser.add_argument("--mixing", choices=KINDS, help="a gated recurrence of that kind between the tokens")
    parser.add_argument("--sequences", type=int, default=1, help="the tokens are that many sequences (with --mixing)")
    parser.add_argument("--generate", type=int, default=0, help="tokens that follow a prompt of eight after the training")
    args = parser.parse_args(argv)
    layers = [hip_layer(make_cell(args.cell, args.seed + i)) for i in range(args.layers)]
    trainer = LMTrainer(layers, args.vocab, args.tokens, args.max_norm, args.lr, seed=args.seed, mixing=args.mixing)
    g = torch.Generator(trainer.device).manual_seed(args.seed + 1)
    successor = torch.randperm(args.vocab, generator=g, device=trainer.device)
    bounds = None
    if args.mixing is not None:
        bounds = torch.linspace(0, args.tokens, max(1, args.sequences) + 1, device=trainer.device).long()
    for k in range(args.steps):
        ids, labels = synthetic_batch(args.vocab, args.tokens, trainer.device, g, successor)
        if bounds is not None:  # of the token before it; the first of a sequence has none
            labels = labels.roll(1)
            labels[bounds[:-1].clamp(max=args.tokens - 1)] = IGNORE
        torch.cuda.synchronize()
        start = time.perf_counter()
        loss, norm = trainer.step(ids, labels, bounds)
        torch.cuda.synchronize()
        print(json.dumps({"step": k, "loss": round(float(loss), 5), "grad_norm": round(float(norm), 5),
                          "ms": round((time.perf_counter() - start) * 1e3, 3)}), flush=True)
    if args.generate > 0:
        prompt = torch.randint(0, args.vocab, (8,), generator=g, device=trainer.device)
        uniform = torch.rand(args.generate, 1, generator=g, dtype=torch.float32, device=trainer.device)
        tokens = trainer.generate(prompt, uniform, temperature=0.8, top_p=0.95)
        print(json.dumps({"prompt": prompt.tolist(), "tokens": tokens[:, 0].tolist()}), flush=True)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
