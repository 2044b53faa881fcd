"""The embedding of a language model on the HIP library: rows of a table, scaled, and the table's gradient.

    out_n = scale * weight[ids_n],    gw_v = scale * sum over the n with ids_n = v of g_n

    table = TokenEmbedding(weight, scale=1.0)     # weight [V, d] float32 or bfloat16 on the GPU, read at every call
    x = table.forward(ids)                        # [N, d] of the weight's type
    gw = table.backward(ids, g)                   # [V, d], also table.grad
    table.backward(ids, g, into=head.grad)        # added to a gradient that is there: a head that shares the weight

The gradient sorts the positions by their tokens and adds each token's rows in float32, in a fixed order (the positions' own for
up to 64 of them, pieces of 64, four rows at a time, for more): results repeat bit for bit. Whole gradients are zero in the rows of other tokens; with
``into`` those rows are neither read nor written.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .loss import MAX_VOCAB, MAX_WIDTH, rows_of
from .runtime import MAX_TOKENS, StreamUses, _device, _value_type, current_stream

_ID_BYTES = {torch.int32: 4, torch.int64: 8}
_FROM_END = 16


@functools.lru_cache(maxsize=4096)
def _gradient_workspace(value_type: int, n: int, d_model: int, vocab: int) -> int:
    return _lib.query_bytes(_lib.load().hffn_embedding_gradient_workspace, value_type, n, d_model, vocab)


class TokenEmbedding:
    """One table (see the module docstring). Ids are int32 or int64 [N], any stride; one outside [0, V) gives a row of NaN and
    has no part in the gradient, nor has ``padding_index``; with ``from_end`` those from -V on are ids too, as tensors are indexed. The buffer of ``grad`` is the object's own, made by its first
    ``backward`` without ``into`` and overwritten by the next. Calls are queued on PyTorch's current stream; calls of one object
    on several streams have to be ordered by the caller. Autograd records none of them: a g that requires gradients is refused, the
    weight's gradient is the one returned."""

    def __init__(self, weight: torch.Tensor, *, scale: float = 1.0, padding_index: int | None = None) -> None:
        self.device = _device(weight.device)
        if weight.dim() != 2 or not weight.is_contiguous() or weight.numel() == 0:
            raise ValueError(f"weight must be a contiguous, non-empty [V, d] tensor, not {list(weight.shape)}")
        if weight.shape[0] > MAX_VOCAB or weight.shape[1] > MAX_WIDTH:
            raise ValueError(f"weight of {list(weight.shape)}: at most [{MAX_VOCAB}, {MAX_WIDTH}]")
        self.value_type = _value_type(weight, "weight")
        self.weight, self.scale = weight.detach(), float(scale)
        self.vocab, self.d_model = weight.shape
        if padding_index is not None and not 0 <= padding_index < self.vocab:
            raise ValueError(f"padding_index={padding_index} outside [0, {self.vocab})")
        self.padding_index = padding_index
        self.grad: torch.Tensor | None = None  # gw of the last backward without into
        self._streams = StreamUses()
        self._lib = _lib.load()

    def _ids(self, ids: torch.Tensor, from_end: bool) -> tuple:
        if ids.dim() != 1 or ids.dtype not in _ID_BYTES or ids.get_device() != 0:
            raise ValueError(f"ids: an int32 or int64 [N] tensor on cuda:0 is required, not {ids.dtype} {list(ids.shape)} on {ids.device}")
        n = ids.shape[0]
        if n > MAX_TOKENS:
            raise ValueError(f"ids: N={n} above {MAX_TOKENS}")
        return n, (ids.data_ptr(), ids.stride(0) if n > 1 else 1, _ID_BYTES[ids.dtype] + (_FROM_END if from_end else 0))

    def forward(self, ids: torch.Tensor, *, from_end: bool = False, outside: torch.Tensor | None = None) -> torch.Tensor:
        """The scaled rows of tokens ids [N]: a new [N, d] tensor of the weight's type. ``outside``, int32 [1] on the device, becomes 1
        if an id has no row, and is not written else."""
        n, args = self._ids(ids, from_end)
        if outside is not None and (outside.dtype != torch.int32 or outside.shape != (1,) or outside.get_device() != 0):
            raise ValueError(f"outside: an int32 [1] tensor on {self.device} is required, not {outside.dtype} {list(outside.shape)} on {outside.device}")
        out = self.weight.new_empty(n, self.d_model)
        if n:
            _lib.check(self._lib.hffn_embedding_guarded(self.value_type, self.weight.data_ptr(), *args, self.scale, out.data_ptr(),
                                                        None if outside is None else outside.data_ptr(), self.d_model, self.vocab, n,
                                                        current_stream(self.device)), "embedding")
        return out

    def backward(self, ids: torch.Tensor, g: torch.Tensor, into: torch.Tensor | None = None, *, from_end: bool = False) -> torch.Tensor:
        """The weight's gradient, for g [N, d] of the forward's output, of the weight's type and any row stride: ``self.grad``, or
        ``into``, a contiguous [V, d] tensor of that type that the sums are added to."""
        n, args = self._ids(ids, from_end)
        g, stride = rows_of(g, "g", self.d_model, self.weight.dtype)
        if g.shape[0] != n:
            raise ValueError(f"g: {g.shape[0]} rows for {n} ids")
        queue = current_stream(self.device)
        if into is None:
            if self.grad is None:
                self._streams.allocated()
                self.grad = torch.empty_like(self.weight)
            self._streams.use(queue, self.device, (self.grad,))
            to = self.grad
        else:
            to = into
            if to.shape != self.weight.shape or to.dtype != self.weight.dtype or not to.is_contiguous() or to.get_device() != 0:
                raise ValueError(f"into must be a contiguous {self.weight.dtype} {list(self.weight.shape)} tensor on {self.device}")
        if n:
            work = torch.empty(_gradient_workspace(self.value_type, n, self.d_model, self.vocab), dtype=torch.uint8, device=self.device)
            _lib.check(self._lib.hffn_embedding_gradient(self.value_type, g.data_ptr(), stride, *args, -1 if self.padding_index is None else self.padding_index,
                                                         self.scale, int(into is not None), to.data_ptr(), work.data_ptr(), work.numel(), self.d_model,
                                                         self.vocab, n, queue), "embedding gradient")
            if into is not None:
                torch.autograd.graph.increment_version(to)
        elif into is None:
            to.zero_()
        return to
