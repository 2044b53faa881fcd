"""Softmax cross entropy of a language-model head on the HIP library: the loss of every token (scoring, evaluation), or the
mean loss with the gradients of the hidden rows and of the head's weight (a training step), without the logits.

For hidden rows ``x [N, d]``, a weight ``[V, d]`` and labels: ``l_t = log sum_v exp(x_t . w_v) - x_t . w_label(t)``; with
``p = softmax(x W^T)`` and ``D = (p - onehot) / counted``: ``gx = D W``, ``gw = D^T x``. Logits are computed in pieces of the
vocabulary and not kept: the sums of exponentials first, then piece by piece the softmax (16 bits an entry, 32 in float32
and for a few tokens) and its two products. Tokens whose label is ``ignore_index`` take no part: their losses and rows of ``gx``
are zero whatever their rows of x hold, and the products run over the others alone.

    head = HeadLoss(weight, max_tokens=2048)          # weight [V, d] float32 or bfloat16 on the GPU, read at every call
    losses = head.losses(x, labels)                   # float32 [N]
    loss, gx, gw = head.step(x, labels)               # the mean and its gradients; gw is head.grad

Sums are float32 throughout (over tokens and slices of the vocabulary in fixed orders: results repeat bit for bit). bfloat16 steps
of more than 64 tokens round D to bfloat16 for its two products, which makes the gradients' error 1.1 to 1.4 times what their own
rounding makes it (more where three tokens or fewer of them count); float32 calls multiply entries of 22 bits or more and keep D to 2^-38, so that a vocabulary row whose probability
stays below that for every token gets no gradient. Whose gradients need more than bfloat16 steps give passes float32 tensors. An
infinity in a float32 row makes what it enters NaN.
"""
from __future__ import annotations

import torch

from . import _lib
from .runtime import MAX_TOKENS, StreamUses, _device, _value_type, current_stream

REDUCTIONS = ("mean", "sum")
PIECE_BYTES = 512 << 20
MAX_WIDTH, MAX_VOCAB = 1 << 15, 1 << 24
_LABEL_BYTES = {torch.int32: 4, torch.int64: 8}


def rows_of(t: torch.Tensor, name: str, width: int, dtype: torch.dtype) -> tuple[torch.Tensor, int]:
    """``t`` as rows of ``width`` entries the kernels read, and their stride: itself where a row's entries are adjacent and rows
    do not overlap, else a contiguous copy. Raises ``ValueError`` for another shape, type or device, and where autograd would
    expect the call to be recorded."""
    if t.dim() != 2 or t.dtype != dtype or t.get_device() != 0 or t.shape[1] != width:
        raise ValueError(f"{name}: a {dtype} [N, {width}] tensor on cuda:0 is required, not {t.dtype} {list(t.shape)} on {t.device}")
    if t.shape[0] > MAX_TOKENS:
        raise ValueError(f"{name}: N={t.shape[0]} above {MAX_TOKENS}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires gradients, and autograd does not record this call: pass it detached, or under torch.no_grad()")
    if t.is_contiguous():
        return t, width
    if t.stride(1) == 1 and t.stride(0) >= width:
        return t, t.stride(0)
    return t.contiguous(), width


class HeadLoss:
    """The loss of one head (see the module docstring). Buffers are the object's own and grow with the calls; what a
    call returns are views of them that the next call overwrites. Calls are queued on PyTorch's current stream; calls of one
    object on several streams have to be ordered by the caller. Autograd records none of them: the gradients are those that
    ``step`` returns, the weight's too where it requires gradients, and an x that does is refused. A captured graph holds the
    buffers of its capture: ``reserve`` the sizes that later calls will have before it, so that none of these replaces them."""

    def __init__(self, weight: torch.Tensor, max_tokens: int = 1, ignore_index: int = -100, reduction: str = "mean",
                 piece_bytes: int = PIECE_BYTES) -> None:
        """``max_tokens``: the calls the buffers are first sized for (``losses``; ``step``'s own come with its first call or
        ``reserve``). ``piece_bytes``: what a piece of the vocabulary's softmax may take in ``step`` (N tokens times its rows, 2
        bytes an entry in bfloat16 above 64 tokens, 4 else; 256 rows at least, 8.4 million and 2^35 entries at most): the last
        piece's logits are computed once, the others' twice."""
        self.device = _device(weight.device)
        if weight.dim() != 2 or not weight.is_contiguous() or weight.numel() == 0:
            raise ValueError(f"weight must be a contiguous, non-empty [V, d] tensor, not {list(weight.shape)}")
        if weight.shape[0] > MAX_VOCAB or weight.shape[1] > MAX_WIDTH:
            raise ValueError(f"weight of {list(weight.shape)}: at most [{MAX_VOCAB}, {MAX_WIDTH}]")
        if reduction not in REDUCTIONS:
            raise ValueError(f"reduction is one of {REDUCTIONS}, not {reduction!r}")
        if piece_bytes < 1:
            raise ValueError(f"piece_bytes={piece_bytes} must be positive")
        self.piece_bytes = int(piece_bytes)
        self.value_type = _value_type(weight, "weight")
        self.weight, self.ignore_index, self.reduction = weight.detach(), int(ignore_index), reduction
        self.vocab, self.d_model = weight.shape
        self._lib = _lib.load()
        self._aligned = int(weight.data_ptr() % 16 == 0)
        self._workspace: torch.Tensor | None = None
        self._losses: torch.Tensor | None = None
        self._gx: torch.Tensor | None = None
        self._loss: torch.Tensor | None = None
        self.grad: torch.Tensor | None = None  # gw of the last step
        self._streams = StreamUses()
        self._sized = [0, 0]  # tokens the buffers were last sized for, for losses and for step (more may need less: fewer pieces)
        self.reserve(max_tokens, gradients=False)

    def _bytes(self, n: int, gradients: bool) -> int:
        return _lib.query_bytes(self._lib.hffn_loss_workspace, self.value_type, n, self.d_model, self.vocab, self._aligned, int(gradients), self.piece_bytes)

    def _new(self, *shape: int, dtype: torch.dtype) -> torch.Tensor:
        self._streams.allocated()
        return torch.empty(shape, dtype=dtype, device=self.device)

    def reserve(self, n: int, gradients: bool = True) -> None:
        """Size the buffers for calls of ``n`` tokens (``gradients``: for ``step`` too); allocates what must grow."""
        if not 1 <= n <= MAX_TOKENS:
            raise ValueError(f"N={n} outside [1, {MAX_TOKENS}]")
        if n == self._sized[gradients]:
            return
        need = self._bytes(n, gradients)
        if self._workspace is None or self._workspace.numel() < need:
            self._workspace = self._new(need, dtype=torch.uint8)
        if self._losses is None or self._losses.numel() < n:
            self._losses = self._new(n, dtype=torch.float32)
        if gradients and (self._gx is None or self._gx.shape[0] < n):
            self._gx = self._new(n, self.d_model, dtype=self.weight.dtype)
        if gradients and self.grad is None:
            self.grad = self._new(self.vocab, self.d_model, dtype=self.weight.dtype)
            self._loss = self._new(dtype=torch.float32)
        self._sized[gradients] = n

    def workspace_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self._workspace, self._losses, self._gx) if t is not None)

    def _call(self, x: torch.Tensor, labels: torch.Tensor, gradients: bool) -> tuple:
        """The checked arguments both entries share, and the stream; the buffers are sized."""
        x, stride = rows_of(x, "x", self.d_model, self.weight.dtype)
        n = x.shape[0]
        if labels.dim() != 1 or labels.shape[0] != n or labels.dtype not in _LABEL_BYTES or labels.get_device() != 0:
            raise ValueError(f"labels: an int32 or int64 [{n}] tensor on {self.device} is required, not {labels.dtype} "
                             f"{list(labels.shape)} on {labels.device}")
        stream = current_stream(self.device)
        self.reserve(max(n, 1), gradients)
        self._streams.use(stream, self.device, (self._workspace, self._losses, self._gx, self._loss, self.grad))
        return x, (self.value_type, x.data_ptr(), stride, self.weight.data_ptr(), labels.data_ptr(), labels.stride(0) if n > 1 else 1,
                   _LABEL_BYTES[labels.dtype], self.ignore_index), stream

    def losses(self, x: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
        """float32 [N]: the negative log likelihood of every token's label; 0 where it is ``ignore_index``, NaN where it lies
        outside the vocabulary. ``x``: [N, d] of the weight's type, any row stride."""
        x, args, stream = self._call(x, labels, False)
        n = x.shape[0]
        if n:
            _lib.check(self._lib.hffn_losses(*args, self._losses.data_ptr(), self._workspace.data_ptr(), self._workspace.numel(),
                                             self.d_model, self.vocab, n, stream), "losses")
        return self._losses[:n]

    def step(self, x: torch.Tensor, labels: torch.Tensor, scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(loss, gx, gw): the mean (or sum) of the counted tokens' losses, float32 0-d, and the gradients of ``scale`` times it
        with respect to x ([N, d], zero rows for ignored tokens) and to the weight ([V, d], also ``self.grad``), both of the
        weight's type. Where every token is ignored all three are zero; a label outside the vocabulary makes them NaN."""
        x, args, stream = self._call(x, labels, True)
        n = x.shape[0]
        if n == 0:
            return self._loss.zero_(), self._gx[:0], self.grad.zero_()
        _lib.check(self._lib.hffn_loss_step(*args, int(self.reduction == "mean"), scale, self.piece_bytes, self._loss.data_ptr(), self._gx.data_ptr(),
                                            self.grad.data_ptr(), self._workspace.data_ptr(), self._workspace.numel(), self.d_model,
                                            self.vocab, n, stream), "loss step")
        return self._loss, self._gx[:n], self.grad
