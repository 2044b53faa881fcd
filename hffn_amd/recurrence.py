"""A gated linear recurrence between the tokens of sequences on the HIP library: forward and backward as a scan over all tokens
at once, and one token of each sequence at a time.

    z_t = sigmoid(gate_t + bias),    h_t = (1 - z_t) h_t-1 + v_t        (per channel, from a state or zero)

where ``v`` is ``z x`` (``kind="tied"``: what is let go is what comes in), ``sqrt(1 - (1 - z)^2) x`` (``"normed"``: rows of unit
variance keep it) or ``x`` itself (``"free"``).

    mixer = GatedRecurrence(bias, kind="tied")
    h, last = mixer.forward(x, gate, bounds, state)                  # sequences laid end to end, and their states behind
    gx, ggate, gstate = mixer.backward(x, gate, h, gh, bounds, state, glast)   # and mixer.gradients(): the bias's
    h = mixer.step(x, gate, state)                                   # one token each, the state in place

``bounds`` [S + 1] tells where each sequence begins, and where the last one ends; without it the rows are one sequence.
States are float32, and 1 - z is never rounded to a float by itself, so that channels that forget a millionth per token do
not drift. An infinity stays one for the rest of its sequence, however little of it is kept, until a NaN or its opposite comes in; so does
what leaves float32 on the way, for which h + v may be enough (z up to a half takes h + v first), or a tile's inputs alone. The backward takes h as the forward gave it; nothing is kept between the calls.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .loss import MAX_WIDTH, refuse_recording, rows_of
from .runtime import StreamUses, _device, _value_type, current_stream

KINDS = ("tied", "normed", "free")
MAX_SEQUENCES = 1 << 20
_BOUND_BYTES = {torch.int32: 4, torch.int64: 8}


@functools.lru_cache(maxsize=4096)
def _workspace(n: int, d_model: int, gradients: bool) -> int:
    return _lib.query_bytes(_lib.load().hffn_scan_workspace, n, d_model, int(gradients))


class GatedRecurrence:
    """One recurrence (see the module docstring). The bias is a float32 [d] tensor, held as given and read at every call; x, gate, h
    and their gradients are float32 or bfloat16 [N, d] rows, all of one type, those that come in with any row stride, those
    returned new and contiguous; sums are taken in float32, in an order that goes by the rows' places in the batch (the last bits of a sequence
    depend on where it begins there, not on the other sequences). Rows outside every sequence are read by none, and zero in h and in the
    gradients. Calls are queued on PyTorch's current stream; calls of ``backward``
    of one object on several streams have to be ordered by the caller. Autograd records none of them: gradients are those of ``backward``
    and ``gradients()``, and rows that require gradients are refused."""

    def __init__(self, bias: torch.Tensor, kind: str = "tied") -> None:
        self.device = _device(bias.device)
        if kind not in KINDS:
            raise ValueError(f"kind is one of {KINDS}, not {kind!r}")
        if not (bias.dtype == torch.float32 and bias.dim() == 1 and bias.is_contiguous()):
            raise ValueError(f"bias must be a contiguous float32 [d] tensor, not {bias.dtype} {list(bias.shape)}")
        self.d_model = bias.numel()
        if not 1 <= self.d_model <= MAX_WIDTH:
            raise ValueError(f"{self.d_model} channels outside [1, {MAX_WIDTH}]")
        self.bias, self.kind, self._kind = bias.detach(), kind, KINDS.index(kind)
        self._gradients: dict[str, torch.Tensor] = {}
        self._streams = StreamUses()
        self._lib = _lib.load()

    def parameters(self) -> dict[str, torch.Tensor]:
        return {"bias": self.bias}

    def gradients(self) -> dict[str, torch.Tensor]:
        """By parameter, float32 [d], of the last backward (empty before the first); the next one overwrites them."""
        return self._gradients

    def _rows(self, t: torch.Tensor, name: str, like: torch.Tensor) -> tuple[torch.Tensor, int]:
        t, stride = rows_of(t, name, self.d_model, like.dtype)
        if t.shape[0] != like.shape[0]:
            raise ValueError(f"{name}: {t.shape[0]} rows for {like.shape[0]}")
        return t, stride

    def _bounds(self, bounds: torch.Tensor | None) -> tuple[torch.Tensor | None, tuple]:
        if bounds is None:
            return None, (None, 8, 1)
        if bounds.dim() != 1 or not 2 <= bounds.shape[0] <= MAX_SEQUENCES + 1 or bounds.dtype not in _BOUND_BYTES or bounds.get_device() != 0:
            raise ValueError(f"bounds: an int32 or int64 [S + 1] tensor on cuda:0 is required, S in [1, {MAX_SEQUENCES}], not {bounds.dtype} "
                             f"{list(bounds.shape)} on {bounds.device}")
        bounds = bounds.contiguous()
        return bounds, (bounds.data_ptr(), _BOUND_BYTES[bounds.dtype], bounds.shape[0] - 1)

    def _states(self, t: torch.Tensor | None, name: str, sequences: int) -> torch.Tensor | None:
        if t is None:
            return None
        if t.dim() != 2 or t.dtype != torch.float32 or t.get_device() != 0 or t.shape[1] != self.d_model:
            raise ValueError(f"{name}: a float32 [S, {self.d_model}] tensor on cuda:0 is required, not {t.dtype} {list(t.shape)} on {t.device}")
        if t.shape[0] != sequences:
            raise ValueError(f"{name}: {t.shape[0]} rows for {sequences} sequences")
        refuse_recording(t, name)
        return t.contiguous()

    def forward(self, x: torch.Tensor, gate: torch.Tensor, bounds: torch.Tensor | None = None,
                state: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(h [N, d], last): last is float32 [S, d], each sequence's h behind its last token, unrounded (where it has none, its
        state); ``state`` float32 [S, d] is what the sequences begin from (``None``: zeros)."""
        value_type = _value_type(x, "x")
        x, x_stride = self._rows(x, "x", x)
        gate, gate_stride = self._rows(gate, "gate", x)
        bounds, bound_args = self._bounds(bounds)
        state = self._states(state, "state", bound_args[2])
        n, d = x.shape
        h = x.new_empty(n, d)
        last = torch.empty((bound_args[2], d), dtype=torch.float32, device=self.device)
        if n == 0:
            return h, last.zero_() if state is None else last.copy_(state)
        work = torch.empty(_workspace(n, d, False), dtype=torch.uint8, device=self.device)
        _lib.check(self._lib.hffn_scan(value_type, self._kind, x.data_ptr(), x_stride, gate.data_ptr(), gate_stride, self.bias.data_ptr(), *bound_args,
                                       None if state is None else state.data_ptr(), h.data_ptr(), last.data_ptr(), work.data_ptr(), work.numel(), d, n,
                                       current_stream(self.device)), "recurrence")
        return h, last

    def backward(self, x: torch.Tensor, gate: torch.Tensor, h: torch.Tensor, gh: torch.Tensor, bounds: torch.Tensor | None = None,
                 state: torch.Tensor | None = None, glast: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
        """(gx, ggate, gstate) for gh of the forward's h and glast of its last (``None``: zeros), where h is the forward's; gstate is
        float32 [S, d], ``None`` without a state. The bias's gradient goes to ``gradients()``."""
        value_type = _value_type(x, "x")
        x, x_stride = self._rows(x, "x", x)
        gate, gate_stride = self._rows(gate, "gate", x)
        h, h_stride = self._rows(h, "h", x)
        gh, gh_stride = self._rows(gh, "gh", x)
        bounds, bound_args = self._bounds(bounds)
        state = self._states(state, "state", bound_args[2])
        glast = self._states(glast, "glast", bound_args[2])
        n, d = x.shape
        gx = x.new_empty(n, d)
        ggate = torch.empty_like(gx)
        gstate = None if state is None else torch.empty_like(state)
        if not self._gradients:
            self._gradients["bias"] = torch.empty_like(self.bias)
        g_bias = self._gradients["bias"]
        stream = current_stream(self.device)
        self._streams.use(stream, self.device, (g_bias,))
        if n == 0:
            g_bias.zero_()
            return gx, ggate, gstate if gstate is None else gstate.zero_() if glast is None else gstate.copy_(glast)
        work = torch.empty(_workspace(n, d, True), dtype=torch.uint8, device=self.device)
        _lib.check(self._lib.hffn_scan_backward(
            value_type, self._kind, x.data_ptr(), x_stride, gate.data_ptr(), gate_stride, h.data_ptr(), h_stride, gh.data_ptr(), gh_stride,
            self.bias.data_ptr(), *bound_args, None if state is None else state.data_ptr(), None if glast is None else glast.data_ptr(), gx.data_ptr(),
            ggate.data_ptr(), g_bias.data_ptr(), None if gstate is None else gstate.data_ptr(), work.data_ptr(), work.numel(), d, n, stream),
                   "recurrence backward")
        return gx, ggate, gstate

    def step(self, x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor) -> torch.Tensor:
        """h [N, d] of one token of each of N sequences; ``state``, float32 [N, d] rows of any stride (no two in one place), becomes
        theirs behind it."""
        value_type = _value_type(x, "x")
        x, x_stride = rows_of(x, "x", self.d_model, x.dtype)
        gate, gate_stride = self._rows(gate, "gate", x)
        n, d = x.shape
        if state.dtype != torch.float32 or state.shape != x.shape or state.get_device() != 0 or not state.is_contiguous() and (
                d > 1 and state.stride(1) != 1 or n > 1 and state.stride(0) < d):
            raise ValueError(f"state: a float32 {[n, d]} tensor on cuda:0 of rows with adjacent entries that do not overlap is required, not {state.dtype} "
                             f"{list(state.shape)} of strides {list(state.stride())} on {state.device}")
        refuse_recording(state, "state")
        h = x.new_empty(n, d)
        if n:
            _lib.check(self._lib.hffn_scan_step(value_type, self._kind, x.data_ptr(), x_stride, gate.data_ptr(), gate_stride, self.bias.data_ptr(),
                                                state.data_ptr(), state.stride(0) if n > 1 else d, h.data_ptr(), d, n, current_stream(self.device)),
                       "recurrence step")
            torch.autograd.graph.increment_version(state)
        return h
