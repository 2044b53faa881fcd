"""The boundary between two blocks of a residual stack on the HIP library, forward and backward in one pass over the rows:

    u = post_norm(f)  (or f),    r = x + scale * gate * u,    h = norm(r)

``x`` is the residual stream, ``f`` the output of the block that ends, ``h`` the input of the one that begins. The norms are layer
norms (``kind="layer"``: weight and, where given, bias) or RMS norms (``kind="rms"``: weight), the gate a vector over the
channels, the scale a number; post norm and gate are optional, and without ``f`` the boundary is the norm alone.

    boundary = ResidualNorm(weight, bias, gate=gate, scale=0.5)
    r, h = boundary.forward(x, f)
    gx, gf = boundary.backward(r, f, gr, gh)   # and boundary.gradients(): the parameters' gradients

The backward takes r and f as the forward gave and read them and computes the rows' statistics again: nothing is kept
between the calls.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from .loss import rows_of
from .runtime import StreamUses, _device, _value_type, current_stream

KINDS = ("layer", "rms")
PARAMETERS = ("weight", "bias", "gate", "post_weight", "post_bias")
MAX_WIDTH = 16384


@functools.lru_cache(maxsize=4096)
def _backward_workspace(n: int, d_model: int) -> int:
    return _lib.query_bytes(_lib.load().hffn_residual_norm_backward_workspace, n, d_model)


def _pointer(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


class ResidualNorm:
    """One boundary (see the module docstring). Parameters are float32 [d] tensors, held as given and read at every call; rows are
    float32 or bfloat16 [N, d] with any row stride, all of one type. r, h, gx and gf are new contiguous tensors of that
    type; sums are taken in float32. Calls are queued on PyTorch's current stream. Autograd records none of them: gradients are those
    of ``backward`` and ``gradients()``, and rows that require gradients are refused."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, *, gate: torch.Tensor | None = None,
                 post_weight: torch.Tensor | None = None, post_bias: torch.Tensor | None = None, scale: float = 1.0,
                 kind: str = "layer", eps: float = 1e-5) -> None:
        self.device = _device(weight.device)
        if kind not in KINDS:
            raise ValueError(f"kind is one of {KINDS}, not {kind!r}")
        if kind == "rms" and (bias is not None or post_bias is not None):
            raise ValueError("an RMS norm has no bias")
        if post_bias is not None and post_weight is None:
            raise ValueError("post_bias needs post_weight")
        if not eps >= 0.0:
            raise ValueError(f"eps={eps} must not be negative")
        self.d_model = weight.numel()
        if not 1 <= self.d_model <= MAX_WIDTH:
            raise ValueError(f"{self.d_model} channels outside [1, {MAX_WIDTH}]")
        self.kind, self.scale, self.eps = kind, float(scale), float(eps)
        self._parameters = {}
        for name, t in zip(PARAMETERS, (weight, bias, gate, post_weight, post_bias)):
            if t is None:
                continue
            if not (t.dtype == torch.float32 and t.dim() == 1 and t.numel() == self.d_model and t.is_contiguous() and t.device == self.device):
                raise ValueError(f"{name} must be a contiguous float32 [{self.d_model}] tensor on {self.device}")
            self._parameters[name] = t.detach()
        self._gradients: dict[str, torch.Tensor] = {}
        self._streams = StreamUses()
        self._lib = _lib.load()

    def parameters(self) -> dict[str, torch.Tensor]:
        return self._parameters

    def gradients(self) -> dict[str, torch.Tensor]:
        """By parameter, float32 [d], of the last backward (empty before the first); the next one overwrites them."""
        return self._gradients

    def _needs_f(self) -> bool:
        return "gate" in self._parameters or "post_weight" in self._parameters

    def _rows(self, t: torch.Tensor | None, name: str, like: torch.Tensor) -> tuple[torch.Tensor | None, int]:
        if t is None:
            return None, 0
        t, stride = rows_of(t, name, self.d_model, like.dtype)
        if t.shape[0] != like.shape[0]:
            raise ValueError(f"{name}: {t.shape[0]} rows for {like.shape[0]}")
        return t, stride

    def forward(self, x: torch.Tensor, f: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(r, h); without ``f`` (boundaries without gate and post norm) r is x itself."""
        value_type = _value_type(x, "x")
        if f is None and self._needs_f():
            raise ValueError("a boundary with a gate or a post norm needs f")
        x, x_stride = self._rows(x, "x", x)
        f, f_stride = self._rows(f, "f", x)
        n, p = x.shape[0], self._parameters
        h = torch.empty_like(x, memory_format=torch.contiguous_format)
        r = x if f is None else torch.empty_like(h)
        if n:
            _lib.check(self._lib.hffn_residual_norm(value_type, x.data_ptr(), x_stride, _pointer(f), f_stride,
                                                    *(_pointer(p.get(name)) for name in PARAMETERS), self.scale, self.eps,
                                                    int(self.kind == "layer"), None if f is None else r.data_ptr(), h.data_ptr(),
                                                    self.d_model, n, current_stream(self.device)), "residual norm")
        return r, h

    def backward(self, r: torch.Tensor, f: torch.Tensor | None, gr: torch.Tensor | None,
                 gh: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor | None]:
        """(gx, gf): the gradients of x and f for those of r (``None``: none but through h) and h, where r is the forward's (the
        input itself where it had no f); gf is ``None`` without ``f``. The parameters' gradients go to ``gradients()``."""
        value_type = _value_type(r, "r")
        if f is None and self._needs_f():
            raise ValueError("a boundary with a gate or a post norm needs f")
        r, r_stride = self._rows(r, "r", r)
        f, f_stride = self._rows(f, "f", r)
        gr, gr_stride = self._rows(gr, "gr", r)
        gh, gh_stride = self._rows(gh, "gh", r)
        n, d, p = r.shape[0], self.d_model, self._parameters
        gx = torch.empty_like(r, memory_format=torch.contiguous_format)
        gf = None if f is None else torch.empty_like(gx)
        g = self._gradients
        if not g:
            g.update((name, torch.empty_like(t)) for name, t in p.items())
        stream = current_stream(self.device)
        self._streams.use(stream, self.device, g.values())
        if n == 0:
            for t in g.values():
                t.zero_()
            return gx, gf
        work = torch.empty(_backward_workspace(n, d), dtype=torch.uint8, device=self.device)
        _lib.check(self._lib.hffn_residual_norm_backward(
            value_type, r.data_ptr(), r_stride, _pointer(f), f_stride, _pointer(gr), gr_stride, gh.data_ptr(), gh_stride,
            p["weight"].data_ptr(), *(_pointer(p.get(name)) for name in PARAMETERS[2:]), self.scale, self.eps, int(self.kind == "layer"),
            gx.data_ptr(), _pointer(gf), *(_pointer(g.get(name)) for name in PARAMETERS), work.data_ptr(), work.numel(), d, n, stream),
                   "residual norm backward")
        return gx, gf
