"""The global norm over many gradients and clipping to it, on the HIP library: two launches for up to 96 tensors (as many
again for every further 96), whatever their sizes, no copy to the host.

    norm = grad_norm(tensors)                              # float32 0-d on the device
    norm = clip_grad_norm_(tensors, max_norm)              # and every entry times min(1, max_norm / (norm + 1e-6))
    norm = clip_grad_norm_(tensors, max_norm, out=floats)  # the scaled entries into other tensors, as for an optimizer that
                                                           # takes float32

Tensors are float32 or bfloat16, of any shape, mixed, empty ones among them; each occupies its memory without gaps (contiguous,
or permuted dimensions of that). Sums are float64; the result does not depend on scheduling.
"""
from __future__ import annotations

import ctypes
import math
from collections.abc import Iterable

import torch

from . import _lib
from .runtime import _VALUE_TYPES, _device

NORM_TYPES = (2.0, math.inf)


def _dense(t: torch.Tensor) -> bool:
    """Whether the entries fill numel() places without gaps or overlaps, in whatever order of the dimensions."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((stride, size) for stride, size in zip(t.stride(), t.shape) if size != 1):
        if stride != expected:
            return False
        expected *= size
    return True


class _Arrays:
    """The host arrays of a call: pointers, entry counts, value types."""

    def __init__(self, tensors: Iterable[torch.Tensor], what: str) -> None:
        self.tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        count = len(self.tensors)
        self.device = self.tensors[0].device if count else torch.device("cuda", 0)
        types = []
        for t in self.tensors:
            kind = _VALUE_TYPES.get(t.dtype)
            if kind is None or t.device != self.device:
                raise ValueError(f"{what}: float32 or bfloat16 tensors of one device are required, not {t.dtype} on {t.device}")
            if not _dense(t):
                raise ValueError(f"{what}: a tensor of shape {list(t.shape)} and strides {list(t.stride())} does not fill its memory")
            types.append(kind)
        at, entries = [t.data_ptr() for t in self.tensors], [t.numel() for t in self.tensors]
        self.pointers, self.counts = (ctypes.c_void_p * count)(*at), (ctypes.c_uint64 * count)(*entries)
        self.types = (ctypes.c_int * count)(*types)
        self.spans = sorted((p, p + n * (2 if kind == _lib.VALUE_BF16 else 4)) for p, n, kind in zip(at, entries, types) if n)


def _check_apart(spans: list, what: str) -> None:
    for (_, end), (start, _) in zip(spans, spans[1:]):
        if start < end:
            raise ValueError(f"{what}: two tensors share memory")


def _call(tensors: Iterable[torch.Tensor], norm_type: float) -> tuple:
    if norm_type not in NORM_TYPES:
        raise ValueError(f"norm_type is 2 or inf, not {norm_type!r}")
    arrays = _Arrays(tensors, "tensors")
    device = _device(arrays.device)
    lib = _lib.load()
    work = torch.empty(_lib.query_bytes(lib.hffn_clip_workspace, len(arrays.tensors)), dtype=torch.uint8, device=device)
    return arrays, lib, work, torch.empty((), device=device), torch.cuda.current_stream(device).cuda_stream


@torch.no_grad()
def grad_norm(tensors: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The 2-norm (or, ``norm_type=inf``, the largest magnitude) over all entries of all tensors: float32 0-d on the device,
    zero for no entries, NaN where an entry is."""
    arrays, lib, work, norm, stream = _call(tensors, norm_type)
    _lib.check(lib.hffn_grad_norm(len(arrays.tensors), arrays.pointers, arrays.counts, arrays.types, int(norm_type == math.inf),
                                  work.data_ptr(), work.numel(), norm.data_ptr(), stream), "gradient norm")
    return norm


@torch.no_grad()
def clip_grad_norm_(tensors: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    out: Iterable[torch.Tensor] | None = None) -> torch.Tensor:
    """``grad_norm`` of the tensors, every entry of which is then scaled by ``min(1, max_norm / (norm + 1e-6))``: in place, or into
    ``out``, a tensor of the same shape and strides for each (float32 or bfloat16, sharing no memory with any). Returns the norm
    before scaling. An infinite norm makes the entries zero (infinite ones NaN), a NaN one makes all NaN; ``max_norm=inf``
    scales nothing while the norm is finite."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm={max_norm} must not be negative")
    arrays, lib, work, norm, stream = _call(tensors, norm_type)
    spans, into = arrays.spans, None
    if out is not None:
        into = _Arrays(out, "out")
        if len(into.tensors) != len(arrays.tensors) or any(a.shape != b.shape or a.stride() != b.stride() or a.device != b.device
                                                           for a, b in zip(arrays.tensors, into.tensors)):
            raise ValueError("out must hold a tensor of the same shape, strides and device for each tensor")
        _check_apart(sorted(spans + into.spans), "out")
    else:
        _check_apart(spans, "tensors")
    _lib.check(lib.hffn_clip(len(arrays.tensors), arrays.pointers, into and into.pointers, arrays.counts, arrays.types,
                             into and into.types, int(norm_type == math.inf), max_norm, work.data_ptr(), work.numel(), norm.data_ptr(),
                             stream), "clip")
    return norm
