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

import functools
import math
from array import array
from collections.abc import Iterable

import torch

from . import _lib
from .runtime import _VALUE_TYPES, _device, current_stream

NORM_TYPES = (2.0, math.inf)
_CUDA = torch.device("cuda", 0)


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


def _table(tensors: Iterable[torch.Tensor], what: str) -> tuple[list, array, array, array, bool]:
    """(tensors, pointers, entry counts, value types, whether all are contiguous) of a call's tensors, checked."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    types = [_VALUE_TYPES.get(t.dtype, -1) for t in tensors]
    if -1 in types or any([t.get_device() for t in tensors]):
        raise ValueError(f"{what}: float32 or bfloat16 tensors of one device, cuda:0, are required; found "
                         + ", ".join(sorted({f"{t.dtype} on {t.device}" for t in tensors})))
    contiguous = all([t.is_contiguous() for t in tensors])
    if not contiguous:
        for t in tensors:
            if not _dense(t):
                raise ValueError(f"{what}: a tensor of shape {list(t.shape)} and strides {list(t.stride())} does not fill its memory")
    return (tensors, array("Q", [t.data_ptr() for t in tensors]), array("Q", [t.numel() for t in tensors]), array("i", types), contiguous)


def _at(values: array) -> int:
    return values.buffer_info()[0]


@functools.lru_cache(maxsize=None)
def _workspace_bytes(count: int) -> int:
    return _lib.query_bytes(_lib.load().hffn_clip_workspace, count)


def _buffers(count: int, norm_type: float) -> tuple:
    if norm_type not in NORM_TYPES:
        raise ValueError(f"norm_type is 2 or inf, not {norm_type!r}")
    device = _device(None) if count == 0 else _CUDA  # the tensors lie there
    work = torch.empty(_workspace_bytes(count), dtype=torch.uint8, device=device)
    return work, torch.empty((), dtype=torch.float32, device=device), current_stream(device)


def grad_norm(tensors: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The 2-norm (or, ``norm_type=inf``, the largest magnitude) over all entries of all tensors: float32 0-d on the device,
    zero for no entries, NaN where an entry is."""
    tensors, pointers, counts, types, _ = _table(tensors, "tensors")
    work, norm, stream = _buffers(len(tensors), norm_type)
    _lib.check(_lib.load().hffn_grad_norm(len(tensors), _at(pointers), _at(counts), _at(types), int(norm_type == math.inf), work.data_ptr(),
                                          work.numel(), norm.data_ptr(), stream), "gradient norm")
    return norm


def clip_grad_norm_(tensors: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    out: Iterable[torch.Tensor] | None = None) -> torch.Tensor:
    """``grad_norm`` of the tensors, every entry of which is then scaled by ``min(1, max_norm / (norm + 1e-6))``: in place, or into
    ``out``, a tensor of the same shape and strides for each (float32 or bfloat16). No two tensors may share memory. Returns the
    norm before scaling; the factor is taken from the float64 norm, so that one beyond float32's range (returned as infinity)
    scales as any other. Infinite entries become NaN and all others zero, a NaN makes all NaN; ``max_norm=inf`` scales nothing
    while the entries are finite. Autograd does not record the scaling; it sees that the tensors (or
    ``out``) were written."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm={max_norm} must not be negative")
    tensors, pointers, counts, types, contiguous = _table(tensors, "tensors")
    to = (None, None)
    if out is not None:
        into, to_pointers, _, to_types, to_contiguous = _table(out, "out")
        same = [t.shape for t in tensors] == [t.shape for t in into]
        if not same or not (contiguous and to_contiguous) and [t.stride() for t in tensors] != [t.stride() for t in into]:
            raise ValueError("out must hold a tensor of the same shape and strides for each tensor")
        to = (_at(to_pointers), _at(to_types))
    work, norm, stream = _buffers(len(tensors), norm_type)
    _lib.check(_lib.load().hffn_clip(len(tensors), _at(pointers), to[0], _at(counts), _at(types), to[1], int(norm_type == math.inf), max_norm,
                                     work.data_ptr(), work.numel(), norm.data_ptr(), stream), "clip")
    torch.autograd.graph.increment_version(tensors if out is None else into)
    return norm
