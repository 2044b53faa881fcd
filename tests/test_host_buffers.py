"""Buffers that the library writes, without a GPU: their types and sizes do not follow PyTorch's default type."""
from __future__ import annotations

import pytest
import torch

from hffn_amd import _lib, clip


@pytest.mark.parametrize("default", (torch.bfloat16, torch.float64))
def test_clip_buffers_hold_what_the_library_is_told(monkeypatch, default):
    monkeypatch.setattr(clip, "_CUDA", torch.device("cpu"))
    monkeypatch.setattr(clip, "current_stream", lambda device: 0)
    torch.set_default_dtype(default)
    try:
        work, norm, _ = clip._buffers(97, 2.0)
    finally:
        torch.set_default_dtype(torch.float32)
    assert work.numel() * work.element_size() >= _lib.query_bytes(_lib.load().hffn_clip_workspace, 97)
    assert norm.dtype == torch.float32
