"""Buffers that the library writes, without a GPU: their types and sizes do not follow PyTorch's default type, and the allocator knows
the streams that use them."""
from __future__ import annotations

import pytest
import torch

from hffn_amd import _lib, clip, loss, norm


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


class Library:
    """Stands in for the library: every call succeeds and does nothing."""

    def __getattr__(self, name):
        return lambda *args: _lib.OK


class Streams:
    """Stands in for PyTorch's streams: the current one, and which buffers were made known to which."""

    def __init__(self, monkeypatch):
        self.current, self.recorded = 1, []
        for module in (loss, norm):
            monkeypatch.setattr(module, "current_stream", lambda device: self.current)
            monkeypatch.setattr(module, "_device", lambda device: torch.device("cpu"))
        monkeypatch.setattr(_lib, "load", Library)
        monkeypatch.setattr(_lib, "query_bytes", lambda function, *sizes: 4096 * sizes[1])
        monkeypatch.setattr(norm, "_backward_workspace", lambda n, d: 4096)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.current)
        monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
        monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: self.recorded.append((t.data_ptr(), stream)))

    def know(self, buffers, stream):
        return all((t.data_ptr(), stream) in self.recorded for t in buffers)


def test_head_loss_buffers_are_known_to_every_stream_that_uses_them(monkeypatch):
    """Constructed on one stream and called on another; grown by ``reserve`` on a third between two calls on the second."""
    streams = Streams(monkeypatch)
    x, labels = torch.zeros(64, 8), torch.zeros(64, dtype=torch.int64)
    head = loss.HeadLoss(torch.zeros(100, 8), max_tokens=16)
    streams.current = 2
    head.losses(x[:16], labels[:16])
    assert streams.know((head._workspace, head._losses), 2)
    streams.current = 3
    head.reserve(64)
    streams.current = 2
    head.step(x, labels)
    assert streams.know((head._workspace, head._losses, head._gx, head._loss, head.grad), 2)
    streams.current = 1
    head.step(x, labels)
    assert streams.know((head._workspace, head._losses, head._gx, head._loss, head.grad), 1)


def test_residual_norm_gradients_are_known_to_every_stream_that_uses_them(monkeypatch):
    streams = Streams(monkeypatch)
    boundary, rows = norm.ResidualNorm(torch.ones(8), torch.zeros(8)), torch.zeros(4, 8)
    boundary.backward(rows, None, None, rows)
    streams.current = 2
    boundary.backward(rows, None, None, rows)
    assert streams.know(boundary.gradients().values(), 2)
