"""Objects whose buffers were made on one stream and are used on another: what is dropped while that stream's work is still
queued goes to no other tensor before the work is done."""
from __future__ import annotations

import pytest
import torch

from hffn_amd.loss import HeadLoss
from hffn_amd.norm import ResidualNorm

pytestmark = pytest.mark.gpu


def busy(stream, products=100):
    """Tens of milliseconds of products on the stream."""
    with torch.cuda.stream(stream):
        a = torch.ones(4096, 4096, device="cuda")
        for _ in range(products):
            a = (a @ a).clamp_(max=1.0)
    return a


def still(done):
    if done.query():
        pytest.skip("the stream's work was done before the memory was asked for")


def pointer_of_the_next(like):
    """Where a tensor of the same size that is allocated now lies; nothing is written to it."""
    return torch.empty(like[0], dtype=torch.uint8, device="cuda").data_ptr() == like[1]


def place(t):
    return t.numel() * t.element_size(), t.data_ptr()


@pytest.mark.parametrize("grown", (False, True))
def test_a_head_dropped_while_another_stream_uses_it(grown):
    x, weight = torch.randn(4000, 64, device="cuda"), torch.randn(20000, 64, device="cuda")
    labels = torch.arange(4000, device="cuda")
    want = HeadLoss(weight).losses(x, labels).clone()
    side = torch.cuda.Stream()
    busy(side, 1)  # the products' own first call takes the host long
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    head = HeadLoss(weight, max_tokens=1 if grown else 4000)
    if grown:  # by reserve, on this stream, after a call on the other
        with torch.cuda.stream(side):
            head.losses(x[:1], labels[:1])
        head.reserve(4000, gradients=False)
    kept = busy(side)
    with torch.cuda.stream(side):
        got = head.losses(x, labels).clone()
    done = side.record_event()
    before = place(head._workspace)
    del head
    reused = pointer_of_the_next(before)
    still(done)
    assert not reused
    torch.cuda.synchronize()
    assert torch.equal(got, want) and kept.numel()


def test_a_boundary_dropped_while_another_stream_uses_it():
    rows, weight = torch.randn(64, 16384, device="cuda"), torch.randn(16384, device="cuda")
    boundary = ResidualNorm(weight)
    boundary.backward(rows, None, None, rows)
    want = boundary.gradients()["weight"].clone()
    side = torch.cuda.Stream()
    busy(side, 1)  # the products' own first call takes the host long
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    kept = busy(side)
    with torch.cuda.stream(side):
        boundary.backward(rows, None, None, rows)
        got = boundary.gradients()["weight"].clone()
    done = side.record_event()
    before = place(boundary.gradients()["weight"])
    del boundary
    reused = [pointer_of_the_next(before) for _ in range(3)]
    still(done)
    assert not any(reused)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and kept.numel()
