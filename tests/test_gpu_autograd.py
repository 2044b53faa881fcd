"""What autograd is told of calls that it does not record: rows that require gradients are refused, and tensors that were written in
place are known to have been."""
from __future__ import annotations

import pytest
import torch

from hffn_amd.clip import clip_grad_norm_
from hffn_amd.loss import HeadLoss
from hffn_amd.norm import ResidualNorm

pytestmark = pytest.mark.gpu


def rows(**options):
    return torch.ones(6, 64, device="cuda", **options)


def test_rows_that_require_gradients_are_refused():
    head, boundary = HeadLoss(torch.ones(30, 64, device="cuda")), ResidualNorm(torch.ones(64, device="cuda"))
    labels, x, g = torch.zeros(6, dtype=torch.int64, device="cuda"), rows(), rows(requires_grad=True)
    calls = {"x requires": [lambda t: head.losses(t, labels), lambda t: head.step(t, labels), lambda t: boundary.forward(t), lambda t: boundary.forward(t, x)],
             "f requires": [lambda t: boundary.forward(x, t), lambda t: boundary.backward(x, t, x, x)],
             "r requires": [lambda t: boundary.backward(t, x, x, x)], "gr requires": [lambda t: boundary.backward(x, x, t, x)],
             "gh requires": [lambda t: boundary.backward(x, x, x, t)]}
    for match, entries in calls.items():
        for call in entries:
            for t in (g, g * 2.0):
                with pytest.raises(ValueError, match=match):
                    call(t)
            call(g.detach())
            with torch.no_grad():
                call(g)


def test_a_weight_that_requires_gradients_gets_its_gradient_from_the_step():
    weight, labels = torch.nn.Parameter(torch.ones(30, 64, device="cuda")), torch.zeros(6, dtype=torch.int64, device="cuda")
    _, _, gw = HeadLoss(weight).step(rows(), labels)
    want = HeadLoss(weight.detach()).step(rows(), labels)[2]
    assert torch.equal(gw, want) and weight.grad is None


def test_clipping_in_place_is_seen_by_autograd():
    """A tensor that a backward still needs may not be scaled in between without an error."""
    saved, other = torch.full((100,), 3.0, device="cuda"), torch.full((100,), 3.0, device="cuda")
    x = torch.ones(100, device="cuda", requires_grad=True)
    y = (x * saved).sum()
    clip_grad_norm_([saved], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y, out = (x * other).sum(), torch.empty(100, device="cuda")
    versions = other._version, out._version
    clip_grad_norm_([other], 1.0, out=[out])
    assert (other._version, out._version) == (versions[0], versions[1] + 1)
    y.backward()
    assert torch.equal(x.grad, other)


def test_clipping_under_inference_mode():
    with torch.inference_mode():
        t = torch.full((100,), 3.0, device="cuda")
        assert abs(float(clip_grad_norm_([t], 1.0)) - 30.0) < 1e-4 and abs(float(t.norm()) - 1.0) < 1e-4
