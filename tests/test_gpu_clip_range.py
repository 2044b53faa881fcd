"""Norms beyond float32: returned as infinity, while the scaling goes by the float64 norm."""
from __future__ import annotations

import math

import pytest
import torch

from hffn_amd.clip import clip_grad_norm_

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("apart", (False, True))
def test_a_norm_beyond_float32(apart):
    """100 entries of 3e38, norm 3e39: the factor 1 / 3e39 lies below float32's normal numbers and has their 2^-149 as its unit."""
    tensor = torch.full((100,), 3e38, dtype=torch.float32, device="cuda")
    out = torch.empty_like(tensor)
    for limit in (1.0, 1e10, 1e38):
        tensor.fill_(3e38)
        norm = clip_grad_norm_([tensor], limit, out=[out] if apart else None)
        want = float(torch.tensor(3e38, dtype=torch.float32)) * limit / (10 * float(torch.tensor(3e38, dtype=torch.float32)))
        got = (out if apart else tensor).double()
        assert float(norm) == math.inf
        assert bool(((got - want).abs() <= 2.0 ** -22 * want + 2.0 ** -149 * 3e38).all())


def test_infinite_entries():
    tensor = torch.tensor([1.0, math.inf, -2.0], dtype=torch.float32, device="cuda")
    assert float(clip_grad_norm_([tensor], 1.0)) == math.inf
    assert tensor[0] == 0 and bool(tensor[1].isnan()) and tensor[2] == 0
