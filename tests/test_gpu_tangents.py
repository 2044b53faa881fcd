"""A forward-mode tangent that a call would drop is refused, as a row that requires gradients is."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from hffn_amd.embedding import TokenEmbedding
from hffn_amd.loss import HeadLoss
from hffn_amd.norm import ResidualNorm
from hffn_amd.recurrence import GatedRecurrence
from hffn_amd.sampling import sample

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    n, d, vocab = 6, 32, 40
    rows, weight, labels, vector = torch.randn(n, d, device="cuda"), torch.randn(vocab, d, device="cuda"), torch.arange(n, device="cuda"), torch.ones(d, device="cuda")
    table, head, norm, mixer = TokenEmbedding(weight), HeadLoss(weight), ResidualNorm(vector, torch.zeros_like(vector)), GatedRecurrence(torch.zeros_like(vector))
    h, state = mixer.forward(rows, rows)
    calls = [("g", lambda t: table.backward(labels, t)), ("x", lambda t: head.losses(t, labels)), ("x", lambda t: head.step(t, labels)), ("x", lambda t: norm.forward(t)),
             ("x", lambda t: mixer.forward(t, rows)), ("gate", lambda t: mixer.forward(rows, t)), ("gh", lambda t: mixer.backward(rows, rows, h, t)),
             ("x", lambda t: mixer.step(t, rows, torch.zeros(n, d, device="cuda"))), ("state", lambda t: mixer.step(rows, rows, t)), ("logits", lambda t: sample(t, torch.zeros(n, device="cuda")))]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(rows, torch.ones_like(rows))
        for name, call in calls:
            with pytest.raises(ValueError, match=f"{name} carries a forward-mode tangent"):
                call(dual)
            call(forward_ad.unpack_dual(dual).primal.clone())
        with pytest.raises(ValueError, match="state carries"):
            mixer.forward(rows, rows, None, forward_ad.make_dual(state, state))
