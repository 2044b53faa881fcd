"""The gradients of a bfloat16 step of a few tokens, in which a single entry of D = softmax - onehot may be all there is: what they lose
is their own rounding.

Bounds: D is held to 2^-16 of an entry, so that a gradient is off by ``2 e + 2^-19 + 2^-16 + terms 2^-23`` of the sum of its terms'
magnitudes (``test_gpu_loss``), and by 2^-8 of itself for its rounding. The 2-norm of the error is that of the exact gradients' own
rounding to bfloat16, to 1.1 times."""
from __future__ import annotations

import math

import pytest
import torch

from hffn_amd.loss import HeadLoss
from test_gpu_loss import IGNORE, make, reference

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def check(x, weight, labels, **options):
    ref = reference(x, weight, labels)
    _, gx, gw = HeadLoss(weight, **options).step(x, labels)
    for name, got, terms in (("gx", gx, weight.shape[0]), ("gw", gw, int((labels != IGNORE).sum()))):
        want, size = ref[name], ref[f"{name}_size"]
        error = (got.double() - want).abs()
        c = 2 * ref["e"] + 2.0 ** -19 + 2.0 ** -16 + terms * 2.0 ** -23
        assert bool((error <= c * (1 + 2.0 ** -8) * size + 2.0 ** -8 * want.abs() + 1e-38).all()), name
        assert float(error.norm()) <= 1.1 * float((want.to(BF16).double() - want).norm()) + 1e-30, name


def with_probability(p, d, vocab, seed):
    """A token whose label has that probability: the label's weight row is as long along x as that takes."""
    x, weight, labels = make(1, d, vocab, BF16, seed=seed)
    row = x[0].double()
    rest = torch.logsumexp((weight.double() @ row)[torch.arange(vocab, device="cuda") != labels[0]], 0)
    logit = rest + math.log(p / (1 - p))
    weight[labels[0]] = (row * (logit / row.square().sum())).to(BF16)
    return x, weight, labels


@pytest.mark.parametrize("p", (0.001, 0.2490, 0.4980, 0.7480, 0.8740))
@pytest.mark.parametrize("d,vocab", [(256, 2000), (1024, 50304), (37, 700)])
def test_one_token_whose_label_is_as_probable_as_that(p, d, vocab):
    """1 - p just above a power of two: there, a bfloat16 D is off by up to 2^-8."""
    for seed in range(4):
        check(*with_probability(p, d, vocab, seed))


@pytest.mark.parametrize("n,d,vocab,ignored", [(2, 64, 257, 0.0), (5, 104, 1000, 0.0), (33, 300, 30001, 0.0), (64, 1001, 5000, 0.0), (64, 2048, 3000, 0.9), (17, 136, 1500, 0.3)])
def test_a_few_tokens(n, d, vocab, ignored):
    x, weight, labels = make(n, d, vocab, BF16, ignored, seed=n)
    labels[0] = 1
    check(x, weight, labels)
    check(x, weight, labels, piece_bytes=1)
