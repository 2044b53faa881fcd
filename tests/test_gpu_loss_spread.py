"""``HeadLoss`` in float32 where entries of one tensor differ by many orders of magnitude: what a token's loss and gradient are does
not depend on how large the entries of other tokens, of vocabulary rows that play no part, or of channels that meet zeros are.

Bounds: as in ``test_gpu_loss``, but token by token: a logit of token t is off by at most ``e_t = d 2^-23 max_v sum_i |x_ti w_vi|``,
v over the rows that can count (a row whose logit lies 10^4 and more below the others has p = 0 whatever its error). The loss is
off by at most ``2 e_t + 2^-19 (1 + loss)``, D_t by ``p (2 e_t + 2^-19)``; gx_t by ``(2 e_t + 2^-19 + V 2^-23)`` of the sum of its
terms' magnitudes, gw by the sum over t of ``(2 e_t + 2^-19 + n 2^-23)`` of each term's. D as the kernels keep it may also be off by
2^-38 (below which a probability counts as nothing), of which each term of a gradient has its share."""
from __future__ import annotations

import math

import pytest
import torch

from hffn_amd.loss import HeadLoss

pytestmark = pytest.mark.gpu

F32 = torch.float32
FLOOR = 2.0 ** -38


def make(n, d, vocab, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, dtype=F32, device="cuda")  # noqa: E731
    x, weight = normal(n, d), normal(vocab, d) / math.sqrt(d)
    return x, weight, torch.randint(0, vocab, (n,), generator=g, device="cuda")


def check(x, weight, labels, without=None, **options):
    head = HeadLoss(weight, **options)
    losses = head.losses(x, labels).clone().double()
    loss, gx, gw = (t.double() for t in head.step(x, labels))
    rows, w, n = x.double(), weight.double(), len(labels)
    sizes = rows.abs() @ w.abs().T
    if without is not None:
        sizes[:, without] = 0.0
    c = 2 * x.shape[1] * 2.0 ** -23 * sizes.amax(1) + 2.0 ** -19
    log_p = torch.log_softmax(rows @ w.T, 1)
    one = torch.nn.functional.one_hot(labels, len(w)).double()
    want = -(log_p * one).sum(1)
    assert bool(((losses - want).abs() <= c + 2.0 ** -19 * want).all()), float((losses - want).abs().max())
    assert abs(float(loss) - float(want.mean())) <= float(c.mean()) + 2.0 ** -19 * float(want.mean())
    D = (log_p.exp() - one) / n
    most = D.abs() * (c[:, None] + max(len(w), n) * 2.0 ** -23) + FLOOR / n
    for got, wanted, bound in ((gx, D @ w, most @ w.abs()), (gw, D.T @ rows, most.T @ rows.abs())):
        assert bool(((got - wanted).abs() <= bound + 2.0 ** -23 * wanted.abs() + 1e-38).all()), float(((got - wanted).abs() / bound).max())
    return head


@pytest.mark.parametrize("large", (1e5, 1e7, 1e9, 1e20))
@pytest.mark.parametrize("n,d,vocab", [(100, 256, 1000), (70, 37, 900), (300, 130, 700), (1500, 64, 513), (4200, 40, 300)])
def test_one_large_token(n, d, vocab, large):
    """A token whose entries are up to 10^20 times the others': its softmax is one label's, and all others keep their digits."""
    x, weight, labels = make(n, d, vocab, seed=n)
    x[n // 3] *= large
    labels[n // 3] = (x[n // 3].double() @ weight.double().T).argmax()
    check(x, weight, labels)


@pytest.mark.parametrize("large", (1e6, 1e9))
@pytest.mark.parametrize("n,d,vocab", [(100, 256, 1000), (300, 131, 700)])
def test_one_large_vocabulary_row(n, d, vocab, large):
    """A row of the weight that no token comes near: its logits lie far below all others'."""
    x, weight, labels = make(n, d, vocab, seed=n + 1)
    x[:, 5] = x[:, 5].abs() + 0.5
    weight[vocab // 2] = 0.0
    weight[vocab // 2, 5] = -large
    labels[labels == vocab // 2] = 0
    check(x, weight, labels, without=vocab // 2)


@pytest.mark.parametrize("n,d,vocab", [(100, 256, 1000), (200, 36, 2000)])
def test_one_large_channel_that_meets_zeros(n, d, vocab):
    x, weight, labels = make(n, d, vocab, seed=n + 2)
    x[:, 11] *= 1e8
    weight[:, 11] = 0.0
    check(x, weight, labels)


def test_small_rows_keep_their_digits():
    """Most tokens 10^-6 of a few: the small ones' softmax is nearly flat, and its first digits are the weight's."""
    x, weight, labels = make(130, 96, 400, seed=3)
    x[::2] *= 1e-6
    check(x, weight, labels)
    weight[5::7] *= 1e-9
    check(x, weight, labels)


def test_in_pieces():
    x, weight, labels = make(300, 72, 3000, seed=4)
    x[17] *= 1e8
    labels[17] = (x[17].double() @ weight.double().T).argmax()
    one, pieces = HeadLoss(weight), HeadLoss(weight, piece_bytes=1)
    assert pieces._bytes(300, True) < one._bytes(300, True)
    check(x, weight, labels, piece_bytes=1)


def test_masked_and_from_any_workspace():
    """A large token that does not count changes nothing; one that counts gives the same bits again, from any workspace, and calls of
    either kind on one object do not disturb each other."""
    x, weight, labels = make(200, 130, 700, seed=5)
    head = HeadLoss(weight)
    call = lambda rows, at: [t.clone() for t in (head.losses(rows, at), *head.step(rows, at))]  # noqa: E731
    plain = call(x, labels)
    spread = x.clone()
    spread[50] *= 1e9
    masked = labels.clone()
    masked[50] = -100
    without = call(x, masked)
    assert all(torch.equal(a, b) for a, b in zip(call(spread, masked), without))
    first = call(spread, labels)
    head._workspace.fill_(255)
    assert all(torch.equal(a, b) for a, b in zip(call(spread, labels), first))
    head._workspace.fill_(255)
    assert all(torch.equal(a, b) for a, b in zip(call(x, labels), plain))


def test_a_row_that_is_not_finite_stays_in_its_row():
    x, weight, labels = make(150, 64, 500, seed=6)
    head = HeadLoss(weight)
    want = head.losses(x, labels).clone()
    for value in (math.inf, -math.inf, math.nan):
        x[20, 3] = value
        got = head.losses(x, labels)
        live = torch.arange(150, device="cuda") != 20
        assert torch.equal(got[live], want[live]) and not bool(got[20].isfinite())


def test_improbable_rows_keep_what_float32_of_one_keeps():
    """Vocabulary rows whose logits lie 20 to 30 below all others': D is kept to 2^-38, the gradients' share of that is all they
    lose."""
    x, weight, labels = make(200, 64, 600, seed=7)
    x[:, 0] = 1.0
    weight[100:200, 0] -= torch.linspace(20, 30, 100, device="cuda")
    labels[(labels >= 100) & (labels < 200)] = 7
    check(x, weight, labels)
