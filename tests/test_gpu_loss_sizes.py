"""``HeadLoss`` at sizes where its kernels take other ways than at those of ``test_gpu_loss``, whose oracle and bounds these tests
share."""
from __future__ import annotations

import math

import pytest
import torch

from hffn_amd.loss import HeadLoss
from test_gpu_loss import IGNORE, check_losses, check_step, make, reference

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("n,dtype", [(256, BF16), (128, F32)])
def test_a_piece_whose_rows_pass_32_bits(n, dtype):
    """8.5 million vocabulary rows asked for as one piece: the last tokens of a tile lie 4 GB after its first.

    gx against float64 at tokens at both ends of the tile. Its sum over the vocabulary is taken in 64 parts or more, so that
    (beside test_gpu_loss's terms) 2^-23 of vocab / 64 terms' magnitudes bound it."""
    vocab, d = 8_500_001, 16
    g = torch.Generator("cuda").manual_seed(n)
    x = torch.randn(n, d, generator=g, dtype=F32, device="cuda").to(dtype)
    weight = (torch.randn(vocab, d, generator=g, dtype=F32, device="cuda") / math.sqrt(d)).to(dtype)
    labels = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    head = HeadLoss(weight, piece_bytes=16 << 30)
    _, gx, gw = head.step(x, labels)
    rounding = 2.0 ** -8 if dtype == BF16 else 0.0
    rows, w = x.double(), weight.double()
    lse = torch.stack([torch.logsumexp(rows @ part.T, 1) for part in w.split(1 << 19)]).logsumexp(0)
    e = d * 2.0 ** -23 * max(float((rows.abs() @ part.abs().T).max()) for part in w.split(1 << 19))

    def within(got, want, size, terms):
        bound = (2 * e + 2.0 ** -19 + rounding + terms * 2.0 ** -23) * (1 + rounding) * size + (rounding + 2.0 ** -24) * want.abs()
        return bool(((got.double() - want).abs() <= bound).all())

    for t in (0, 1, n // 2 - 1, n // 2, n - 2, n - 1):
        D = torch.exp(w @ rows[t] - lse[t])
        D[labels[t]] -= 1.0
        D /= n
        assert within(gx[t], D @ w, D.abs() @ w.abs(), vocab / 64), t
    at = torch.cat([labels, torch.arange(0, vocab, 9973, device="cuda"), torch.tensor([vocab - 1], device="cuda")])
    D = (torch.exp(rows @ w[at].T - lse[:, None]) - (labels[:, None] == at).double()) / n
    assert within(gw[at], D.T @ rows, D.abs().T @ rows.abs(), n)


def check(x, weight, labels, **options):
    """Losses, loss and gradients against float64; and the loss against the float64 mean of the losses, which it is to a float32
    rounding (2^-24) of a float64 sum."""
    head = HeadLoss(weight, ignore_index=IGNORE, **options)
    ref = reference(x, weight, labels)
    losses = head.losses(x, labels).clone()
    check_losses(losses, ref)
    counted = int((labels != IGNORE).sum())
    got = head.step(x, labels)
    check_step(got, ref, x, weight, counted)
    mean = float(losses.double().sum()) / max(1, counted)
    assert abs(float(got[0]) - mean) <= 2.0 ** -23 * abs(mean)
    assert abs(float(got[0]) - float(ref["loss"])) <= 2 * ref["e"] + 2.0 ** -19 * (1 + abs(float(ref["loss"])))


BLOCKS, XCDS = 256, 8


def shapes(tiles):
    """How a launch of 256 x 256 tiles takes them: an XCD's share of 32 blocks, a tile each and again; a last round that fills at
    most half (a quarter) of the blocks goes as halves (quarters)."""
    kinds, blocks = set(), BLOCKS // XCDS
    for share in {tiles * (k + 1) // XCDS - tiles * k // XCDS for k in range(XCDS)}:
        rest = share % blocks
        cut = rest != 0 and 2 * rest <= blocks
        if share - (rest if cut else 0) > 0:
            kinds.add("whole")
        if share - (rest if cut else 0) > blocks:
            kinds.add("whole again")
        if cut:
            kinds.add(("halves" if 4 * rest > blocks else "quarters") + (" after whole" if share > blocks else ""))
    return kinds


def products(n, counted, d, vocab):
    """The tiles of the three products of a bfloat16 step in one piece, above 64 tokens: logits, gx, gw."""
    up = lambda a, b: -(-a // b)  # noqa: E731
    live, rows, across = up(counted, 256), up(vocab, 256), up(d, 256)
    splits = min(up(BLOCKS, across * up(n, 256)), max(1, rows * 4 // 8))
    return rows * live, across * live * splits, across * rows


LARGE = [
    (1024, 72, 36 * 256 - 5, 0.0, ({"whole"}, {"halves"}, {"quarters"})),
    (1100, 320, 60 * 256, 0.0, ({"quarters after whole", "whole"}, {"quarters after whole", "whole"}, {"halves"})),
    (1000, 600, 88 * 256 - 100, 0.0, ({"halves after whole", "whole"}, {"quarters after whole", "whole"}, {"quarters after whole", "whole"})),
    (2048, 300, 200 * 256, 0.0, ({"quarters after whole", "whole", "whole again"}, {"whole"}, {"whole", "whole again"})),
    (4100, 72, 70 * 256 + 1, 0.0, ({"whole", "whole again"}, {"quarters after whole", "whole"}, {"halves", "quarters"})),
    (13056, 1280, 1100, 0.0, ({"whole"}, {"whole", "whole again"}, {"quarters"})),
    (1500, 264, 21000, 0.5, None),
    (4100, 72, 70 * 256 + 1, 0.1, None),
    (777, 1104, 32003, 0.3, None),
]


@pytest.mark.parametrize("n,d,vocab,ignored,kinds", LARGE)
def test_whole_tiles_halves_and_several_a_block(n, d, vocab, ignored, kinds):
    """bfloat16 calls whose products run whole 256 x 256 tiles, several a block one after the other, and last rounds of each cut."""
    x, weight, labels = make(n, d, vocab, BF16, ignored, seed=n)
    if kinds is not None:
        assert tuple(shapes(tiles) for tiles in products(n, int((labels != IGNORE).sum()), d, vocab)) == kinds
    check(x, weight, labels)


@pytest.mark.parametrize("counted", (255, 256, 257, 264, 520))
def test_counted_tokens_around_a_tile(counted):
    x, weight, labels = make(777, 136, 30000, BF16, seed=counted)
    labels[torch.randperm(777, generator=torch.Generator("cuda").manual_seed(counted), device="cuda")[counted:]] = IGNORE
    check(x, weight, labels)


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("rows", (20 * 256, 40 * 256))
def test_pieces_of_many_tiles(rows, dtype):
    """Several pieces of a large vocabulary, the last one shorter: every product of every piece over many tiles."""
    n = 1300
    x, weight, labels = make(n, 264, 90 * 256 + 77, dtype, 0.05, seed=rows)
    size = rows * -(-n // 256) * 256 * (2 if dtype == BF16 else 4)
    one, pieces = HeadLoss(weight), HeadLoss(weight, piece_bytes=size)
    assert pieces._bytes(n, True) < one._bytes(n, True)
    check(x, weight, labels, piece_bytes=size)


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("n", (1, 33, 64))
def test_few_tokens_with_several_tiles_a_block(n, dtype):
    """gw of a few tokens: 705 tiles (bfloat16) of 128 x 128 on 512 blocks."""
    x, weight, labels = make(n, 300, 30001, dtype, seed=n)
    check(x, weight, labels)


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("n,d,vocab", [(2, 32768, 300), (70, 32768, 513), (3, 20001, 400), (65, 20001, 300), (2, 9001, 16500)])
def test_the_widest_rows(n, d, vocab, dtype):
    x, weight, labels = make(n, d, vocab, dtype, seed=d)
    check(x, weight, labels)
