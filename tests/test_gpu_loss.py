"""``hffn_amd.loss.HeadLoss`` against the definition in float64, through the C ABI, on the GPU.

Bounds. A logit is a float32 sum of d products of operands kept to 22 bits or more: off by at most
``e = d 2^-23 max_tv sum_i |x_ti w_vi|`` (a rounding of at most 2^-23 of the sum of magnitudes per addition). The loss, a
difference of a log-sum and a logit, is then off by at most 2 e and the roundings of exponentials, logarithm and the result
(2^-19 of 1 + |loss|). D = p - onehot is off by at most p (2 e + 2^-19), and, for bfloat16, rounded by 2^-8 of an entry. A
gradient is a float32 sum of K terms of D and the other operand: off by at most (2 e + 2^-19 [+ 2^-8] + K 2^-23) of the sum of
its terms' magnitudes, and rounded to its type (2^-8 of itself for bfloat16). Beside these worst cases the 2-norm of a float32
gradient's error stays below 1e-5 of the gradient's (22-bit operands, roundings that do not conspire)."""
from __future__ import annotations

import math

import pytest
import torch

from hffn_amd.loss import HeadLoss

pytestmark = pytest.mark.gpu

IGNORE = -100
BF16, F32 = torch.bfloat16, torch.float32


def make(n, d, vocab, dtype, ignored=0.0, seed=0, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    x, weight = (std * normal(n, d)).to(dtype), (normal(vocab, d) / math.sqrt(d)).to(dtype)
    labels = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    return x, weight, labels.masked_fill(torch.rand(n, generator=g, device="cuda") < ignored, IGNORE)


def reference(x, weight, labels, reduction="mean", scale=1.0):
    """Losses, loss, gradients and the magnitudes their bounds are taken from, float64."""
    rows = (labels != IGNORE).nonzero()[:, 0]
    x, w, at = x.double()[rows], weight.double(), labels[rows].long()
    n = labels.shape[0]
    losses, gx = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, w.shape[1], dtype=torch.float64, device="cuda")
    gx_size, gw, gw_size, e = gx.clone(), torch.zeros_like(w), torch.zeros_like(w), 0.0
    factor = scale / max(1, len(rows)) if reduction == "mean" else scale
    for part in torch.arange(len(rows), device="cuda").split(512):
        log_p = torch.log_softmax(x[part] @ w.T, 1)
        e = max(e, w.shape[1] * 2.0 ** -23 * float((x[part].abs() @ w.abs().T).max()))
        one = torch.zeros_like(log_p)
        one[torch.arange(len(part), device="cuda"), at[part]] = 1.0
        losses[rows[part]] = -(log_p * one).sum(1)
        p = log_p.exp()
        D = factor * (p - one)
        gx[rows[part]], gx_size[rows[part]] = D @ w, D.abs() @ w.abs()
        gw += D.T @ x[part]
        gw_size += D.abs().T @ x[part].abs()
    loss = losses.sum() * (factor / scale if scale else 0.0)
    return {"losses": losses, "loss": loss, "gx": gx, "gw": gw, "gx_size": gx_size, "gw_size": gw_size, "e": e}


def check_losses(got, ref):
    assert got.dtype == F32
    bound = 2 * ref["e"] + 2.0 ** -19 * (1 + ref["losses"].abs())
    assert bool(((got.double() - ref["losses"]).abs() <= bound).all()), float((got.double() - ref["losses"]).abs().max())


def check_step(got, ref, x, weight, counted):
    loss, gx, gw = got
    dtype = weight.dtype
    assert gx.dtype == gw.dtype == dtype and gx.shape == x.shape and gw.shape == weight.shape and loss.shape == ()
    assert abs(float(loss) - float(ref["loss"])) <= max(1, counted) * (2 * ref["e"] + 2.0 ** -19) + 2.0 ** -19 * abs(float(ref["loss"]))
    rounding = 2.0 ** -8 if dtype == BF16 else 0.0
    for name, value, terms in (("gx", gx, weight.shape[0]), ("gw", gw, max(1, counted))):
        error = (value.double() - ref[name]).abs()
        c = 2 * ref["e"] + 2.0 ** -19 + rounding + terms * 2.0 ** -23
        bound = c * (1 + rounding) * ref[f"{name}_size"] + (rounding + 2.0 ** -24) * ref[name].abs() + 1e-38
        assert bool((error <= bound).all()), (name, float((error / bound).max()))
        if dtype == F32 and float(ref[name].norm()) > 0:
            assert float(error.norm() / ref[name].norm()) <= 1e-5, name


def run_both(n, d, vocab, dtype, ignored=0.0, seed=0, std=1.0):
    x, weight, labels = make(n, d, vocab, dtype, ignored, seed, std)
    head = HeadLoss(weight, ignore_index=IGNORE)
    ref = reference(x, weight, labels)
    check_losses(head.losses(x, labels), ref)
    check_step(head.step(x, labels), ref, x, weight, int((labels != IGNORE).sum()))


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("n,d,vocab", [
    (1, 64, 256), (1, 1, 1), (1, 2048, 3000), (2, 17, 2), (63, 64, 255), (64, 128, 257), (65, 100, 1000), (128, 520, 31),
    (129, 1001, 513), (255, 32, 2999), (9, 104, 100), (50, 1608, 385), (200, 1104, 129), (4097, 72, 640), (5000, 40, 257), (257, 320, 1024), (300, 1104, 777), (700, 96, 512), (1030, 64, 300),
])
def test_sizes(n, d, vocab, dtype):
    run_both(n, d, vocab, dtype)


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("ignored", (0.3, 0.95))
def test_ignored_tokens(ignored, dtype):
    run_both(333, 192, 1500, dtype, ignored=ignored, seed=3)


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_peaked_distributions(dtype):
    run_both(150, 256, 900, dtype, seed=4, std=12.0)


def test_a_vocabulary_in_pieces():
    """More tokens times vocabulary than one piece holds, float32: the pieces' gradients add up."""
    run_both(1300, 64, 50304, F32, ignored=0.02, seed=5)


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("n,vocab", [(7, 1500), (64, 2049), (65, 1500), (300, 2300), (600, 1281)])
def test_small_pieces(n, vocab, dtype):
    """Pieces of 256 and of 512 vocabulary rows: the same losses, the same gradients within their bounds."""
    x, weight, labels = make(n, 136, vocab, dtype, ignored=0.2, seed=14)
    ref = reference(x, weight, labels)
    rows = -(-n // 64) * 64 if n <= 64 else -(-n // 256) * 256
    for piece in (1, 512 * rows * (2 if dtype == BF16 else 4)):
        head = HeadLoss(weight, piece_bytes=piece)
        check_step(head.step(x, labels), ref, x, weight, int((labels != IGNORE).sum()))
        assert head.workspace_bytes() < HeadLoss(weight, max_tokens=n).workspace_bytes() + 64 * rows * 136 * 4 + 512 * rows * 8 + (1 << 16)


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_fewer_tokens_may_need_more_workspace(dtype):
    """Fewer tokens run in fewer, larger pieces: calls of any order on one object, each with the workspace it needs."""
    x, weight, labels = make(900, 64, 2000, dtype, seed=21)
    head = HeadLoss(weight, piece_bytes=800000)
    bytes_of = []
    for n in (300, 65, 64, 900, 700):
        bytes_of.append(head._bytes(n, True))
        check_step(head.step(x[:n], labels[:n]), reference(x[:n], weight, labels[:n]), x[:n], weight, n)
    assert bytes_of[0] < bytes_of[1] or bytes_of[3] < bytes_of[4]


@pytest.mark.parametrize("n,d,vocab", [(1, 1024, 50304), (3, 36, 513), (64, 2052, 700), (33, 30, 90), (17, 96, 66000)])
def test_a_few_float32_tokens(n, d, vocab):
    """Float32 weights read as they are (rows of whole 16-byte pieces) or from a padded copy."""
    run_both(n, d, vocab, F32, seed=15)


@pytest.mark.parametrize("ignored", (0.0, 0.4))
@pytest.mark.parametrize("n,d,vocab", [(1, 4, 16384), (3, 36, 16385), (64, 2052, 16400), (33, 28, 20001), (64, 37, 16400), (65, 36, 33000),
                                       (128, 100, 32768), (128, 100, 32767), (150, 64, 50304), (192, 8, 49152), (193, 8, 65536)])
def test_float32_weights_read_as_they_are(n, d, vocab, ignored):
    """Sizes on both sides of the rule that reads a float32 weight without packing it, with tiles that end anywhere."""
    run_both(n, d, vocab, F32, ignored=ignored, seed=22)


@pytest.mark.parametrize("n,d,vocab", [(1, 1001, 16384), (5, 1, 20000), (130, 33, 40000), (64, 63, 16385), (2, 2, 17000), (40, 96, 16500)])
def test_float32_rows_that_start_anywhere(n, d, vocab):
    """A weight whose rows, or whose first entry, lie on 4-byte boundaries only."""
    x, weight, labels = make(n, d, vocab, F32, ignored=0.1, seed=24)
    at = torch.empty(vocab * d + 1, device="cuda")[1:].view(vocab, d)
    at.copy_(weight)
    ref = reference(x, weight, labels)
    for w in (weight, at):
        head = HeadLoss(w)
        check_losses(head.losses(x, labels), ref)
        check_step(head.step(x, labels), ref, x, w, int((labels != IGNORE).sum()))


@pytest.mark.parametrize("rows,d", [(256, 136), (4096, 136), (16384, 136), (256, 37), (4096, 135)])
def test_pieces_of_a_float32_weight_read_as_it_is(rows, d):
    x, weight, labels = make(50, d, 17000, F32, ignored=0.2, seed=23)
    head = HeadLoss(weight, piece_bytes=rows * 64 * 4)
    check_step(head.step(x, labels), reference(x, weight, labels), x, weight, int((labels != IGNORE).sum()))
    labels.fill_(IGNORE)
    loss, gx, gw = head.step(x, labels)
    assert float(loss) == 0.0 and not gx.any() and not gw.any() and not head.losses(x, labels).any()


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_every_token_ignored(dtype):
    x, weight, _ = make(70, 96, 500, dtype)
    labels = torch.full((70,), IGNORE, device="cuda")
    x[3] = float("nan")
    head = HeadLoss(weight)
    assert torch.equal(head.losses(x, labels), torch.zeros(70, device="cuda"))
    loss, gx, gw = head.step(x, labels)
    assert float(loss) == 0.0 and not bool(gx.any()) and not bool(gw.any())


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_no_tokens(dtype):
    x, weight, labels = make(0, 96, 500, dtype)
    head = HeadLoss(weight)
    assert head.losses(x, labels).shape == (0,)
    loss, gx, gw = head.step(x, labels)
    assert float(loss) == 0.0 and gx.shape == (0, 96) and not bool(gw.any())


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_values_of_ignored_rows_do_not_matter(dtype):
    x, weight, labels = make(200, 130, 700, dtype, ignored=0.4, seed=6)
    head = HeadLoss(weight)
    losses = head.losses(x, labels).clone()
    loss, gx, gw = (t.clone() for t in head.step(x, labels))
    masked = (labels == IGNORE).nonzero()[:, 0]
    x[masked[::3]], x[masked[1::3]], x[masked[2::3]] = float("nan"), float("inf"), torch.finfo(dtype).min
    assert torch.equal(head.losses(x, labels), losses)
    for a, b in zip(head.step(x, labels), (loss, gx, gw)):
        assert torch.equal(a, b)
    assert not bool(gx[masked].any())


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_a_label_outside_the_vocabulary_is_not_a_number(dtype):
    for outside in (-1, 400, 1 << 40):
        x, weight, labels = make(90, 64, 400, dtype)
        labels[17] = outside
        head = HeadLoss(weight)
        losses = head.losses(x, labels)
        assert bool(losses[17].isnan()) and int(losses.isnan().sum()) == 1
        loss, gx, gw = head.step(x, labels)
        assert bool(loss.isnan()) and bool(gx.isnan().all()) and bool(gw.isnan().all())


def test_weight_rows_of_zero_and_of_other_scales():
    """Rows of zeros (padding of a vocabulary) and rows 1e-9 and 1e3 times the others get their gradients all the same."""
    x, weight, labels = make(140, 160, 600, F32, seed=7)
    weight[::7] = 0.0
    weight[1::7] *= 1e-9
    weight[2::7] *= 1e3
    x[5] *= 1e-6
    head = HeadLoss(weight)
    ref = reference(x, weight, labels)
    check_losses(head.losses(x, labels), ref)
    check_step(head.step(x, labels), ref, x, weight, 140)


@pytest.mark.parametrize("which", ("weight", "x", "both", "first rows"))
def test_lone_large_entries(which):
    """One entry 1e4 times the others in float32 tensors, wherever it lies, and tensors whose other rows are zeros."""
    x, weight, labels = make(300, 160, 2000, F32, ignored=0.1, seed=13)
    x *= 1e-2
    if which in ("weight", "both"):
        weight[1234, 77] = 1e4 * 0.08
    if which in ("x", "both"):
        x[int((labels != IGNORE).nonzero()[37]), 131] = 1e4 * 1e-2
    if which == "first rows":
        weight[3:], x[5:] = 0.0, 0.0
    head = HeadLoss(weight)
    ref = reference(x, weight, labels)
    check_losses(head.losses(x, labels), ref)
    check_step(head.step(x, labels), ref, x, weight, int((labels != IGNORE).sum()))


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_zero_weight_and_zero_rows(dtype):
    x, weight, labels = make(66, 64, 300, dtype)
    for a, b in ((x, torch.zeros_like(weight)), (torch.zeros_like(x), weight)):
        head = HeadLoss(b)
        ref = reference(a, b, labels)
        check_losses(head.losses(a, labels), ref)
        check_step(head.step(a, labels), ref, a, b, 66)


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_strides_label_types_and_alignment(dtype):
    x, weight, labels = make(120, 96, 640, dtype, ignored=0.1, seed=8)
    head = HeadLoss(weight)
    want = [t.clone() for t in (head.losses(x, labels), *head.step(x, labels))]
    wide = torch.zeros(120, 3, 96, dtype=dtype, device="cuda")
    wide[:, 1] = x
    shifted = torch.zeros(120 * 97 + 1, dtype=dtype, device="cuda")[1:].view(120, 97)[:, :96]
    shifted.copy_(x)
    pairs = torch.stack([labels, labels + 1], 1)[:, 0]
    odd = torch.zeros(weight.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(weight)
    odd.copy_(weight)
    for rows, at, h in ((wide[:, 1], labels, head), (shifted, labels, head), (x.T.contiguous().T, labels, head), (x, labels.int(), head),
                        (x, pairs, head), (x, labels, HeadLoss(odd))):
        for a, b in zip((h.losses(rows, at), *h.step(rows, at)), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_repeats_bit_for_bit_and_from_any_workspace(dtype):
    """The same bits again, after larger and smaller calls, and with the workspace full of NaN."""
    x, weight, labels = make(300, 200, 1111, dtype, ignored=0.2, seed=9)
    head = HeadLoss(weight, max_tokens=300)
    want = [t.clone() for t in (head.losses(x, labels), *head.step(x, labels))]
    head.step(x[:7], labels[:7])
    head._workspace.fill_(255)
    head._gx.fill_(float("nan"))
    head.grad.fill_(float("nan"))
    for a, b in zip((head.losses(x, labels), *head.step(x, labels)), want):
        assert torch.equal(a, b)


def test_reduction_and_scale():
    x, weight, labels = make(77, 64, 500, F32, ignored=0.3, seed=10)
    ref = reference(x, weight, labels, "sum", 0.25)
    check_step(HeadLoss(weight, reduction="sum").step(x, labels, scale=0.25), ref, x, weight, int((labels != IGNORE).sum()))


def test_gradients_against_differences():
    """Central differences of the kernel's own loss along random directions: off by h^2 of third derivatives (h = 1e-2) and
    by the loss's rounding over h (2^-19 3 / 1e-2 for a loss of about 7)."""
    x, weight, labels = make(40, 48, 800, F32, ignored=0.2, seed=11)
    _, gx, gw = (t.clone() for t in HeadLoss(weight).step(x, labels))
    counted = (labels != IGNORE).sum()
    h = 1e-2
    for seed in range(3):
        g = torch.Generator("cuda").manual_seed(seed)
        dx, dw = torch.randn(x.shape, generator=g, device="cuda"), torch.randn(weight.shape, generator=g, device="cuda")
        ends = [HeadLoss(weight + s * h * dw).losses(x + s * h * dx, labels).double().sum() / counted for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * h)
        along = (gx.double() * dx).sum() + (gw.double() * dw).sum()
        assert abs(float(slope - along)) <= 2e-2 * max(1.0, abs(float(along)))


def test_replayed_from_a_graph(device):
    """Captured once, replayed with other inputs, eager calls between the replays."""
    x, weight, labels = make(96, 128, 1000, BF16, ignored=0.1, seed=12)
    other = HeadLoss(weight)
    head = HeadLoss(weight, max_tokens=96)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        head.step(x, labels)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = head.step(x, labels)
    for seed in range(3):
        x2, _, labels2 = make(96, 128, 1000, BF16, ignored=0.1, seed=20 + seed)
        x.copy_(x2)
        labels.copy_(labels2)
        graph.replay()
        want = other.step(x, labels)
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)


def test_refusals(device):
    x, weight, labels = make(8, 64, 100, F32)
    head = HeadLoss(weight)
    for bad, at, match in ((x.bfloat16(), labels, "x:"), (x[:, :32], labels, "x:"), (x[0], labels, "x:"), (x.cpu(), labels, "x:"),
                           (x, labels[:5], "labels"), (x, labels.float(), "labels"), (x, labels.cpu(), "labels"), (x, labels[None], "labels")):
        for call in (head.losses, head.step):
            with pytest.raises(ValueError, match=match):
                call(bad, at)
    for make_head, match in ((lambda: HeadLoss(weight.T), "contiguous"), (lambda: HeadLoss(weight[:0]), "non-empty"),
                             (lambda: HeadLoss(weight.half()), "float32 or bfloat16"), (lambda: HeadLoss(weight, reduction="none"), "reduction"),
                             (lambda: HeadLoss(weight, max_tokens=0), "N=0"), (lambda: HeadLoss(weight, piece_bytes=0), "piece_bytes"), (lambda: HeadLoss(weight[0]), "contiguous")):
        with pytest.raises(ValueError, match=match):
            make_head()
