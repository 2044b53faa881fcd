"""``hffn_amd.norm.ResidualNorm`` against the definition in float64 (gradients: against autograd of it, and differences).

Bounds. Row sums of d float32 terms are off by at most d 2^-23 of their terms' magnitudes; the terms here are of one size, so
statistics are off by about that share, and an output by a few times it of the row's largest magnitude: 16 d 2^-23 for d up to a
few hundred, where random roundings leave far less for longer rows (sqrt(d)): ``c = 64 sqrt(d) 2^-23`` of the row's largest
output. Column sums over n rows add n 2^-23 of the terms' magnitudes. bfloat16 rounds outputs by 2^-8."""
from __future__ import annotations

import math

import pytest
import torch

from hffn_amd.norm import ResidualNorm

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-5


def make(n, d, dtype, kind, post, gate, bias=True, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    p = {"weight": 1 + 0.2 * normal(d)}
    if kind == "layer" and bias:
        p["bias"] = 0.3 * normal(d)
    if gate:
        p["gate"] = 1 + 0.3 * normal(d)
    if post:
        p["post_weight"] = 1 + 0.2 * normal(d)
        if kind == "layer" and bias:
            p["post_bias"] = 0.3 * normal(d)
    rows = {name: (std * normal(n, d) + mean).to(dtype) for name, std, mean in
            (("x", 1.5, 0.3), ("f", 0.7, -0.2), ("gr", 0.4, 0.0), ("gh", 0.5, 0.1))}
    return p, rows


def boundary(p, kind, scale=0.7, eps=EPS):
    return ResidualNorm(p["weight"], p.get("bias"), gate=p.get("gate"), post_weight=p.get("post_weight"), post_bias=p.get("post_bias"),
                        scale=scale, kind=kind, eps=eps)


def norm64(v, weight, bias, kind, eps=EPS):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v / (v.square().mean(1, keepdim=True) + eps).sqrt() * weight
    return v if bias is None else v + bias


def branch64(f, p, kind, scale=0.7, eps=EPS):
    u = norm64(f, p["post_weight"], p.get("post_bias"), kind, eps) if "post_weight" in p else f
    return scale * (u * p["gate"] if "gate" in p else u)


def close(got, want, d, dtype, name, more=0.0):
    assert got.dtype == dtype and got.shape == want.shape
    rounding = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    c = 64 * math.sqrt(d) * 2.0 ** -23
    most = want.abs().amax(1, keepdim=True) if want.dim() == 2 else want.abs().max()
    error = (got.double() - want).abs()
    bound = rounding * want.abs() + c * (most + 1) + more
    assert bool((error <= bound).all()), (name, float((error / bound).max()))


def check(n, d, dtype, kind, post, gate, bias=True, seed=0, mutate=None, eps=EPS):
    p, rows = make(n, d, dtype, kind, post, gate, bias, seed)
    if mutate:
        mutate(rows)
    b = boundary(p, kind, eps=eps)
    q = {name: t.double().requires_grad_() for name, t in p.items()}
    x, f, gr, gh = (rows[name].double() for name in ("x", "f", "gr", "gh"))
    r, h = b.forward(rows["x"], rows["f"])
    with torch.no_grad():
        want_r = x + branch64(f, q, kind, eps=eps)
        close(r, want_r, d, dtype, "r")
        close(h, norm64(want_r, q["weight"], q.get("bias"), kind, eps), d, dtype, "h")
    gx, gf = b.backward(r, rows["f"], rows["gr"], rows["gh"])
    r64, f64 = r.double().requires_grad_(), f.requires_grad_()
    first = [name for name in ("weight", "bias") if name in q]
    want_gx, *want_first = torch.autograd.grad(norm64(r64, q["weight"], q.get("bias"), kind, eps), [r64, *(q[k] for k in first)], gh)
    want_gx = want_gx + gr
    rest = [name for name in ("gate", "post_weight", "post_bias") if name in q]
    want_gf, *want_rest = torch.autograd.grad(branch64(f64, q, kind, eps=eps), [f64, *(q[k] for k in rest)], want_gx)
    close(gx, want_gx, d, dtype, "gx")
    close(gf, want_gf, d, dtype, "gf")
    gradients = b.gradients()
    assert set(gradients) == set(first + rest) == set(p)
    for name, want in zip(first + rest, want_first + want_rest):
        # terms of up to about 5 x 5 each, n of them: n 2^-23 of their sum of magnitudes at most
        close(gradients[name], want, d, F32, name, more=n * n * 2.0 ** -23 * 0.5 + n * 64 * math.sqrt(d) * 2.0 ** -23)


KINDS = [("layer", False, False), ("layer", True, True), ("layer", True, False), ("rms", False, True), ("rms", True, True), ("rms", False, False)]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("kind,post,gate", KINDS)
@pytest.mark.parametrize("n,d", [(1, 1024), (3, 64), (37, 1001), (130, 512), (33, 2560)])
def test_sizes(n, d, kind, post, gate, dtype):
    check(n, d, dtype, kind, post, gate)


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("n,d", [(5, 1), (2, 2), (4, 7), (9, 1024), (9, 1025), (9, 1032), (5, 4096), (5, 4100), (3, 4097), (3, 8192), (2, 16384), (2, 16383),
                                 (2100, 64), (1500, 1040)])
def test_widths_and_long_batches(n, d, dtype):
    if d <= 2:  # a layer norm of one or two entries leaves nothing or signs only: RMS
        check(n, d, dtype, "rms", True, True, eps=1e-2)
    else:
        check(n, d, dtype, "layer", True, True, seed=1)


def test_layer_norms_without_bias():
    check(20, 96, F32, "layer", True, True, bias=False)


@pytest.mark.parametrize("kind", ("layer", "rms"))
def test_rows_of_one_value(kind):
    """Rows without variance, and rows of zeros: eps alone is under the root."""
    def mutate(rows):
        rows["x"][::2], rows["f"][::2] = 3.0, 0.0
        rows["x"][1::4], rows["f"][1::4] = 0.0, 0.0
    check(16, 128, F32, kind, False, True, mutate=mutate, eps=1e-2)


@pytest.mark.parametrize("dtype", (F32, BF16))
def test_norm_alone(dtype):
    """Without a block before it: r is x, and the gradient through h may be all there is."""
    p, rows = make(50, 200, dtype, "layer", False, False)
    b = boundary(p, "layer")
    r, h = b.forward(rows["x"])
    assert r is rows["x"]
    x = rows["x"].double().requires_grad_()
    want = norm64(x, p["weight"].double(), p["bias"].double(), "layer")
    close(h, want.detach(), 200, dtype, "h")
    (g,) = torch.autograd.grad(want, x, rows["gh"].double())
    gx, gf = b.backward(r, None, None, rows["gh"])
    assert gf is None
    close(gx, g, 200, dtype, "gx")
    gx, _ = b.backward(r, None, rows["gr"], rows["gh"])
    close(gx, g + rows["gr"].double(), 200, dtype, "gx with gr")


def test_no_rows():
    p, rows = make(0, 64, F32, "layer", True, True)
    b = boundary(p, "layer")
    r, h = b.forward(rows["x"], rows["f"])
    gx, gf = b.backward(r, rows["f"], rows["gr"], rows["gh"])
    assert r.shape == h.shape == gx.shape == gf.shape == (0, 64)
    assert all(not bool(g.any()) for g in b.gradients().values()) and set(b.gradients()) == set(p)


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("d", (128, 72, 1024))
def test_strides_and_alignment(d, dtype):
    """Rows apart, rows that start off a 16-byte boundary, transposed and broadcast ones: the bits of contiguous rows up to the
    order of a row's sums, and of aligned strided rows exactly."""
    p, rows = make(40, d, dtype, "layer", True, True, seed=2)
    b = boundary(p, "layer")
    want = [t.clone() for t in (*b.forward(rows["x"], rows["f"]), *b.backward(rows["x"], rows["f"], rows["gr"], rows["gh"]))]

    def spread(t, pad, start):
        out = torch.zeros(t.shape[0] * (d + pad) + start, dtype=dtype, device="cuda")[start:].view(t.shape[0], d + pad)[:, :d]
        out.copy_(t)
        return out

    for change, exact in ((lambda t: spread(t, 16, 0), True), (lambda t: spread(t, 3, 1), False), (lambda t: t.T.contiguous().T, True)):
        s = {name: change(t) for name, t in rows.items()}
        got = (*b.forward(s["x"], s["f"]), *b.backward(s["x"], s["f"], s["gr"], s["gh"]))
        for name, a, w in zip(("r", "h", "gx", "gf"), got, want):
            if exact:
                assert torch.equal(a, w), name
            else:
                close(a, w.double(), d, dtype, name, more=2.0 ** -8 * float(w.abs().max()) if dtype == BF16 else 0.0)
    one = rows["gr"][:1].expand(40, d)
    assert torch.equal(b.backward(rows["x"], rows["f"], one, rows["gh"])[0], b.backward(rows["x"], rows["f"], one.contiguous(), rows["gh"])[0])


def test_repeats_bit_for_bit():
    p, rows = make(1000, 768, BF16, "layer", True, True, seed=3)
    b = boundary(p, "layer")
    first = [t.clone() for t in (*b.backward(rows["x"], rows["f"], rows["gr"], rows["gh"]), *b.gradients().values())]
    b.backward(rows["x"][:5], rows["f"][:5], rows["gr"][:5], rows["gh"][:5])
    again = (*b.backward(rows["x"], rows["f"], rows["gr"], rows["gh"]), *b.gradients().values())
    assert all(torch.equal(a, c) for a, c in zip(first, again))


def test_a_row_of_nan_stays_in_its_row():
    p, rows = make(12, 256, F32, "layer", True, True, seed=4)
    b = boundary(p, "layer")
    want = b.forward(rows["x"], rows["f"])
    rows["x"][7, 3], rows["f"][9, 100] = float("nan"), float("inf")
    r, h = b.forward(rows["x"], rows["f"])
    live = [k for k in range(12) if k not in (7, 9)]
    assert torch.equal(r[live], want[0][live]) and torch.equal(h[live], want[1][live])
    assert bool(h[[7, 9]].isnan().all())


@pytest.mark.parametrize("kind", ("layer", "rms"))
def test_gradients_against_differences(kind):
    """Central differences of sum(gr r + gh h) from the kernel's own forward, summed in float64: h^2 and the outputs' rounding
    (2^-22 of a few thousand terms) over h, at h = 1e-2."""
    p, rows = make(30, 96, F32, kind, True, True, seed=5)
    scalar = lambda q, x, f: sum(float((a.double() * g.double()).sum()) for a, g in zip(  # noqa: E731
        boundary(q, kind).forward(x, f), (rows["gr"], rows["gh"])))
    b = boundary(p, kind)
    r, _ = b.forward(rows["x"], rows["f"])
    gx, gf = b.backward(r, rows["f"], rows["gr"], rows["gh"])
    h = 1e-2
    for seed in range(3):
        g = torch.Generator("cuda").manual_seed(seed)
        dx, df = (torch.randn(30, 96, generator=g, device="cuda") for _ in range(2))
        dp = {name: torch.randn(96, generator=g, device="cuda") for name in p}
        ends = [scalar({k: t + s * h * dp[k] for k, t in p.items()}, rows["x"] + s * h * dx, rows["f"] + s * h * df) for s in (1, -1)]
        along = float((gx.double() * dx).sum() + (gf.double() * df).sum()) + sum(float((b.gradients()[k].double() * dp[k]).sum()) for k in p)
        assert abs((ends[0] - ends[1]) / (2 * h) - along) <= 1e-2 * (abs(along) + math.sqrt(30 * 96))


def test_replayed_from_a_graph(device):
    p, rows = make(64, 512, BF16, "rms", True, True, seed=6)
    b, other = boundary(p, "rms"), boundary(p, "rms")

    def both(c):
        r, h = c.forward(rows["x"], rows["f"])
        return (r, h, *c.backward(r, rows["f"], rows["gr"], rows["gh"]), *c.gradients().values())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both(b)
    for seed in range(3):
        _, fresh = make(64, 512, BF16, "rms", True, True, seed=30 + seed)
        for name, t in rows.items():
            t.copy_(fresh[name])
        graph.replay()
        want = both(other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(captured, want))


def test_refusals(device):
    p, rows = make(6, 64, F32, "layer", True, True)
    b, x, f = boundary(p, "layer"), rows["x"], rows["f"]
    for call, match in ((lambda: b.forward(x), "needs f"), (lambda: b.forward(x, f.bfloat16()), "f:"), (lambda: b.forward(x, f[:3]), "3 rows"),
                        (lambda: b.forward(x[:, :32], f), "x:"), (lambda: b.forward(x.cpu(), f), "x:"), (lambda: b.forward(x.half(), f), "float32 or bfloat16"),
                        (lambda: b.backward(x, None, x, x), "needs f"), (lambda: b.backward(x, f, x, x[:2]), "2 rows"),
                        (lambda: b.backward(x, f, x.bfloat16(), x), "gr:"),
                        (lambda: ResidualNorm(p["weight"], p["bias"], kind="rms"), "no bias"), (lambda: ResidualNorm(p["weight"], kind="batch"), "kind"),
                        (lambda: ResidualNorm(p["weight"], post_bias=p["bias"]), "post_weight"), (lambda: ResidualNorm(p["weight"].bfloat16()), "weight"),
                        (lambda: ResidualNorm(p["weight"], gate=p["gate"][:5]), "gate"), (lambda: ResidualNorm(p["weight"], eps=-1.0), "eps"),
                        (lambda: ResidualNorm(torch.ones(16385, device=device)), "channels")):
        with pytest.raises(ValueError, match=match):
            call()
