"""``GatedRecurrence`` where infinities, NaN and the ends of float32 pass through: (1 - z) h + v by its definition.

The definition runs on the host in float64, 1 - z as sigmoid(-a), which is never zero here (|a| below 700). What is not finite has to be the same
infinity or a NaN as well, everything else the bits of a run without what was planted: it lies in other channels or sequences, or
before the plant. Where |a| exceeds 80, z or 1 - z is below 2^-115 and it, or its product with the rest of a gradient's formula, may be
zero in float32: there an infinite G gives an infinity or, as 0 inf, a NaN. Values at the ends of float32 are compared within four roundings
of 2^-24 a row (the factor's and the sigmoid's, the product's, the sum's), of which half goes on to the next: eight in all."""
from __future__ import annotations

import math

import pytest
import torch

from hffn_amd.recurrence import KINDS, GatedRecurrence

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
BOUNDS = [0, 700, 700, 701, 1500]
N, S, INF = BOUNDS[-1], len(BOUNDS) - 1, math.inf


def draw(*shape, dtype=F32, seed=0, std=1.0):
    return (std * torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), dtype=F32, device="cuda")).to(dtype)


def inputs(d, dtype, seed=0):
    """x, gate (both signs, some far out), bias, state, bounds."""
    gate = draw(N, d, dtype=dtype, seed=seed + 1, std=3.0)
    gate[::97] *= 20.0
    return draw(N, d, dtype=dtype, seed=seed), gate, draw(d, seed=seed + 2), draw(S, d, seed=seed + 3), torch.tensor(BOUNDS, device="cuda")


def gates(gate, bias):
    a = (gate.double() + bias.double()).cpu()
    return torch.sigmoid(a), torch.sigmoid(-a)


def input_of(kind, z, c):
    """dv/dx and its derivative by z."""
    if kind == "tied":
        return z, torch.ones_like(z)
    if kind == "free":
        return torch.ones_like(z), torch.zeros_like(z)
    root = (z * (1 + c)).sqrt()
    return root, c / root


def forward64(kind, x, gate, bias, state):
    z, c = gates(gate, bias)
    v = input_of(kind, z, c)[0] * x.double().cpu()
    h, last = torch.empty_like(v), state.double().cpu().clone()
    for s, (begin, end) in enumerate(zip(BOUNDS, BOUNDS[1:])):
        for t in range(begin, end):
            last[s] = h[t] = c[t] * last[s] + v[t]
    return h, last


def backward64(kind, x, gate, bias, h, gh, state, glast):
    """h as the forward stored it."""
    z, c = gates(gate, bias)
    dx, dz = input_of(kind, z, c)
    x, h, gh = x.double().cpu(), h.double().cpu(), gh.double().cpu()
    gx, ggate, gstate = torch.empty_like(x), torch.empty_like(x), glast.double().cpu().clone()
    for s, (begin, end) in enumerate(zip(BOUNDS, BOUNDS[1:])):
        for t in reversed(range(begin, end)):
            whole = gh[t] + gstate[s]
            before = h[t - 1] if t > begin else state[s].double().cpu()
            gx[t] = whole * dx[t]
            ggate[t] = whole * (dz[t] * x[t] - before) * z[t] * c[t]
            gstate[s] = c[t] * whole
    return gx, ggate, gstate


def compare(got, want, clean, either=None):
    """What is not finite: as in `want` (in `either`: not finite). Everything else: as in `clean`."""
    got, clean = got.cpu(), clean.cpu()
    plain = want.isfinite()
    assert bool((got.isfinite() == plain).all())
    assert torch.equal(got[plain], clean[plain])
    told = ~plain if either is None else ~plain & ~either
    odd = got[told].double(), want[told]
    assert bool(((odd[0] == odd[1]) | (odd[0].isnan() & odd[1].isnan())).all())
    return int((~plain).sum())


PLANTS = [("state", 0, INF), ("state", 3, -INF), ("state", 2, INF), ("state", 1, INF), ("state", 0, math.nan), ("x", 5, INF), ("x", 350, -INF), ("x", 700, INF), ("x", 1100, math.nan), ("x", 1499, INF)]


@pytest.mark.parametrize("dtype,d", [(F32, 131), (BF16, 130), (BF16, 131)])
@pytest.mark.parametrize("kind", KINDS)
def test_forward(kind, d, dtype):
    x, gate, bias, state, bounds = inputs(d, dtype)
    mixer = GatedRecurrence(bias, kind)
    clean = mixer.forward(x, gate, bounds, state)
    places = {"x": x.clone(), "state": state.clone()}
    for k, (name, row, value) in enumerate(PLANTS):
        places[name][row, 3 + 11 * k] = value
    places["x"][400, 3] = -INF  # meets the state's: a NaN from there on
    places["x"][690, 3 + 11] = INF
    planted = (places["x"], gate, bounds, places["state"])
    want = forward64(kind, places["x"], gate, bias, places["state"])
    got = mixer.forward(*planted)
    # by channel: both sequences' states, one row's, the NaN's, what x plants up to its sequence's end
    assert compare(got[0], want[0], clean[0]) == 700 + 799 + 1 + 0 + 700 + 695 + 350 + 1 + 400 + 1 + 10
    compare(got[1], want[1], clean[1])
    assert bool(got[0][399, 3] == INF) and bool(got[0][400:700, 3].isnan().all()) and bool(got[0][701:, 3].isfinite().all())
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(mixer.forward(*planted), got))


@pytest.mark.parametrize("dtype,d", [(F32, 131), (BF16, 130), (BF16, 131)])
@pytest.mark.parametrize("kind", KINDS)
def test_backward(kind, d, dtype):
    x, gate, bias, state, bounds = inputs(d, dtype, seed=10)
    mixer = GatedRecurrence(bias, kind)
    h, _ = mixer.forward(x, gate, bounds, state)
    gh, glast = draw(N, d, dtype=dtype, seed=20), draw(S, d, seed=21)
    clean = [t.clone() for t in (*mixer.backward(x, gate, h, gh, bounds, state, glast), mixer.gradients()["bias"])]
    bad_gh, bad_glast = gh.clone(), glast.clone()
    for k, (place, row, value) in enumerate([(bad_glast, 0, INF), (bad_glast, 3, -INF), (bad_glast, 2, INF), (bad_glast, 1, INF), (bad_gh, 690, -INF), (bad_gh, 350, INF), (bad_gh, 700, INF),
                                             (bad_gh, 1499, math.nan), (bad_gh, 0, INF), (bad_gh, 710, -INF)]):
        place[row, 2 + 11 * k] = value
    bad_gh[300, 2] = -INF  # meets glast's
    want = backward64(kind, x, gate, bias, h, bad_gh, state, bad_glast)
    got = (*mixer.backward(x, gate, h, bad_gh, bounds, state, bad_glast), mixer.gradients()["bias"])
    far = (gate.double() + bias.double()).abs().cpu() > 80.0
    # by channel: from the sequence's end, or the planted row, down to its begin
    assert compare(got[0], want[0], clean[0], far) == 700 + 799 + 1 + 0 + 691 + 351 + 1 + 799 + 1 + 10
    compare(got[1], want[1], clean[1], far)
    compare(got[2], want[2], clean[2])
    hit = torch.zeros(d, dtype=torch.bool)
    hit[[2 + 11 * k for k in range(10) if k != 3]] = True  # the sequence without rows has no part in the bias's gradient
    assert torch.equal(got[3].cpu()[~hit], clean[3].cpu()[~hit]) and not bool(got[3].cpu()[hit].isfinite().any())


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("kind", KINDS)
def test_step(kind, dtype):
    d, n = 67, 9
    x, gate, bias, state = draw(n, d, dtype=dtype), draw(n, d, dtype=dtype, seed=1, std=4.0), draw(d, seed=2), draw(n, d, seed=3)
    mixer = GatedRecurrence(bias, kind)
    clean_state = state.clone()
    clean = mixer.step(x, gate, clean_state)
    state[0, ::2], state[1, 1::2], x[2, ::3], state[3], x[3] = INF, -INF, -INF, INF, -INF
    z, c = gates(gate, bias)
    want = c * state.double().cpu() + input_of(kind, z, c)[0] * x.double().cpu()
    h = mixer.step(x, gate, state)
    compare(h, want, clean)
    compare(state, want, clean_state)
    assert bool(h[3].isnan().all())


@pytest.mark.parametrize("n", (1, 2, 40, 1000))
def test_ends_of_float32(n):
    """h + v up to float32's largest: the definition's values. Beyond it: an infinity, and on to the last row, no NaN."""
    d = 70
    gate, bias = torch.zeros(n, d, device="cuda"), torch.zeros(d, device="cuda")
    mixer = GatedRecurrence(bias, "free")
    x, state = torch.full((n, d), 1.0e38, device="cuda"), torch.full((1, d), 2.2e38, device="cuda")  # 2.2 / 2 + 1 = 2.1, and on to 2
    h, last = mixer.forward(x, gate, None, state)
    want = 2e38 + 0.2e38 * 0.5 ** torch.arange(1, n + 1, dtype=torch.float64)
    assert bool(((h.double().cpu() - want[:, None]).abs() <= 8 * 2.0 ** -24 * want[:, None]).all())  # errors are halved from row to row
    assert torch.equal(last, h[-1:])
    step = state.clone()
    assert torch.equal(mixer.step(x[:1], gate[:1], step), h[:1]) and torch.equal(step, h[:1])
    for sign in (1.0, -1.0):
        h, last = mixer.forward(2 * sign * x, gate, None, sign * state)  # 2.2 / 2 + 2 = 3.1, then 3.1 / 2 + 2 = 3.55: beyond
        assert bool((h[1:] == sign * INF).all()) and bool(((h[0].double() / (sign * 3.1e38) - 1).abs() <= 4 * 2.0 ** -24).all()) and torch.equal(last, h[-1:])
        gx, _, gstate = mixer.backward(x, gate, x, 2 * sign * x, None, state, 1.5 * sign * state)
        assert bool((gx == sign * INF).all()) and bool((gstate == sign * INF).all())
        # z a little below a half: h - z h + v begins with h + v = 4.2e38, which is beyond although the row is not
        h, last = mixer.forward(2 * sign * x, gate - 0.01, None, sign * state)
        assert bool((h == sign * INF).all()) and bool((last == sign * INF).all())


def test_an_infinity_through_many_tiles():
    """From the first row to the last of the longest call a product of factors that float32 does not hold lies between them."""
    n, d = 40000, 66
    x, gate, bias = draw(n, d, dtype=BF16), draw(n, d, dtype=BF16, seed=1), draw(d, seed=2)
    mixer = GatedRecurrence(bias, "normed")
    state = torch.zeros(1, d, device="cuda")
    clean, _ = mixer.forward(x, gate, None, state)
    state[0, 5] = -INF
    h, last = mixer.forward(x, gate, None, state)
    assert bool((h[:, 5] == -INF).all()) and bool(last[0, 5] == -INF)
    h[:, 5] = clean[:, 5]
    assert torch.equal(h, clean)
