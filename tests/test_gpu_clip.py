"""``hffn_amd.clip`` against float64 norms on the GPU. The norm's sums are float64 (relative error below n 2^-52), rounded once to
float32: 2^-23 of the norm bounds it. A scaled entry is one float32 product of a float32 factor (2^-24 + 2^-23 of it) and,
for bfloat16, rounded (2^-8)."""
from __future__ import annotations

import math

import pytest
import torch

from hffn_amd.clip import clip_grad_norm_, grad_norm

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def make(sizes, seed=0, dtypes=(F32, BF16), std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return [(std * torch.randn(size, generator=g, device="cuda")).to(dtypes[k % len(dtypes)]) for k, size in enumerate(sizes)]


def norm64(tensors, kind=2.0):
    all_ = torch.cat([t.double().flatten() for t in tensors]) if tensors else torch.zeros(0, dtype=torch.float64)
    if all_.numel() == 0:
        return 0.0
    return float(all_.abs().max()) if kind == math.inf else float(all_.square().sum().sqrt())


def check(tensors, limit, kind=2.0, out=None):
    before = [t.double() for t in tensors]
    want = norm64(before, kind)
    norm = clip_grad_norm_(tensors, limit, kind, out)
    assert norm.dtype == F32 and norm.shape == ()
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    factor = min(1.0, limit / (want + 1e-6))
    for b, t in zip(before, tensors if out is None else out):
        bound = (2.0 ** -22 + (2.0 ** -8 if t.dtype == BF16 else 0.0)) * (factor * b).abs() + (1e-38 if factor < 1 else 0.0)
        assert bool(((t.double() - factor * b).abs() <= bound).all())
    if out is not None:
        assert all(torch.equal(t.double(), b) for t, b in zip(tensors, before))
    elif factor == 1.0:
        assert all(torch.equal(t.double(), b) for t, b in zip(tensors, before))


SIZES = [(), (1,), (3, 5), (8192,), (8193,), (0,), (4, 0, 2), (100_003,), (7, 11, 13), (1 << 20,)]


@pytest.mark.parametrize("kind", (2.0, math.inf))
@pytest.mark.parametrize("limit", (0.5, 1e9, 0.0, math.inf))
def test_sizes_and_limits(limit, kind):
    check(make(SIZES), limit, kind)
    check(make(SIZES, dtypes=(BF16,)), limit, kind)


@pytest.mark.parametrize("count", (1, 95, 96, 97, 193, 400))
def test_many_tensors(count):
    check(make([(1 + 37 * k % 1000,) for k in range(count)], seed=count), 1.0)


@pytest.mark.parametrize("start", range(1, 9))
@pytest.mark.parametrize("dtype", (F32, BF16))
def test_alignment(dtype, start):
    """Entries that start anywhere, alone and with a scaled copy that starts elsewhere."""
    for size in (1, 2, 5, 17, 8200):
        whole = make([(size + 16,)], seed=size, dtypes=(dtype,))[0]
        check([whole.clone()[start:start + size]], 0.1)
        for to in (F32, BF16):
            for shift in (0, 3, start):
                out = torch.full((size + 16,), 7.0, dtype=to, device="cuda")
                check([whole[start:start + size]], 0.1, out=[out[shift:shift + size]])
                assert bool((out[:shift] == 7).all()) and bool((out[shift + size:] == 7).all())


def test_out_of_other_types():
    for limit in (0.5, 1e9):
        tensors = make(SIZES, seed=2)
        check(tensors, limit, out=[torch.empty_like(t, dtype=F32) for t in tensors])
        check(tensors, limit, out=[torch.empty_like(t, dtype=BF16) for t in tensors])


def test_orders_of_dimensions():
    base = make([(24, 40, 3)], dtypes=(F32,))[0]
    check([base.permute(2, 0, 1), make([(5, 6)], 1)[0].T], 0.5)


def test_sizes_of_entries():
    """Squares far outside float32."""
    for std in (1e-30, 1e30):
        tensors = make([(1000,), (50,)], dtypes=(F32,), std=std)
        assert abs(float(grad_norm(tensors)) - norm64(tensors)) <= 2.0 ** -23 * norm64(tensors)
    check(make([(1000,), (50,)], dtypes=(F32,), std=1e30), 1e28)


def test_not_numbers():
    for value in (math.nan, math.inf, -math.inf):
        for kind in (2.0, math.inf):
            tensors = make([(100,), (9000,)], dtypes=(F32,))
            tensors[1][8500] = value
            kept = [t.clone() for t in tensors]
            norm = float(clip_grad_norm_(tensors, 1.0, kind))
            if math.isnan(value):
                assert math.isnan(norm) and all(bool(t.isnan().all()) for t in tensors)
            else:
                assert norm == math.inf and not bool(tensors[0].any()) and int(tensors[1].isnan().sum()) == 1
            assert torch.equal(grad_norm(kept, kind).isnan(), torch.tensor(math.isnan(value), device="cuda"))


def test_nothing_to_measure():
    for tensors in ([], [torch.empty(0, device="cuda")]):
        assert float(grad_norm(tensors)) == 0.0 and float(clip_grad_norm_(tensors, 1.0)) == 0.0


def test_one_tensor_and_generators():
    t = make([(100,)])[0]
    assert torch.equal(grad_norm(t), grad_norm(x for x in [t]))


def test_repeats_bit_for_bit():
    tensors = make([(3_000_001,), (17,), (500_000,)], seed=3)
    first = grad_norm(tensors)
    assert all(torch.equal(grad_norm(tensors), first) for _ in range(3))


def test_replayed_from_a_graph(device):
    tensors, outs = make([(5000,), (33, 7)], seed=4), [torch.empty(5000, device="cuda"), torch.empty(33, 7, device="cuda")]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_grad_norm_(tensors, 1.0, out=outs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(tensors, 1.0, out=outs)
    for seed in range(3):
        for t, fresh in zip(tensors, make([(5000,), (33, 7)], seed=10 + seed)):
            t.copy_(fresh)
        graph.replay()
        eager = [torch.empty_like(t) for t in outs]
        want = clip_grad_norm_(tensors, 1.0, out=eager)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_refusals(device):
    a, b = torch.ones(100, device=device), torch.ones(100, device=device)
    for call, match in ((lambda: clip_grad_norm_([a, a[50:]], 1.0), "share memory"), (lambda: clip_grad_norm_([a, a], 1.0), "share memory"),
                        (lambda: clip_grad_norm_([a], -1.0), "negative"), (lambda: clip_grad_norm_([a], math.nan), "negative"),
                        (lambda: clip_grad_norm_([a], 1.0, 1.0), "norm_type"), (lambda: grad_norm([a.half()]), "float32 or bfloat16"),
                        (lambda: grad_norm([a, b.cpu()]), "one device"), (lambda: grad_norm([a[::2]]), "does not fill"),
                        (lambda: grad_norm([a[:1].expand(5)]), "does not fill"),
                        (lambda: clip_grad_norm_([a], 1.0, out=[a]), "share memory"), (lambda: clip_grad_norm_([a], 1.0, out=[b, a]), "shape"),
                        (lambda: clip_grad_norm_([a], 1.0, out=[b[:50]]), "shape"), (lambda: clip_grad_norm_([a, b], 1.0, out=[a + 1, a[:0]]), "shape")):
        with pytest.raises(ValueError, match=match):
            call()
    assert torch.equal(a, torch.ones_like(a))
