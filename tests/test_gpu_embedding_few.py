"""The gradient of up to 512 positions, which takes one launch and no order: against the definition, and bit for bit against the same positions
among so many without a row (an id of -1) that they are ordered."""
from __future__ import annotations

import pytest
import torch

from hffn_amd.embedding import TokenEmbedding
from test_gpu_embedding import BF16, F32, check, check_gradient, draw, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("n,d,vocab", [(1, 1, 1), (2, 3, 70000), (15, 1, 40000), (16, 2, 33000), (17, 64, 1000), (63, 255, 50), (64, 256, 300), (65, 257, 300), (511, 1001, 2003),
                                       (512, 1024, 5000), (512, 8, 3), (513, 8, 3), (1023, 7, 100000), (1024, 2048, 999), (1024, 8, 3), (1025, 8, 3), (1000, 4100, 17)])
def test_sizes(n, d, vocab, dtype):
    check(n, d, vocab, dtype, scale=0.125, padding=vocab // 3 if n % 2 else None, seed=n + d)


def same_as_ordered(ids, d, vocab, dtype, padding=None, stride=0):
    n = len(ids)
    g = draw(1100, d + stride, dtype=dtype, seed=n + d)[:, :d]
    more = torch.cat([ids, torch.full((1100 - n,), -1, dtype=ids.dtype, device="cuda")])
    table = TokenEmbedding(draw(vocab, d, dtype=dtype), scale=0.3, padding_index=padding)
    got = table.backward(ids, g[:n]).clone()
    check_gradient(got, table.weight, ids, g[:n], float(torch.tensor(0.3, dtype=F32)), padding=padding)
    assert torch.equal(got, table.backward(more, g))
    base = draw(vocab, d, dtype=dtype, seed=3)
    got = table.backward(ids, g[:n], base.clone())
    check_gradient(got, table.weight, ids, g[:n], float(torch.tensor(0.3, dtype=F32)), base=base, padding=padding)
    assert torch.equal(got, table.backward(more, g, base.clone()))


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("n", (1, 40, 64, 65, 128, 129, 448, 449, 500, 512, 513))
def test_runs_have_the_bits_of_the_order(n, dtype):
    """One token everywhere, a few, many; in order, shuffled; rows that start on 16 bytes and ones that do not."""
    shuffled = torch.randperm(n, generator=torch.Generator("cuda").manual_seed(n), device="cuda")
    for d, stride in ((256, 0), (257, 0), (1000, 24), (60, 1)):
        for ids in (torch.full((n,), 11, device="cuda"), torch.arange(n, device="cuda") // 65, (torch.arange(n, device="cuda") % 3)[shuffled], tokens(n, 30, n), tokens(n, 2000, n, power=6.0)):
            same_as_ordered(ids, d, 2003, dtype, padding=2, stride=stride)


def test_long_runs_that_begin_side_by_side():
    """The first positions of seven tokens of more than 64 positions each lie in one block."""
    for n in (490, 512):
        ids = torch.arange(n, device="cuda") % 7
        same_as_ordered(ids, 300, 40, F32)
        same_as_ordered(ids.int().flip(0), 264, 15, BF16, padding=14)


@pytest.mark.parametrize("offset", (1, 3))
def test_a_gradient_that_starts_anywhere(offset):
    """`into` and the whole gradient by the C entry, at an address that no 16 bytes divide: what lies around it stays."""
    from hffn_amd import _lib
    from hffn_amd.runtime import current_stream
    n, d, vocab = 300, 36, 5001
    ids, g = tokens(n, vocab, 8), draw(n, d, seed=9)
    room = torch.full((vocab * d + 8,), 7.0, device="cuda")
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    lib = _lib.load()
    for into in (0, 1):
        _lib.check(lib.hffn_embedding_gradient(0, g.data_ptr(), d, ids.data_ptr(), 1, 8, -1, 1.0, into, room.data_ptr() + 4 * offset, work.data_ptr(), work.numel(), d, vocab, n,
                                               current_stream(g.device)), "gradient")
        got = room[offset:offset + vocab * d].view(vocab, d)
        if into == 0:
            check_gradient(got, got, ids, g, 1.0)
            base = got.clone()
        else:
            check_gradient(got, got, ids, g, 1.0, base=base)
        assert bool((room[:offset] == 7.0).all()) and bool((room[offset + vocab * d:] == 7.0).all())


def test_no_position_has_a_row():
    for n in (1, 700):
        table = TokenEmbedding(draw(333, 20), padding_index=5)
        g = draw(n, 20, seed=1)
        table.backward(torch.arange(n, device="cuda") % 333, g)
        for ids in (torch.full((n,), 5, device="cuda"), torch.full((n,), -9, device="cuda"), torch.full((n,), 333, device="cuda")):
            assert not bool(table.backward(ids, g).any())
            base = draw(333, 20, seed=2)
            assert torch.equal(table.backward(ids, g, base.clone()), base)


def test_replayed_from_a_graph(device):
    n, d, vocab = 512, 520, 4000
    table, ids, g = TokenEmbedding(draw(vocab, d, dtype=BF16)), tokens(n, vocab), draw(n, d, dtype=BF16, seed=1)
    table.backward(ids, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        table.backward(ids, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = table.backward(ids, g)
    other = TokenEmbedding(table.weight)
    for seed in range(4):
        ids.copy_(tokens(n, vocab, 20 + seed))
        g.copy_(draw(n, d, dtype=BF16, seed=30 + seed))
        graph.replay()
        want = other.backward(ids, g)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
