"""``TokenEmbedding`` with ids that count from the table's end and with the word that tells of ids without a row. Both give the rows of
tensor indexing, bit for bit; a scale of 1 changes none."""
from __future__ import annotations

import pytest
import torch

from hffn_amd.embedding import TokenEmbedding
from test_gpu_embedding import BF16, F32, check_gradient, draw, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("ids_dtype", (torch.int32, torch.int64))
@pytest.mark.parametrize("n,d,vocab", [(1, 8, 1), (77, 33, 100), (3000, 64, 500), (20000, 16, 1000)])
def test_negative_ids(n, d, vocab, ids_dtype, dtype):
    weight, g, ids = draw(vocab, d, dtype=dtype, seed=n), draw(n, d, dtype=dtype, seed=n + 1), tokens(n, vocab, n + 2)
    mixed = torch.where(torch.arange(n, device="cuda") % 3 == 0, ids, ids - vocab).to(ids_dtype)
    table, outside = TokenEmbedding(weight, padding_index=vocab // 2), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(table.forward(mixed, from_end=True, outside=outside), weight[ids]) and int(outside) == 0
    want = table.backward(ids, g).clone()
    assert torch.equal(table.backward(mixed, g, from_end=True), want)
    check_gradient(want, weight, ids, g, 1.0, padding=vocab // 2)
    base = draw(vocab, d, dtype=dtype, seed=n + 3)
    assert torch.equal(table.backward(mixed, g, base.clone(), from_end=True), table.backward(ids, g, base.clone()))
    rows = table.forward(mixed, outside=outside)  # without it a negative id has no row
    assert bool(rows[mixed < 0].isnan().all()) and torch.equal(rows[mixed >= 0], weight[ids[mixed >= 0]])
    assert int(outside) == int((mixed < 0).any())


@pytest.mark.parametrize("from_end", (False, True))
@pytest.mark.parametrize("bad", (50, -51, 2 ** 31 - 1, -2 ** 31, 2 ** 63 - 1, -2 ** 63))
def test_an_id_without_a_row_is_told_of(bad, from_end):
    """One among many, first, last and in the middle; the word is left as it was where there is none."""
    weight = draw(50, 12)
    table, n = TokenEmbedding(weight), 4099
    good, g = tokens(n, 50, 5), draw(n, 12, seed=6)
    for place in (0, 2000, n - 1):
        ids, outside = good.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
        ids[place] = bad
        rows = table.forward(ids, from_end=from_end, outside=outside)
        assert int(outside) == 1 and bool(rows[place].isnan().all())
        assert int(rows.isnan().any(1).sum()) == 1
        check_gradient(table.backward(ids, g, from_end=from_end), weight, ids, g, 1.0)
        table.forward(good, from_end=from_end, outside=outside)
        assert int(outside) == 1


def test_refusals(device):
    table, ids = TokenEmbedding(draw(50, 12)), tokens(9, 50)
    word = torch.zeros(1, dtype=torch.int32, device=device)
    for bad in (word.long(), word.float(), word[0], word.expand(2), word.cpu(), word[:0]):
        with pytest.raises(ValueError, match="outside"):
            table.forward(ids, outside=bad)
