"""Host-side checks of the C entries of the embedding that take ids from the table's end and tell of ids without a row."""
from __future__ import annotations

from test_host_lm_operators import BIG, F32, P, at, no_gpu, refused

from hffn_amd import _lib
from hffn_amd.embedding import _FROM_END


@no_gpu
def test_refusals():
    lib = _lib.load()

    def guarded(vt=F32, w=P, ids=P, size=8, out=P, outside=P, d=64, v=100, n=5):
        return lib.hffn_embedding_guarded(vt, w, ids, 1, size, 1.0, out, outside, d, v, n, None)

    def gradient(size):
        return lib.hffn_embedding_gradient(F32, P, 64, P, 1, size, -1, 1.0, 0, P, P, BIG, 64, 100, 5, None)

    refused(guarded(outside=at(2)), "misaligned outside")
    for change, fragment in ((dict(vt=2), "value type"), (dict(n=0), "n=0"), (dict(v=0), "vocab=0"), (dict(w=None), "null"), (dict(ids=None), "null"), (dict(out=None), "null"),
                             (dict(out=at(2)), "misaligned rows")):
        refused(guarded(**change), fragment)
    for size in (_FROM_END, _FROM_END + 2, _FROM_END + 12, 2 * _FROM_END + 8, -1):
        refused(guarded(size=size), "4 or 8")
        refused(gradient(size), "4 or 8")
        refused(lib.hffn_embedding(F32, P, P, 1, size, 1.0, P, 64, 100, 5, None), "4 or 8")
    refused(guarded(ids=at(4), size=_FROM_END + 8), "misaligned ids")
