"""Host-side checks of the training operators' C entries without a GPU: sizes of workspaces, and refusals before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

from hffn_amd import _lib
from hffn_amd.clip import clip_grad_norm_, grad_norm
from hffn_amd.loss import HeadLoss
from hffn_amd.norm import ResidualNorm

P = ctypes.c_void_p(4096)  # never dereferenced: every call below fails validation first
F32, BF16 = 0, 1
BIG = 1 << 40
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="uses placeholder pointers: never run where a launch could reach a GPU")


def refused(status: int, fragment: str) -> None:
    assert status == _lib.OK - 1
    assert fragment in _lib.load().hffn_last_error().decode()


def loss_bytes(vt, n, d, vocab, aligned=1, gradients=1, piece=0):
    return _lib.query_bytes(_lib.load().hffn_loss_workspace, vt, n, d, vocab, aligned, gradients, piece)


@no_gpu
def test_loss_entries_refuse_bad_arguments():
    lib = _lib.load()
    good = dict(vt=F32, x=P, xs=64, w=P, labels=P, ls=1, lb=8, ig=-100, losses=P, work=P, bytes=BIG, d=64, v=100, n=5)

    def losses(**change):
        a = {**good, **change}
        return lib.hffn_losses(a["vt"], a["x"], a["xs"], a["w"], a["labels"], a["ls"], a["lb"], a["ig"], a["losses"], a["work"], a["bytes"], a["d"],
                               a["v"], a["n"], None)

    def step(loss=P, gx=P, gw=P, piece=0, **change):
        a = {**good, **change}
        return lib.hffn_loss_step(a["vt"], a["x"], a["xs"], a["w"], a["labels"], a["ls"], a["lb"], a["ig"], 1, 1.0, piece, loss, gx, gw, a["work"],
                                  a["bytes"], a["d"], a["v"], a["n"], None)

    for call in (losses, step):
        for change, fragment in ((dict(vt=2), "value type"), (dict(n=0), "n=0"), (dict(n=1 << 19), "token count"), (dict(d=0), "d_model=0"),
                                 (dict(d=32769, xs=32769), "d_model"), (dict(v=0), "vocab=0"), (dict(v=(1 << 24) + 1), "vocab"),
                                 (dict(x=None), "null"), (dict(w=None), "null"), (dict(labels=None), "null"), (dict(work=None), "null"),
                                 (dict(xs=63), "row stride 63"), (dict(lb=2), "labels of 4 or 8"), (dict(labels=ctypes.c_void_p(4100)), "misaligned labels"),
                                 (dict(x=ctypes.c_void_p(4098)), "align"), (dict(vt=BF16, w=ctypes.c_void_p(4097)), "align"),
                                 (dict(work=ctypes.c_void_p(4096 + 128)), "256-byte"), (dict(bytes=100), "needed")):
            refused(call(**change), fragment)
    refused(losses(losses=None), "null")
    for name in ("loss", "gx", "gw"):
        refused(step(**{name: None}), "null")
    need = loss_bytes(F32, 5, 64, 100)
    refused(step(bytes=need - 1), f"{need} needed")
    odd = loss_bytes(BF16, 5, 64, 100, aligned=0)  # a bfloat16 weight that is not 16-byte aligned is packed
    assert odd > loss_bytes(BF16, 5, 64, 100)
    refused(step(vt=BF16, bytes=odd - 1, w=ctypes.c_void_p(4098)), f"{odd} needed")


def test_loss_workspace_sizes():
    lib, out = _lib.load(), ctypes.c_uint64()
    refused(lib.hffn_loss_workspace(F32, 5, 64, 100, 1, 1, 0, None), "null")
    refused(lib.hffn_loss_workspace(7, 5, 64, 100, 1, 1, 0, ctypes.byref(out)), "value type")
    for vt in (F32, BF16):
        assert loss_bytes(vt, 512, 1024, 50304) > loss_bytes(vt, 512, 1024, 50304, gradients=0)
        # smaller pieces take less, down to 256 rows; a piece as large as the vocabulary is the most
        pieces = [loss_bytes(vt, 2048, 256, 50304, piece=p) for p in (1, 16 << 20, 64 << 20, 1 << 40, 1 << 50)]
        assert pieces == sorted(pieces) and pieces[-2] == pieces[-1]
        assert loss_bytes(vt, 2048, 256, 50304) == loss_bytes(vt, 2048, 256, 50304, piece=512 << 20)
    # the logits of 8192 tokens would be 824 MB in bfloat16; bfloat16 weights are read in place
    assert loss_bytes(BF16, 8192, 2048, 50304) < (512 << 20) + (1 << 28)
    assert loss_bytes(BF16, 8, 1024, 50304, gradients=0) < 10 << 20
    # a float32 weight is read as it is for a few tokens of a large vocabulary, packed otherwise
    weight = 4 * 50304 * 1024
    assert loss_bytes(F32, 8, 1024, 50304, gradients=0) < weight < loss_bytes(F32, 512, 1024, 50304, gradients=0)
    assert loss_bytes(F32, 8, 1024, 50304, aligned=0, gradients=0) < weight
    assert loss_bytes(BF16, 8, 1024, 50304, gradients=0) < weight // 2 < loss_bytes(BF16, 8, 1024, 50304, aligned=0, gradients=0)
    # the largest call the entries take is a finite number of bytes
    assert 0 < loss_bytes(F32, 1 << 18, 32768, 1 << 24) < 1 << 50


@no_gpu
def test_norm_entries_refuse_bad_arguments():
    lib = _lib.load()

    def forward(vt=F32, x=P, xs=64, f=P, fs=64, w=P, bias=None, gate=None, pw=None, pb=None, eps=1e-5, layer=1, r=P, h=P, d=64, n=5):
        return lib.hffn_residual_norm(vt, x, xs, f, fs, w, bias, gate, pw, pb, 1.0, eps, layer, r, h, d, n, None)

    def backward(vt=F32, r=P, rs=64, f=P, fs=64, gr=P, grs=64, gh=P, ghs=64, w=P, gate=None, pw=None, pb=None, eps=1e-5, layer=1, gx=P, gf=P, gw=P,
                 gb=None, gg=None, gpw=None, gpb=None, work=P, bytes_=BIG, d=64, n=5):
        return lib.hffn_residual_norm_backward(vt, r, rs, f, fs, gr, grs, gh, ghs, w, gate, pw, pb, 1.0, eps, layer, gx, gf, gw, gb, gg, gpw, gpb, work,
                                               bytes_, d, n, None)

    for call in (forward, backward):
        for change in (dict(vt=3), dict(n=0), dict(n=1 << 19), dict(d=0), dict(d=16385), dict(w=None), dict(fs=63), dict(eps=-1.0), dict(eps=float("nan")),
                       dict(w=ctypes.c_void_p(4098)), dict(f=ctypes.c_void_p(4098)), dict(f=None, gate=P, gg=P) if call is backward else dict(f=None, gate=P),
                       dict(pb=P, gpb=P) if call is backward else dict(pb=P)):
            assert call(**change) == _lib.OK - 1, change
    refused(forward(x=None), "null")
    refused(forward(h=None), "null")
    refused(forward(r=None), "null")
    refused(forward(layer=0, bias=P), "bias")
    refused(backward(gh=None), "null")
    refused(backward(gw=None), "null")
    refused(backward(gate=P), "gradients")
    refused(backward(gg=P), "gradients")
    refused(backward(work=ctypes.c_void_p(4104)), "16-byte")
    need = _lib.query_bytes(lib.hffn_residual_norm_backward_workspace, 5, 64)
    refused(backward(bytes_=need - 1), f"{need} needed")


@no_gpu
def test_clip_entries_refuse_bad_arguments():
    lib = _lib.load()
    need = _lib.query_bytes(lib.hffn_clip_workspace, 2)

    def arrays(pointers, counts=(8, 8), types=(F32, F32)):
        return ((ctypes.c_void_p * 2)(*pointers), (ctypes.c_uint64 * 2)(*counts), (ctypes.c_int * 2)(*types))

    def clip(pointers=(4096, 8192), out=None, out_types=None, limit=1.0, bytes_=need, work=P, norm=P, **table):
        p, counts, types = arrays(pointers, **table)
        to = None if out is None else (ctypes.c_void_p * 2)(*out)
        kinds = None if out_types is None else (ctypes.c_int * 2)(*out_types)
        return lib.hffn_clip(2, p, to, counts, types, kinds, 0, limit, work, bytes_, norm, None)

    refused(clip(limit=-1.0), "negative")
    refused(clip(limit=float("nan")), "negative")
    refused(clip(types=(F32, 5)), "array 1: unknown value type")
    refused(clip(counts=(8, (1 << 38) + 1)), "array 1")
    refused(clip(pointers=(4096, None)), "array 1: null")
    refused(clip(pointers=(4096, 8194)), "align")
    refused(clip(pointers=(4096, 4096 + 28)), "share memory")
    refused(clip(out=(16384, 4096 + 16), out_types=(F32, F32)), "share memory")
    refused(clip(out=(16384, 32768)), "null")
    refused(clip(bytes_=need - 1), f"{need} needed")
    refused(clip(work=ctypes.c_void_p(4100)), "8-byte")
    refused(clip(norm=None), "null")
    p, counts, types = arrays((4096, 8192), types=(F32, -1))
    refused(lib.hffn_grad_norm(2, p, counts, types, 0, P, need, P, None), "unknown value type")


@no_gpu
def test_the_python_entries_need_the_device():
    with pytest.raises((ValueError, RuntimeError)):
        HeadLoss(torch.zeros(4, 8))
    with pytest.raises((ValueError, RuntimeError)):
        ResidualNorm(torch.ones(8))
    for call in (grad_norm, lambda t: clip_grad_norm_(t, 1.0)):
        with pytest.raises(ValueError, match="cuda:0"):
            call([torch.zeros(3)])
