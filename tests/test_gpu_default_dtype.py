"""Every object of the package allocates what its kernels write in the kernels' own types, whatever type PyTorch gives to new
tensors by default: the same types and the same bits under a bfloat16 and a float64 default as under float32."""
from __future__ import annotations

import pytest
import torch

from hffn_amd.bench_train import make_cell
from hffn_amd.clip import clip_grad_norm_, grad_norm
from hffn_amd.ffn import hip_layer
from hffn_amd.loss import HeadLoss
from hffn_amd.norm import ResidualNorm
from hffn_amd.runtime import HFFNRuntime
from hffn_amd.train_lm import LMTrainer
from hffn_amd.train_runtime import HFFNTrainRuntime

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
CELL = "128_256_d020"


@pytest.fixture(params=(BF16, torch.float64), ids=("bfloat16", "float64"))
def default_dtype(request):
    yield request.param
    torch.set_default_dtype(F32)


def draw(*shape, dtype=F32, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=F32, device="cuda").to(dtype)


def head(dtype):
    weight, x = 0.1 * draw(700, 136, seed=1).to(dtype), draw(300, 136, dtype=dtype, seed=2)
    labels = torch.arange(300, device="cuda") % 700
    loss = HeadLoss(weight.to(dtype), max_tokens=7)
    return [t.clone() for t in (loss.losses(x, labels), *loss.step(x, labels))]


def norm(dtype):
    rows = [draw(600, 1001, dtype=dtype, seed=k) for k in range(4)]
    vectors = [1 + 0.1 * draw(1001, seed=10 + k) for k in range(5)]
    b = ResidualNorm(vectors[0], vectors[1], gate=vectors[2], post_weight=vectors[3], post_bias=vectors[4])
    r, h = b.forward(rows[0], rows[1])
    return [r, h, *b.backward(r, rows[1], rows[2], rows[3]), *b.gradients().values()]


def clip(dtype):
    tensors = [draw(5000, dtype=dtype), draw(40, 33, seed=1)]
    return [grad_norm(tensors), clip_grad_norm_(tensors, 0.5), *tensors]


def layers(dtype):
    layer = hip_layer(make_cell(CELL, 3))
    x, gy = draw(130, 128, seed=4), draw(130, 128, seed=5)
    out = [HFFNRuntime([layer], "cuda").forward(0, x[:n]).clone() for n in (1, 16, 130)]
    train = HFFNTrainRuntime(HFFNRuntime([layer], "cuda"), max_tokens=130)
    z = torch.empty(256 * 136, dtype=F32, device="cuda")
    train.forward(0, x, z)
    return [*out, train.backward(0, gy).clone(), *(t.clone() for t in train.gradients(0).values())]


def model(dtype):
    trainer = LMTrainer([hip_layer(make_cell(CELL, 3))], 300, 60, seed=1)
    ids = torch.arange(60, device="cuda")
    out = [t.clone() for t in trainer.step(ids, ids + 1)]
    return [*out, *(t.clone() for t in trainer.parameters()), trainer.losses(ids, ids + 1).clone()]


@pytest.mark.parametrize("dtype", (F32, BF16))
@pytest.mark.parametrize("run", (head, norm, clip, layers, model))
def test_the_default_type_does_not_matter(run, dtype, default_dtype):
    want = run(dtype)
    torch.set_default_dtype(default_dtype)
    got = run(dtype)
    torch.set_default_dtype(F32)
    assert [t.dtype for t in got] == [t.dtype for t in want]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
