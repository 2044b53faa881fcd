"""The training-side operators whose time on the GPU is tracked: the head's loss, the residual norm, gradient clipping.

A case is one call of a program that trains (or scores with) a stack of HFFN layers under a language-model head:

* ``loss``: softmax cross entropy over a vocabulary from hidden rows and the head's weight. ``losses`` is the loss of every
  token (scoring, evaluation), ``step`` the mean loss with the gradients of the hidden rows and of the weight;
* ``norm``: the boundary between two blocks, ``r = x + scale gate * post_norm(f)`` and ``h = norm(r)``, forward or backward;
* ``clip``: the global norm over every gradient of a model, and the gradients scaled to at most a limit, in place or into
  float32 buffers for the optimizer.

Hidden widths, vocabulary, layer counts and densities are those of the package's Pythia shapes and test layers, and odd ones
beside them. Everything is drawn on the GPU from the seed.
"""
from __future__ import annotations

import math

import torch

own = False

IGNORE = -100
EPS = 1e-5
SCALE = 0.7
WEIGHT_STD, GRAD_STD = 0.02, 1e-3
WIDTHS = (256, 512, 768, 1024, 2048, 2560, 400, 1104)
VOCAB = 50304
MOST_LOSS = 8192 * 50304 * 2048  # tokens x vocabulary x width of the largest call
MOST_NORM = 8192 * 2560          # tokens x width
MOST_CLIP = 160_000_000          # gradient entries


def _loss(name, direction, tokens, d_model, vocab, type_, ignored=0.0):
    case = {"op": "loss", "direction": direction, "tokens": tokens, "d_model": d_model, "vocab": vocab, "type": type_,
            "ignored": ignored}
    return {"name": name, **case} if name else case


def _norm(name, direction, tokens, d_model, type_, kind, post, gate):
    case = {"op": "norm", "direction": direction, "tokens": tokens, "d_model": d_model, "type": type_, "kind": kind,
            "post": post, "gate": gate}
    return {"name": name, **case} if name else case


def _clip(name, limit, layers, d_model, d_ff, density, vocab, head):
    case = {"op": "clip", "direction": limit, "layers": layers, "d_model": d_model, "d_ff": d_ff, "density": density,
            "vocab": vocab, "head": head}
    return {"name": name, **case} if name else case


def listed():
    return [
        # Scoring one token of a sequence that is being decoded, the wide bfloat16 head: the lowest latency asked for.
        _loss("loss_score_2048_bf16_n1", "losses", 1, 2048, VOCAB, "bf16"),
        # Perplexity of a batch of short prompts on the smallest float32 model.
        _loss("loss_eval_512_f32_n512", "losses", 512, 512, VOCAB, "float32"),
        # A ragged fine-tuning batch: an odd vocabulary, a third of the positions masked out of the loss.
        _loss("loss_step_1104_bf16_n777_masked", "step", 777, 1104, 32003, "bf16", 0.3),
        # A training step of the 410M shape, float32 like the training runtime's layers.
        _loss("loss_step_1024_f32_n512", "step", 512, 1024, VOCAB, "float32"),
        # The same shape in bfloat16 on one 2048-token sequence.
        _loss("loss_step_1024_bf16_n2048", "step", 2048, 1024, VOCAB, "bf16"),
        # The largest: four 2048-token sequences of the 1.4B shape.
        _loss("loss_step_2048_bf16_n8192", "step", 8192, 2048, VOCAB, "bf16"),
        # One token of a decoded sequence through a block boundary.
        _norm("norm_decode_1024_f32_n1", "forward", 1, 1024, "float32", "layer", False, False),
        # A long bfloat16 batch of the 2.8B shape, norms on both sides of the block.
        _norm("norm_forward_2560_bf16_n8192", "forward", 8192, 2560, "bf16", "rms", True, True),
        # The backward of a training step, every gradient.
        _norm("norm_backward_1024_f32_n2048", "backward", 2048, 1024, "float32", "layer", True, True),
        # An odd width, rows that start anywhere.
        _norm("norm_backward_1001_f32_n333", "backward", 333, 1001, "float32", "rms", False, True),
        # The gradients of the smallest model's layers at 20 %, below the limit: an ordinary step, only the norm counts.
        _clip("clip_512_l6_d20_within", "within", 6, 512, 2048, 0.2, 0, "float32"),
        # The 24 layers of the 410M shape at 50 % and its bfloat16 head, above the limit, scaled into float32 buffers.
        _clip("clip_1024_l24_d50_head_beyond", "beyond", 24, 1024, 4096, 0.5, VOCAB, "bf16"),
    ]


def draw(rng):
    log = lambda low, high: math.exp(rng.uniform(math.log(low), math.log(high)))  # noqa: E731
    op = rng.choice(("loss", "loss", "norm", "clip"))
    width = rng.choice(WIDTHS) if rng.random() < 0.5 else round(log(128, 2560))
    if op == "loss":
        vocab = VOCAB if rng.random() < 0.4 else round(log(1000, 65536))
        tokens = max(1, min(round(log(1, 8192)), MOST_LOSS // (vocab * width)))
        type_ = rng.choice(("float32", "bf16", "bf16"))
        if type_ == "float32":
            tokens = min(tokens, 2048)
        return _loss("", rng.choice(("losses", "step", "step")), tokens, width, vocab, type_, rng.choice((0.0, 0.0, 0.3, 0.8)))
    if op == "norm":
        tokens = max(1, min(round(log(1, 16384)), MOST_NORM // width))
        return _norm("", rng.choice(("forward", "backward")), tokens, width, rng.choice(("float32", "bf16")),
                     rng.choice(("layer", "rms")), rng.random() < 0.5, rng.random() < 0.5)
    vocab = rng.choice((0, round(log(1000, 50304))))
    slots = 2 * 4 * width * max(1, round(0.2 * width))
    layers = max(1, min(round(log(1, 24)), (MOST_CLIP - vocab * width) // slots))
    return _clip("", rng.choice(("within", "beyond")), layers, width, 4 * width, 0.2, vocab, rng.choice(("float32", "bf16")))


# ------------------------------------------------------------------------------------------------------------- inputs

def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _normal(generator, shape, std=1.0):
    return torch.randn(shape, generator=generator, device="cuda") * std


def _loss_inputs(case, generator):
    """Hidden rows that lean towards their labels' weight rows by a few nats, as a trained model's do; labels of which
    the low ids are the frequent ones; masked positions hold the ignored label."""
    n, d, v = case["tokens"], case["d_model"], case["vocab"]
    weight = _normal(generator, (v, d), WEIGHT_STD)
    labels = (v * torch.rand(n, generator=generator, device="cuda") ** 2).long().clamp_(max=v - 1)
    lean = torch.rand((n, 1), generator=generator, device="cuda") * 8.0 / (WEIGHT_STD * WEIGHT_STD * d)
    x = _normal(generator, (n, d)) + lean * weight[labels]
    masked = torch.rand(n, generator=generator, device="cuda") < case["ignored"]
    return {"x": x.to(_type(case["type"])), "weight": weight.to(_type(case["type"])), "labels": labels.masked_fill(masked, IGNORE)}


def _norm_inputs(case, generator):
    """The residual stream with a few large channels, the block's output, parameters near one (weights) and zero
    (biases), and for the backward the gradients of r and h."""
    n, d, t = case["tokens"], case["d_model"], _type(case["type"])
    large = 1.0 + 10.0 * (torch.rand(d, generator=generator, device="cuda") < 0.01)
    state = {"f": (_normal(generator, (n, d), 0.5) + 0.1).to(t)}
    stream = (_normal(generator, (n, d)) * large + 0.2).to(t)
    state["weight"] = 1.0 + _normal(generator, d, 0.1)
    state["bias"] = _normal(generator, d, 0.1) if case["kind"] == "layer" else None
    state["gate"] = 1.0 + _normal(generator, d, 0.3) if case["gate"] else None
    state["post_weight"] = 1.0 + _normal(generator, d, 0.1) if case["post"] else None
    state["post_bias"] = _normal(generator, d, 0.1) if case["post"] and case["kind"] == "layer" else None
    if case["direction"] == "forward":
        return {"x": stream, **state}
    return {"r": stream, **state, "gr": _normal(generator, (n, d), 0.1).to(t), "gh": _normal(generator, (n, d), 0.1).to(t)}


def _clip_sizes(case):
    """Entries of every gradient: for each layer the values and biases of both sides and a norm's two; then the head's."""
    d, h = case["d_model"], case["d_ff"]
    slots = h * max(1, round(case["density"] * d))
    return [slots, h, slots, d, d, d] * case["layers"], case["vocab"] * d


def _flat(sizes, dtype):
    """One zeroed buffer and its views of the given sizes, each on a 256-byte boundary as separate allocations are."""
    step = 256 // torch.empty((), dtype=dtype).element_size()
    starts = [0]
    for size in sizes:
        starts.append(starts[-1] + -(-size // step) * step)
    flat = torch.zeros(starts[-1], dtype=dtype, device="cuda")
    return flat, [flat[start:start + size] for start, size in zip(starts, sizes)]


def _clip_inputs(case, generator):
    """Gradients of a few sizes of entry; the limit lies at twice the norm (within) or a third of it (beyond)."""
    sizes, head = _clip_sizes(case)
    body, tensors = _flat(sizes, torch.float32)
    for tensor, std in zip(tensors, (1.0, 3.0, 0.5, 2.0, 1.0, 1.0) * case["layers"]):
        tensor.normal_(0.0, GRAD_STD * std, generator=generator)
    flats = [body]
    if head:
        flat, views = _flat([head], _type(case["head"]))
        flat.copy_(_normal(generator, flat.shape, GRAD_STD))
        flat[head:] = 0
        flats, tensors = flats + [flat], tensors + views
    norm = math.sqrt(sum(float(flat.double().square().sum()) for flat in flats))
    state = {"flats": flats, "tensors": tensors, "limit": norm * (2.0 if case["direction"] == "within" else 1.0 / 3.0)}
    if case["direction"] == "beyond":
        out, views = _flat(sizes, torch.float32)
        state["outs"], state["out_tensors"] = [out], views
        if head:
            out, views = _flat([head], torch.float32)
            state["outs"], state["out_tensors"] = state["outs"] + [out], state["out_tensors"] + views
    return state


def _inputs(case, seed):
    generator = torch.Generator("cuda").manual_seed(seed)
    return {"loss": _loss_inputs, "norm": _norm_inputs, "clip": _clip_inputs}[case["op"]](case, generator)


def prepare(case, seed):
    state = {**_inputs(case, seed), "op": case["op"], "direction": case["direction"], "kind": case.get("kind")}
    if own and case["op"] == "loss":
        from hffn_amd.loss import HeadLoss
        state["head"] = HeadLoss(state["weight"], max_tokens=case["tokens"], ignore_index=IGNORE)
    if own and case["op"] == "norm":
        from hffn_amd.norm import ResidualNorm
        state["boundary"] = ResidualNorm(state["weight"], state["bias"], gate=state["gate"], post_weight=state["post_weight"],
                                         post_bias=state["post_bias"], scale=SCALE, kind=case["kind"], eps=EPS)
    return state


# --------------------------------------------------------------------------------------------------------------- run

def _run_loss(s):
    if own:
        if s["direction"] == "losses":
            return {"losses": s["head"].losses(s["x"], s["labels"])}
        loss, gx, gw = s["head"].step(s["x"], s["labels"])
        return {"loss": loss, "gx": gx, "gw": gw}
    x, weight, labels = s["x"].float(), s["weight"].float(), s["labels"]
    valid = labels != IGNORE
    at = labels.clamp(min=0)[:, None]
    logits = x @ weight.T
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    losses = torch.where(valid, (top + torch.log(total) - logits.gather(1, at))[:, 0], 0.0)
    if s["direction"] == "losses":
        return {"losses": losses}
    share = valid.float() / valid.sum().clamp(min=1)
    p = e / total
    p.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
    p *= share[:, None]
    return {"loss": (losses * share).sum(), "gx": (p @ weight).to(s["x"].dtype), "gw": (p.T @ x).to(s["weight"].dtype)}


def _plain_norm(v, kind):
    """(v less its mean for a layer norm, times its inverse deviation; the inverse deviation)."""
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    inverse = torch.rsqrt(v.square().mean(1, keepdim=True) + EPS)
    return v * inverse, inverse


def _plain_norm_back(g, hat, inverse, kind):
    """The gradient of the norm's input, from that of the normalised rows."""
    along = hat * (g * hat).mean(1, keepdim=True)
    return inverse * (g - along - g.mean(1, keepdim=True)) if kind == "layer" else inverse * (g - along)


def _run_norm(s):
    if own:
        if s["direction"] == "forward":
            r, h = s["boundary"].forward(s["x"], s["f"])
            return {"r": r, "h": h}
        gx, gf = s["boundary"].backward(s["r"], s["f"], s["gr"], s["gh"])
        return {"gx": gx, "gf": gf, "gradients": s["boundary"].gradients()}
    kind, dtype, f = s["kind"], s["f"].dtype, s["f"].float()
    post = s["post_weight"] is not None
    if post:
        f_hat, f_inverse = _plain_norm(f, kind)
        u = f_hat * s["post_weight"]
        if s["post_bias"] is not None:
            u = u + s["post_bias"]
    else:
        u = f
    if s["direction"] == "forward":
        r = s["x"].float() + SCALE * (u if s["gate"] is None else s["gate"] * u)
        h = _plain_norm(r, kind)[0] * s["weight"]
        if s["bias"] is not None:
            h = h + s["bias"]
        return {"r": r.to(dtype), "h": h.to(dtype)}
    gh = s["gh"].float()
    hat, inverse = _plain_norm(s["r"].float(), kind)
    gx = s["gr"].float() + _plain_norm_back(gh * s["weight"], hat, inverse, kind)
    gradients = {"weight": (gh * hat).sum(0)}
    if s["bias"] is not None:
        gradients["bias"] = gh.sum(0)
    gu = SCALE * gx
    if s["gate"] is not None:
        gradients["gate"] = (gu * u).sum(0)
        gu = gu * s["gate"]
    gf = gu
    if post:
        gradients["post_weight"] = (gu * f_hat).sum(0)
        if s["post_bias"] is not None:
            gradients["post_bias"] = gu.sum(0)
        gf = _plain_norm_back(gu * s["post_weight"], f_hat, f_inverse, kind)
    return {"gx": gx.to(dtype), "gf": gf.to(dtype), "gradients": gradients}


def _run_clip(s):
    """The plain form sums over each buffer whole (the gaps between its tensors are zeros)."""
    within = s["direction"] == "within"
    if own:
        from hffn_amd.clip import clip_grad_norm_
        norm = clip_grad_norm_(s["tensors"], s["limit"], out=None if within else s["out_tensors"])
        return {"norm": norm, "clipped": s["flats"] if within else s["outs"]}
    norm = torch.stack([flat.float().square().sum() for flat in s["flats"]]).sum().sqrt()
    coefficient = (s["limit"] / (norm + 1e-6)).clamp(max=1.0)
    if within:
        return {"norm": norm, "clipped": [flat.mul_(coefficient) for flat in s["flats"]]}
    return {"norm": norm, "clipped": [flat.float() * coefficient for flat in s["flats"]]}


def run(state):
    return {"loss": _run_loss, "norm": _run_norm, "clip": _run_clip}[state["op"]](state)


def work(case):
    """Inputs read once, outputs written once. The loss multiplies every counted token by every vocabulary row once
    (losses) or three times (step: logits, both gradients); the others are a few operations an entry."""
    if case["op"] == "loss":
        n, d, v, size = case["tokens"], case["d_model"], case["vocab"], 2 if case["type"] == "bf16" else 4
        step = case["direction"] == "step"
        matrices = (n * d + v * d) * size
        return {"bytes": float(matrices * (2 if step else 1) + 8 * n + (4 if step else 4 * n)),
                "flops": 2.0 * n * (1.0 - case["ignored"]) * d * v * (3 if step else 1)}
    if case["op"] == "norm":
        n, d, size = case["tokens"], case["d_model"], 2 if case["type"] == "bf16" else 4
        vectors = 1 + (case["kind"] == "layer") * (1 + case["post"]) + case["gate"] + case["post"]
        back = case["direction"] == "backward"
        return {"bytes": float(n * d * size * (6 if back else 4) + 4 * d * vectors * (2 if back else 1)),
                "flops": float(n * d * (24 if back else 10))}
    sizes, head = _clip_sizes(case)
    body, read = sum(sizes), 2 if case["head"] == "bf16" else 4
    beyond = case["direction"] == "beyond"
    return {"bytes": float((4 * body + read * head) + (4 * (body + head) if beyond else 0)),
            "flops": float((body + head) * (3 if beyond else 2))}


# ------------------------------------------------------------------------------------------------------------- exact

def _exact_loss(case, s):
    """The definition: -log softmax at the label, in pieces of the tokens; the gradients of the mean."""
    x, w, labels = s["x"].double(), s["weight"].double(), s["labels"]
    counted = (labels != IGNORE).nonzero()[:, 0]
    losses = torch.zeros(case["tokens"], dtype=torch.float64, device="cuda")
    gx, gw = torch.zeros_like(x), torch.zeros_like(w)
    for rows in counted.split(1024):
        log_p = torch.log_softmax(x[rows] @ w.T, dim=1)
        losses[rows] = -log_p[torch.arange(len(rows), device="cuda"), labels[rows]]
        if case["direction"] == "step":
            g = log_p.exp_()
            g[torch.arange(len(rows), device="cuda"), labels[rows]] -= 1.0
            g /= len(counted)
            gx[rows] = g @ w
            gw += g.T @ x[rows]
    if case["direction"] == "losses":
        return {"losses": losses}
    return {"loss": losses.sum() / max(1, len(counted)), "gx": gx, "gw": gw}


def _exact_norm(case, s):
    """The definition in float64, differentiated by autograd for the backward."""
    names = ("weight", "bias", "gate", "post_weight", "post_bias")
    p = {name: s[name].double().requires_grad_() for name in names if s[name] is not None}

    def norm(v, weight, bias):
        if case["kind"] == "layer":
            centred = v - v.mean(-1, keepdim=True)
            return centred / (v.var(-1, unbiased=False, keepdim=True) + EPS).sqrt() * weight + bias
        return v / (v.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight

    f = s["f"].double().requires_grad_()
    branch = norm(f, p["post_weight"], p.get("post_bias")) if case["post"] else f
    branch = SCALE * branch * p["gate"] if case["gate"] else SCALE * branch
    if case["direction"] == "forward":
        r = s["x"].double() + branch
        return {"r": r.detach(), "h": norm(r, p["weight"], p.get("bias")).detach()}
    r = s["r"].double().requires_grad_()  # r as stored: the branch adds to x, whose gradient is r's
    h = norm(r, p["weight"], p.get("bias"))
    first = [name for name in ("weight", "bias") if name in p]
    g_r, *g_first = torch.autograd.grad(h, [r, *(p[name] for name in first)], s["gh"].double())
    g_r = g_r + s["gr"].double()
    rest = [name for name in ("gate", "post_weight", "post_bias") if name in p]
    g_f, *g_rest = torch.autograd.grad(branch, [f, *(p[name] for name in rest)], g_r)
    return {"gx": g_r, "gf": g_f, "gradients": dict(zip(first + rest, g_first + g_rest))}


def _exact_clip(case, s):
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(t.double()) for t in s["tensors"]]))
    factor = min(1.0, s["limit"] / (float(norm) + 1e-6))
    return {"norm": norm, "clipped": [flat.double() * factor for flat in s["flats"]]}


def exact(case, seed):
    return {"loss": _exact_loss, "norm": _exact_norm, "clip": _exact_clip}[case["op"]](case, _inputs(case, seed))
