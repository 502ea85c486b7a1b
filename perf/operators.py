"""Timed cases of the training operators around a large vocabulary: layer norm, the vocabulary's softmax cross entropy
taken in pieces without keeping the logits, and AdamW with its moments held in 8 bits.

Each case runs in a plain form (elementary torch operations in 32 bits) or through the framework's own entry points
(`own`), on the same inputs, and `exact` gives the operator's definition in 64 bits."""
import math
import random

import numpy as np
import torch

own = False

BLOCK = 256                     # elements that share one scale of the 8-bit moments
GOLDEN = 0x9E3779B97F4A7C15     # SplitMix64's increment
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
MODEL = {"beta1": 0.9, "beta2": 0.95, "learning_rate": 3e-4, "epsilon": 1e-8, "weight_decay": 0.1, "max_norm": 1.0}


def listed():
    return [
        # One token's row of the width-768 model while it generates: launch latency.
        {"name": "ln_fwd_token", "op": "layer_norm", "backward": False, "rows": 1, "cols": 768, "type": "f32"},
        # The width-768 model's training micro-batch of 32 x 2048 tokens: memory bandwidth.
        {"name": "ln_fwd_step", "op": "layer_norm", "backward": False, "rows": 65536, "cols": 768, "type": "bf16"},
        # The width-256 model's micro-batch of 8 x 512 tokens, in the f32 the reference model keeps.
        {"name": "ln_bwd_small", "op": "layer_norm", "backward": True, "rows": 4096, "cols": 256, "type": "f32"},
        # The width-768 micro-batch's gradient with the reduction of the gain's and bias's gradients.
        {"name": "ln_bwd_step", "op": "layer_norm", "backward": True, "rows": 65536, "cols": 768, "type": "bf16"},
        # A packed batch of odd length and a wide, odd feature count: no row starts on a vector boundary.
        {"name": "ln_bwd_odd", "op": "layer_norm", "backward": True, "rows": 3001, "cols": 5003, "type": "bf16"},
        # Scoring one generated token against a medium vocabulary: one pass over the weight.
        {"name": "ce_loss_token", "op": "cross_entropy", "gradients": False, "rows": 1, "width": 768,
         "vocabulary": 32000, "type": "bf16", "storage": "transposed"},
        # Perplexity of an evaluation batch over an odd-sized vocabulary.
        {"name": "ce_loss_eval", "op": "cross_entropy", "gradients": False, "rows": 4096, "width": 512,
         "vocabulary": 50021, "type": "bf16", "storage": "transposed"},
        # f32 training of the width-256 model with a small odd vocabulary and a ragged token count.
        {"name": "ce_grad_f32", "op": "cross_entropy", "gradients": True, "rows": 1021, "width": 256,
         "vocabulary": 10007, "type": "f32", "storage": "transposed"},
        # A bf16 training micro-batch whose output layer is stored [width, vocabulary] like the model's Linear.
        {"name": "ce_grad_step", "op": "cross_entropy", "gradients": True, "rows": 8192, "width": 768,
         "vocabulary": 32768, "type": "bf16", "storage": "row_major"},
        # The largest: a long micro-batch over a large tied vocabulary, whose logits alone would be 8.6 GB in f32.
        {"name": "ce_grad_large", "op": "cross_entropy", "gradients": True, "rows": 16384, "width": 768,
         "vocabulary": 131072, "type": "bf16", "storage": "transposed"},
        # Many ragged tensors of a small model with bf16 gradients: launch latency and block tails.
        {"name": "adamw8_ragged", "op": "adamw8", "blocks": 6, "width": 250, "ffn": 1001, "head": 1027,
         "gradient": "bf16"},
        # The width-768 model's 111.8 million parameters with f32 gradients.
        {"name": "adamw8_model", "op": "adamw8", "blocks": 12, "width": 768, "ffn": 3072, "head": 16384,
         "gradient": "f32"},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "cross_entropy", "cross_entropy", "adamw8"])
    if op == "layer_norm":
        cols = _log(rng, 64, 8192)
        if rng.random() < 0.5:
            cols = max(64, cols // 8 * 8)
        rows = _log(rng, 1, min(65536, 65536 * 768 // cols))
        return {"op": op, "backward": rng.random() < 0.6, "rows": rows, "cols": cols,
                "type": rng.choice(["f32", "bf16"])}
    if op == "cross_entropy":
        kind = rng.choice(["f32", "bf16", "bf16"])
        width = 8 * _log(rng, 8, 128)
        if rng.random() < 0.15:
            width += rng.choice([1, 2, 3, 4])
        vocabulary = _log(rng, 1000, 131072)
        rows = _log(rng, 1, min(16384, int((2e11 if kind == "f32" else 1.6e12) / (width * vocabulary))))
        return {"op": op, "gradients": rng.random() < 0.6, "rows": rows, "width": width, "vocabulary": vocabulary,
                "type": kind, "storage": rng.choice(["transposed", "transposed", "row_major"])}
    width = _log(rng, 48, 768)
    return {"op": op, "blocks": rng.randint(1, 12), "width": width, "ffn": 4 * width + rng.choice([0, 0, 1, 5]),
            "head": _log(rng, 256, 16384), "gradient": rng.choice(["f32", "bf16"])}


# ------------------------------------------------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tensors(case):
    """(elements, decayed) of every parameter tensor of the decoder the case describes."""
    w, f, h = case["width"], case["ffn"], case["head"]
    block = [(w * 3 * w, True), (3 * w, False), (w * w, True), (w, False), (w * f, True), (f, False), (f * w, True),
             (w, False), (w, False), (w, False)]
    return block * case["blocks"] + [(w * h, True), (h, False), (w, False)]


def _starts(case):
    """First element of every tensor in the flat arrays, each on a block boundary, and the arrays' length."""
    starts, at = [], 0
    for n, _ in _tensors(case):
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return starts, at


def prepare(case, seed):
    g = _generator(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    if case["op"] == "layer_norm":
        rows, cols, dtype = case["rows"], case["cols"], TYPES[case["type"]]
        # A residual stream: a few channels far larger than the rest, and a mean that is not zero.
        channel = 1.0 + 8.0 * (torch.rand(cols, generator=g, device="cuda") < 0.01)
        x = torch.randn(rows, cols, generator=g, device="cuda")
        state = {"case": case, "input": (x.mul_(channel).add_(0.25 * channel)).to(dtype),
                 "gain": normal(cols, std=0.2).add_(1.0), "bias": normal(cols, std=0.1), "epsilon": 1e-5}
        if case["backward"]:
            wide = state["input"].float()
            mean = wide.mean(1)
            state["mean"], state["inv_std"] = mean, (wide - mean[:, None]).square().mean(1).add(1e-5).rsqrt()
            state["output_grad"] = normal(rows, cols, std=1e-2, dtype=dtype)
        return state
    if case["op"] == "cross_entropy":
        rows, width, vocabulary, dtype = case["rows"], case["width"], case["vocabulary"], TYPES[case["type"]]
        w = normal(vocabulary, width, std=width ** -0.5)
        targets = torch.randint(0, vocabulary, (rows,), generator=g, device="cuda", dtype=torch.int32)
        # A model part of the way through training: the right token leads by up to a few nats.
        lead = 8.0 * torch.rand(rows, 1, generator=g, device="cuda")
        hidden = normal(rows, width) + lead * w[targets.long()]
        if rows > 1:
            # Padding and prompt tokens carry no target.
            targets.masked_fill_(torch.rand(rows, generator=g, device="cuda") < 0.05, -1)
        weight = w.to(dtype) if case["storage"] == "transposed" else w.t().contiguous().to(dtype)
        return {"case": case, "hidden": hidden.to(dtype), "weight": weight, "targets": targets,
                "grad_scale": 1.0 / rows}
    starts, total = _starts(case)
    blocks = total // BLOCK
    live = torch.zeros(total, device="cuda", dtype=torch.bool)
    decay = torch.zeros(blocks, device="cuda")
    for (n, decayed), at in zip(_tensors(case), starts):
        live[at:at + n] = True
        decay[at // BLOCK:(at + n + BLOCK - 1) // BLOCK] = MODEL["weight_decay"] if decayed else 0.0
    # Gradients whose size differs from block to block, and moments that fit them.
    spread = torch.exp(normal(blocks)).mul_(1e-3)
    gradient = normal(blocks, BLOCK).mul_(spread[:, None]).view(-1).mul_(live)
    first = normal(total, std=32.0).round_().clamp_(-127, 127).mul_(live).to(torch.int8)
    second = normal(total, std=40.0).add_(120.0).round_().clamp_(1, 255).mul_(live).to(torch.uint8)
    parameter = normal(total, std=0.02).mul_(live)
    return {"case": case, "parameter": parameter, "shadow": parameter.to(torch.bfloat16),
            "gradient": gradient.to(TYPES[case["gradient"]]), "first": first, "first_scale": 2.0 * spread,
            "second": second, "second_scale": spread.square().mul_(6.0), "decay": decay, "step": 100,
            "seed": seed * 1000003}


# ------------------------------------------------------------------------------------------------------- plain forms


def _layer_norm_plain(s):
    x = s["input"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    inv_std = torch.rsqrt((centred * centred).mean(1, keepdim=True) + s["epsilon"])
    y = centred * inv_std * s["gain"] + s["bias"]
    return {"output": y.to(s["input"].dtype), "mean": mean[:, 0], "inv_std": inv_std[:, 0]}


def _layer_norm_grad_plain(s):
    x, dy = s["input"].float(), s["output_grad"].float()
    inv_std = s["inv_std"][:, None]
    normal = (x - s["mean"][:, None]) * inv_std
    dn = dy * s["gain"]
    dx = inv_std * (dn - dn.mean(1, keepdim=True) - normal * (dn * normal).mean(1, keepdim=True))
    return {"input_grad": dx.to(s["input"].dtype), "gain_grad": (dy * normal).sum(0), "bias_grad": dy.sum(0)}


def _cross_entropy_plain(s):
    case = s["case"]
    hidden = s["hidden"].float()
    weight = s["weight"].float() if case["storage"] == "transposed" else s["weight"].float().t()
    logits = hidden @ weight.t()
    top = logits.amax(1, keepdim=True)
    partition = top + torch.log(torch.exp(logits - top).sum(1, keepdim=True))
    live = s["targets"] >= 0
    at = s["targets"].long().clamp(min=0)[:, None]
    losses = torch.where(live, (partition - logits.gather(1, at))[:, 0], 0.0)
    out = {"losses": losses, "loss_sum": losses.sum()}
    if case["gradients"]:
        grad = torch.exp(logits.sub_(partition))
        grad.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float32))
        grad *= torch.where(live, s["grad_scale"], 0.0)[:, None]
        out["d_hidden"] = (grad @ weight).to(s["hidden"].dtype)
        d_weight = grad.t() @ hidden if case["storage"] == "transposed" else hidden.t() @ grad
        out["d_weight"] = d_weight.to(s["weight"].dtype)
    return out


def _draws(seed, total):
    """32 random bits for each element: the halves of SplitMix64's outputs, two elements to an output."""
    def wrap(v):
        v &= (1 << 64) - 1
        return v - (1 << 64) if v >= 1 << 63 else v

    z = torch.arange(1, total // 2 + 1, device="cuda", dtype=torch.int64) * wrap(GOLDEN) + wrap(seed)
    z = (z ^ ((z >> 30) & ((1 << 34) - 1))) * wrap(0xBF58476D1CE4E5B9)
    z = (z ^ ((z >> 27) & ((1 << 37) - 1))) * wrap(0x94D049BB133111EB)
    z = z ^ ((z >> 31) & ((1 << 33) - 1))
    return torch.stack([z & 0xFFFFFFFF, (z >> 32) & 0xFFFFFFFF], 1).view(-1)


def _first_level(q, dtype):
    """The share of its block's scale that a magnitude code of the first moment stands for: (q / 127)^2."""
    return (q * q).to(dtype) * (1.0 / 16129.0)


def _second_level(q, dtype):
    """The same for the second moment: (q / 255)^4."""
    s = (q * q).to(dtype) * (1.0 / 65025.0)
    return s * s


def _encode(values, most, level, root, bits):
    """(magnitude codes, scales) of values >= 0 in blocks: each value goes to one of the two levels around it, to the
    upper one with the probability that keeps its expectation (`bits`: 16 random bits)."""
    blocks = values.view(-1, BLOCK)
    scale = blocks.amax(1)
    scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
    inverse = torch.where(scale > 0, 1.0 / scale, 0.0)
    share = (blocks * inverse[:, None]).view(-1)
    q = torch.where(share > 0, root(share) * most, 0.0).clamp(max=most - 1).to(torch.int32)
    q = (q - (level(q, share.dtype) > share).to(torch.int32)).clamp(min=0)
    q = (q + (level(q + 1, share.dtype) <= share).to(torch.int32)).clamp(max=most - 1)
    low = level(q, share.dtype)
    threshold = low + ((bits.to(share.dtype) + 0.5) * (1.0 / 65536.0)) * (level(q + 1, share.dtype) - low)
    return q + (threshold < share).to(torch.int32), scale


def _adamw8_values(s, dtype):
    """One step's results from the state, in `dtype`: (parameter, first codes and scales, second codes and scales)."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    b1, b2 = f(MODEL["beta1"]), f(MODEL["beta2"])
    nb1, nb2 = f(np.float32(1) - np.float32(b1)), f(np.float32(1) - np.float32(b2))
    step = s["step"]
    c1, c2 = f(1.0 - b1 ** step), f(1.0 - b2 ** step)
    g = s["gradient"].to(dtype)
    norm = torch.sqrt(s["gradient"].double().square().sum()).to(dtype)
    g = g * torch.where(norm > MODEL["max_norm"], MODEL["max_norm"] / norm, 1.0)
    q1, q2 = s["first"].to(torch.int32), s["second"].to(torch.int32)
    m = (torch.sign(q1) * _first_level(q1, dtype)).view(-1, BLOCK) * s["first_scale"].to(dtype)[:, None]
    v = _second_level(q2, dtype).view(-1, BLOCK) * s["second_scale"].to(dtype)[:, None]
    m = m.view(-1) * b1 + g * nb1
    v = v.view(-1) * b2 + (g * nb2) * g
    update = (m / c1) / (torch.sqrt(v / c2) + f(MODEL["epsilon"]))
    w = s["parameter"].to(dtype).view(-1, BLOCK)
    w = (w - f(MODEL["learning_rate"]) * (update.view(-1, BLOCK) + s["decay"].to(dtype)[:, None] * w)).view(-1)
    bits = _draws(s["seed"] + step, m.numel())
    first, first_scale = _encode(m.abs(), 127, _first_level, torch.sqrt, bits & 0xFFFF)
    first = torch.where(m < 0, -first, first)
    second, second_scale = _encode(v, 255, _second_level, lambda x: torch.sqrt(torch.sqrt(x)), bits >> 16)
    second = torch.where(v > 0, second.clamp(min=1), second)
    return w, first, first_scale, second, second_scale


def _moments(first, first_scale, second, second_scale):
    dtype = first_scale.dtype
    m = (torch.sign(first) * _first_level(first, dtype)).view(-1, BLOCK) * first_scale[:, None]
    return m.view(-1), (_second_level(second, dtype).view(-1, BLOCK) * second_scale[:, None]).view(-1)


def _adamw8_plain(s):
    s["step"] += 1
    w, first, first_scale, second, second_scale = _adamw8_values(s, torch.float32)
    s["parameter"].copy_(w)
    s["shadow"].copy_(w)
    s["first"].copy_(first)
    s["second"].copy_(second)
    s["first_scale"].copy_(first_scale)
    s["second_scale"].copy_(second_scale)
    m, v = _moments(first, first_scale, second, second_scale)
    return {"parameter": s["parameter"], "shadow": s["shadow"], "first": m, "second": v}


# ------------------------------------------------------------------------------------------------------- the framework


def _gpu(s):
    from staleynet_b200.matmul import Gpu

    if "gpu" not in s:
        s["gpu"] = Gpu(0)
    return s["gpu"]


def _buffer(s, name, shape, dtype):
    """An output or workspace that the caller keeps from pass to pass."""
    if name not in s:
        s[name] = torch.empty(shape, device="cuda", dtype=dtype)
    return s[name]


def _layer_norm_own(s):
    gpu, x = _gpu(s), s["input"]
    out = _buffer(s, "output", x.shape, x.dtype)
    mean, inv_std = _buffer(s, "out_mean", x.shape[:1], torch.float32), _buffer(s, "out_inv", x.shape[:1],
                                                                              torch.float32)
    gpu.layer_norm_forward(x, s["gain"], s["bias"], out, mean, inv_std, s["epsilon"])
    return {"output": out, "mean": mean, "inv_std": inv_std}


def _layer_norm_grad_own(s):
    gpu, x = _gpu(s), s["input"]
    if "workspace" not in s:
        _buffer(s, "workspace", (gpu.layer_norm_workspace(*x.shape),), torch.uint8)
    dx = _buffer(s, "input_grad", x.shape, x.dtype)
    dg, db = _buffer(s, "gain_grad", x.shape[1:], torch.float32), _buffer(s, "bias_grad", x.shape[1:], torch.float32)
    gpu.layer_norm_backward(s["output_grad"], x, s["gain"], s["mean"], s["inv_std"], dx, dg, db, s["workspace"])
    return {"input_grad": dx, "gain_grad": dg, "bias_grad": db}


def _cross_entropy_own(s):
    from staleynet_b200.matmul import Storage

    gpu, case, x, w = _gpu(s), s["case"], s["hidden"], s["weight"]
    storage = Storage.TRANSPOSED if case["storage"] == "transposed" else Storage.ROW_MAJOR
    losses = _buffer(s, "losses", x.shape[:1], torch.float32)
    total = _buffer(s, "loss_sum", (), torch.float32)
    dx = dw = None
    if case["gradients"]:
        dx, dw = _buffer(s, "d_hidden", x.shape, x.dtype), _buffer(s, "d_weight", w.shape, w.dtype)
    if "workspace" not in s:
        need = gpu.vocabulary_cross_entropy_workspace(x, w, storage=storage, d_hidden=dx, d_weight=dw)
        _buffer(s, "workspace", (need,), torch.uint8)
    gpu.vocabulary_cross_entropy(x, w, s["targets"], losses, total, s["workspace"], storage=storage, d_hidden=dx,
                                 d_weight=dw, grad_scale=s["grad_scale"])
    out = {"losses": losses, "loss_sum": total}
    return out | {"d_hidden": dx, "d_weight": dw} if case["gradients"] else out


def _adamw8_own(s):
    from staleynet_b200.adamw8 import AdamW8, AdamW8Tensor
    from staleynet_b200.matmul import AdamWHyperparameters

    if "plan" not in s:
        starts, total = _starts(s["case"])
        s["first_out"], s["second_out"] = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
        tensors, outs = [], []
        for (n, decayed), at in zip(_tensors(s["case"]), starts):
            part, blocks = slice(at, at + n), slice(at // BLOCK, (at + n + BLOCK - 1) // BLOCK)
            tensors.append(AdamW8Tensor(
                parameter=s["parameter"][part], gradient=s["gradient"][part], first=s["first"][part],
                first_scale=s["first_scale"][blocks], second=s["second"][part],
                second_scale=s["second_scale"][blocks], shadow=s["shadow"][part],
                weight_decay=MODEL["weight_decay"] if decayed else 0.0, first_draw=at // 2))
            outs.append((s["first_out"][part], s["second_out"][part]))
        s["plan"], s["outs"] = AdamW8(_gpu(s), tensors), outs
        s["plan"].bind_moments(outs)
    s["step"] += 1
    hyper = AdamWHyperparameters(MODEL["learning_rate"], MODEL["beta1"], MODEL["beta2"], MODEL["epsilon"], 0.0,
                                 s["step"])
    s["plan"].step(hyper, MODEL["max_norm"], s["seed"] + s["step"])
    s["plan"].moments()
    return {"parameter": s["parameter"], "shadow": s["shadow"], "first": s["first_out"], "second": s["second_out"]}


def run(state):
    case = state["case"]
    if case["op"] == "layer_norm":
        if case["backward"]:
            return _layer_norm_grad_own(state) if own else _layer_norm_grad_plain(state)
        return _layer_norm_own(state) if own else _layer_norm_plain(state)
    if case["op"] == "cross_entropy":
        return _cross_entropy_own(state) if own else _cross_entropy_plain(state)
    return _adamw8_own(state) if own else _adamw8_plain(state)


# ------------------------------------------------------------------------------------------------------- definitions


def _exact_layer_norm(s):
    out = {"output": [], "mean": [], "inv_std": []}
    for x in s["input"].split(8192):
        x = x.double()
        mu = x.sum(1) / x.shape[1]
        variance = ((x - mu[:, None]) ** 2).sum(1) / x.shape[1]
        scale = 1.0 / torch.sqrt(variance + s["epsilon"])
        out["output"].append((x - mu[:, None]) * scale[:, None] * s["gain"].double() + s["bias"].double())
        out["mean"].append(mu)
        out["inv_std"].append(scale)
    return {k: torch.cat(v) for k, v in out.items()}


def _exact_layer_norm_grad(s):
    cols = s["input"].shape[1]
    gain, dg, db, dx = s["gain"].double(), 0.0, 0.0, []
    for at in range(0, s["input"].shape[0], 8192):
        part = slice(at, at + 8192)
        x, dy = s["input"][part].double(), s["output_grad"][part].double()
        inv = s["inv_std"][part].double()[:, None]
        n = (x - s["mean"][part].double()[:, None]) * inv
        dg, db = dg + (dy * n).sum(0), db + dy.sum(0)
        d = dy * gain
        dx.append(inv * (d - d.sum(1, keepdim=True) / cols - n * ((d * n).sum(1, keepdim=True) / cols)))
    return {"input_grad": torch.cat(dx), "gain_grad": dg, "bias_grad": db}


def _exact_cross_entropy(s):
    case = s["case"]
    w = s["weight"].double() if case["storage"] == "transposed" else s["weight"].double().t().contiguous()
    losses, d_hidden, d_weight = [], [], torch.zeros_like(w) if case["gradients"] else None
    rows = max(1, int(1e9) // w.shape[0])
    for h, t in zip(s["hidden"].split(rows), s["targets"].split(rows)):
        h, live = h.double(), t >= 0
        z = h @ w.t()
        partition = torch.logsumexp(z, 1)
        index = torch.arange(len(t), device="cuda")[live]
        loss = torch.zeros(len(t), device="cuda", dtype=torch.float64)
        loss[live] = partition[live] - z[index, t[live].long()]
        losses.append(loss)
        if case["gradients"]:
            p = torch.softmax(z, 1)
            p[index, t[live].long()] -= 1.0
            p[~live] = 0.0
            p *= s["grad_scale"]
            d_hidden.append(p @ w)
            d_weight += p.t() @ h
    losses = torch.cat(losses)
    out = {"losses": losses, "loss_sum": losses.sum()}
    if case["gradients"]:
        out["d_hidden"] = torch.cat(d_hidden)
        out["d_weight"] = d_weight if case["storage"] == "transposed" else d_weight.t().contiguous()
    return out


def _exact_adamw8(s):
    """The random bits in numpy's unsigned integers, the codes by a search among the levels."""
    f = lambda v: float(np.float32(v))  # noqa: E731
    b1, b2, step = f(MODEL["beta1"]), f(MODEL["beta2"]), s["step"] + 1
    levels = [(torch.arange(n, device="cuda", dtype=torch.float64) / (n - 1)) ** p for n, p in ((128, 2), (256, 4))]
    g = s["gradient"].double()
    norm = math.sqrt(float(torch.dot(g, g)))
    g = g * (MODEL["max_norm"] / norm if norm > MODEL["max_norm"] else 1.0)
    q = s["first"].long()
    m = torch.sign(q) * levels[0][q.abs()] * s["first_scale"].double().repeat_interleave(BLOCK)
    v = levels[1][s["second"].long()] * s["second_scale"].double().repeat_interleave(BLOCK)
    m, v = b1 * m + (1.0 - b1) * g, b2 * v + (1.0 - b2) * g * g
    rate = m / (1.0 - b1 ** step) / (torch.sqrt(v / (1.0 - b2 ** step)) + f(MODEL["epsilon"]))
    w = s["parameter"].double()
    w = w - f(MODEL["learning_rate"]) * (rate + s["decay"].double().repeat_interleave(BLOCK) * w)
    z = np.arange(1, len(m) // 2 + 1, dtype=np.uint64) * np.uint64(GOLDEN) + np.uint64((s["seed"] + step) % (1 << 64))
    z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    halves = (z ^ (z >> np.uint64(31))).view(np.uint16).astype(np.int32).reshape(-1, 2)

    def hold(values, level, low16):
        scale = values.view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)
        share = torch.where(scale > 0, values / scale, 0.0)
        at = (torch.searchsorted(level, share, right=True) - 1).clamp(0, len(level) - 2)
        chance = (share - level[at]) / (level[at + 1] - level[at])
        return at + ((torch.from_numpy(low16).cuda().double() + 0.5) / 65536.0 < chance), scale

    first, scale1 = hold(m.abs(), levels[0], np.ascontiguousarray(halves[:, 0]))
    second, scale2 = hold(v, levels[1], np.ascontiguousarray(halves[:, 1]))
    second = torch.where(v > 0, second.clamp(min=1), second)
    return {"parameter": w, "shadow": w, "first": torch.sign(m) * levels[0][first] * scale1,
            "second": levels[1][second] * scale2}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        return _exact_layer_norm_grad(s) if case["backward"] else _exact_layer_norm(s)
    if case["op"] == "cross_entropy":
        return _exact_cross_entropy(s)
    return _exact_adamw8(s)


def work(case):
    if case["op"] == "layer_norm":
        n, size = case["rows"] * case["cols"], SIZE[case["type"]]
        if case["backward"]:
            return {"bytes": 3 * n * size + 8 * case["rows"] + 12 * case["cols"], "flops": 14 * n}
        return {"bytes": 2 * n * size + 8 * case["rows"] + 8 * case["cols"], "flops": 8 * n}
    if case["op"] == "cross_entropy":
        n, size = (case["rows"] + case["vocabulary"]) * case["width"], SIZE[case["type"]]
        product = 2 * case["rows"] * case["width"] * case["vocabulary"]
        if case["gradients"]:
            return {"bytes": 2 * n * size + 8 * case["rows"], "flops": 3 * product}
        return {"bytes": n * size + 8 * case["rows"], "flops": product}
    # Read: parameter, gradient, two codes; written: parameter, its bf16 copy, two codes, two moments' values.
    n = sum(count for count, _ in _tensors(case))
    return {"bytes": n * (4 + SIZE[case["gradient"]] + 2 + 4 + 2 + 2 + 8) + n // BLOCK * 16, "flops": 60 * n}


if __name__ == "__main__":
    print([c["name"] for c in listed()], draw(random.Random(0)))
