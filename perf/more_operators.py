"""Performance cases of the leaf encoder's block and of what it learns from and
is served with: the gated feed-forward block with its gradient, products in 8
bits with a scale for each 128 values, and the distillation of a teacher's top
logits.

Each case is a dict of plain values; `kind` names the call:

- forward: y = (act(x Wg^T) * (x Wu^T)) Wd^T, three matrices;
- gradient: the gradients of x and the matrices, from what a forward pass kept;
- step: both, as in a training step;
- product8: rows rounded to e4m3 with a power of two for each 128 values, times
  a weight kept that way;
- serve8: the block with all three matrices kept that way, as it is served;
- loss: each row's Kullback-Leibler divergence from a teacher's top logits;
- loss_gradient: the logits' gradient;
- loss_step: both.

With `own` false the operators run in their plain form, elementary torch
operations in 32 bits; with `own` true as `xgboost.encoder` has them.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BLOCK = 128
_package = None


def _encoder():
    global _package
    if _package is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "xgboost-metal_amd", "python"))
        from xgboost import encoder
        _package = encoder
    return _package


def _block(name, kind, rows, dim, hidden, dtype, activation="silu"):
    return {"name": name, "kind": kind, "rows": rows, "dim": dim, "hidden": hidden, "dtype": dtype,
            "activation": activation}


def _product(name, rows, dim, out, dtype):
    return {"name": name, "kind": "product8", "rows": rows, "dim": dim, "out": out, "dtype": dtype}


def _distil(name, kind, rows, classes, top, dtype, temperature):
    return {"name": name, "kind": kind, "rows": rows, "classes": classes, "top": top, "dtype": dtype,
            "temperature": temperature}


def listed():
    return [
        # One request of a service through a small encoder's block.
        _block("forward_request_16x64x256", "forward", 16, 64, 256, "f32"),
        # A single row through a wide block: the matrices are read for it alone.
        _block("forward_row_1x1024x4096", "forward", 1, 1024, 4096, "bf16"),
        # Encoding a large batch.
        _block("forward_batch_8192x1024x4096", "forward", 8192, 1024, 4096, "f16", "gelu"),
        # Backward pass at odd sizes, in the encoder's default type.
        _block("gradient_odd_2003x200x777", "gradient", 2003, 200, 777, "f32"),
        # Forward and backward of a training step on a large batch.
        _block("step_16384x1024x4096", "step", 16384, 1024, 4096, "bf16"),
        # A projection of odd sizes, served in 8 bits.
        _product("product8_odd_700x1000x1501", 700, 1000, 1501, "f32"),
        # A large one, where the matrix instructions' rate counts.
        _product("product8_8192x4096x4096", 8192, 4096, 4096, "bf16"),
        # The block in 8 bits: a single row, and a batch.
        _block("serve8_row_1x1024x4096", "serve8", 1, 1024, 4096, "bf16"),
        _block("serve8_batch_4096x1024x4096", "serve8", 4096, 1024, 4096, "bf16"),
        # A mini-batch of a classifier learning from one model a class.
        _distil("loss_64x1000", "loss", 64, 1000, 10, "f32", 2.0),
        # Odd sizes, backward alone.
        _distil("loss_gradient_1021x30011", "loss_gradient", 1021, 30011, 32, "f16", 1.0),
        # A training step over a large table of tokens.
        _distil("loss_step_8192x32768", "loss_step", 8192, 32768, 64, "bf16", 1.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _dim(rng, low, high):
    # Mostly whole vectors of 8 values, sometimes any width.
    d = _log_int(rng, low, high)
    return d if rng.random() < 0.3 else max(8, d // 8 * 8)


def draw(rng):
    kind = rng.choice(["forward", "forward", "gradient", "step", "product8", "product8", "serve8", "serve8", "loss",
                       "loss_gradient", "loss_step"])
    # The block in 8 bits is served in 16: its hidden values lie next to borders of
    # e4m3's, where the last bits of any sum in 32 decide, and 24 would show that.
    case = {"kind": kind, "dtype": rng.choice(["bf16", "f16"] if kind == "serve8" else ["f32", "bf16", "bf16", "f16"])}
    if kind in ("forward", "gradient", "step", "serve8"):
        # Rows times both widths stay below the listed ones'; binary32 is slower.
        dim, hidden = _dim(rng, 16, 2048), _dim(rng, 32, 6144)
        most = 16384 * 1024 * 4096 // (8 if case["dtype"] == "f32" else 2)
        case.update(rows=_log_int(rng, 1, max(2, min(16384, most // (dim * hidden)))), dim=dim, hidden=hidden,
                    activation=rng.choice(["silu", "silu", "gelu"]))
    elif kind == "product8":
        dim, out = _dim(rng, 32, 8192), _dim(rng, 16, 8192)
        most = 8192 * 4096 * 4096 // 2
        case.update(rows=_log_int(rng, 1, max(2, min(16384, most // (dim * out)))), dim=dim, out=out)
    else:
        classes = _log_int(rng, 10, 131072)
        case.update(rows=_log_int(rng, 1, min(16384, 8192 * 32768 // 2 // classes)), classes=classes,
                    top=_log_int(rng, 1, min(classes, 128)), temperature=rng.choice([1.0, 1.0, 2.0, 0.7]))
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _generator(seed)
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    rows = case["rows"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = {"kind": kind, "dtype": dtype}
    if kind.startswith("loss"):
        classes, top = case["classes"], case["top"]
        # The teacher is sure of some rows and not of others, the student on its way there.
        teacher = normal(rows, classes).mul_(1.0 + 3.0 * torch.rand(rows, 1, generator=g, device="cuda"))
        values, indices = teacher.topk(top, 1)
        state["logits"] = (0.6 * teacher + normal(rows, classes)).to(dtype)
        # Some rows are padding: the teacher says nothing of them.
        absent = torch.rand(rows, 1, generator=g, device="cuda") < 0.02
        state["indices"] = torch.where(absent, -1, indices)
        state["values"] = values.to(dtype)
        state["temperature"] = case["temperature"]
        if kind != "loss":
            # Of a mean over the rows; binary16 trains with the loss scaled.
            scale = 16384.0 if dtype == torch.float16 else 1.0
            state["grad"] = (0.5 + torch.rand(rows, generator=g, device="cuda")) * (scale / rows)
        if kind == "loss_gradient":
            state["lse"] = (state["logits"].double() / case["temperature"]).logsumexp(1).float()
        return state
    dim = case["dim"]
    # Rows as a norm leaves them, a few columns larger than the others.
    x = normal(rows, dim) * (1.0 + 4.0 * (torch.rand(dim, generator=g, device="cuda") < 0.02))
    state["x"] = x.to(dtype)
    if kind == "product8":
        state["weight"] = _keep8((normal(case["out"], dim) * dim ** -0.5).to(dtype))
        return state
    hidden = case["hidden"]
    state["activation"] = case["activation"]
    matrices = [(normal(hidden, dim) * dim ** -0.5).to(dtype), (normal(hidden, dim) * dim ** -0.5).to(dtype),
                (normal(dim, hidden) * hidden ** -0.5).to(dtype)]
    if kind == "serve8":
        matrices = [_keep8(m) for m in matrices]
    state["gate"], state["up"], state["down"] = matrices
    if kind in ("gradient", "step"):
        state["grad"] = normal(rows, dim).to(dtype)
    if kind == "gradient":
        v = state["x"].float()
        state["kept"] = torch.stack([v @ state["gate"].float().t(), v @ state["up"].float().t()], 1)
    return state


def _keep8(weight):
    """What a program that serves keeps of a weight."""
    return _encoder().quantize_blocks(weight) if own else _plain_quantize(weight)


def _plain_quantize(x):
    """(e4m3 values, their scales): of each 128 values the smallest power of two
    that takes the largest to at most 448."""
    rows, dim = x.shape
    blocks = (dim + _BLOCK - 1) // _BLOCK
    v = torch.zeros(rows, blocks * _BLOCK, device=x.device)
    v[:, :dim] = x
    v = v.view(rows, blocks, _BLOCK)
    mantissa, exponent = torch.frexp(v.abs().amax(2))  # mantissa within [0.5, 1)
    exponent = exponent - 9 + (mantissa > 0.875)
    exponent = torch.where(mantissa == 0, 0, exponent.clamp(-127, 127))
    # Two factors: a power of two below 2^-126 has no reciprocal in 32 bits.
    half = -exponent // 2
    v = torch.ldexp(torch.ldexp(v, half[..., None]), (-exponent - half)[..., None])
    return v.to(torch.float8_e4m3fn), exponent, dim


def _plain_values(kept):
    values, exponent, dim = kept
    v = torch.ldexp(values.float(), exponent[..., None])
    return v.flatten(1)[:, :dim]


def _plain_activation(g, activation):
    if activation == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))


def _plain_slope(g, activation):
    if activation == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    return 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_forward(s):
    x = s["x"].float()
    gate, up = x @ s["gate"].float().t(), x @ s["up"].float().t()
    y = (_plain_activation(gate, s["activation"]) * up) @ s["down"].float().t()
    return y.to(s["dtype"]), gate, up


def _plain_gradient(s, gate, up):
    x, grad = s["x"].float(), s["grad"].float()
    act = _plain_activation(gate, s["activation"])
    dhidden = grad @ s["down"].float()
    dgate, dup = dhidden * up * _plain_slope(gate, s["activation"]), dhidden * act
    dx = dgate @ s["gate"].float() + dup @ s["up"].float()
    results = dx, dgate.t() @ x, dup.t() @ x, grad.t() @ (act * up)
    return tuple(r.to(s["dtype"]) for r in results)


def _plain_serve8(s):
    x = _plain_values(_plain_quantize(s["x"]))
    hidden = _plain_activation(x @ _plain_values(s["gate"]).t(), s["activation"]) * (x @ _plain_values(s["up"]).t())
    return (_plain_values(_plain_quantize(hidden)) @ _plain_values(s["down"]).t()).to(s["dtype"])


def _plain_teacher(s):
    """The teacher's probabilities, their logarithms (0 where there is none), and the columns."""
    classes = s["logits"].shape[1]
    present = (s["indices"] >= 0) & (s["indices"] < classes)
    t = torch.where(present, s["values"].float() / s["temperature"], -torch.inf)
    top = t.amax(1, keepdim=True)
    top = torch.where(top > -torch.inf, top, 0.0)
    e = torch.exp(t - top)
    total = e.sum(1, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    return p, torch.where(p > 0, t - top - torch.log(total), 0.0), torch.where(present, s["indices"], 0)


def _plain_loss(s):
    z = s["logits"].float() / s["temperature"]
    top = z.amax(1)
    lse = top + torch.log(torch.exp(z - top[:, None]).sum(1))
    p, log_p, at = _plain_teacher(s)
    log_q = z.gather(1, at) - lse[:, None]
    return torch.where(p > 0, p * (log_p - log_q), 0.0).sum(1) * s["temperature"] ** 2, lse


def _plain_loss_gradient(s, lse):
    p, _, at = _plain_teacher(s)
    d = torch.exp(s["logits"].float() / s["temperature"] - lse[:, None]) * p.sum(1, keepdim=True)
    d.scatter_add_(1, at, -p)
    return (d * (s["grad"] * s["temperature"])[:, None]).to(s["dtype"])


def run(state):
    s, kind = state, state["kind"]
    if own:
        e = _encoder()
        if kind == "forward":
            return e.feed_forward(s["x"], s["gate"], s["up"], s["down"], activation=s["activation"])
        if kind == "gradient":
            return e.feed_forward_gradient(s["grad"], s["x"], s["kept"], s["gate"], s["up"], s["down"],
                                           activation=s["activation"])
        if kind == "step":
            y, kept = e.feed_forward(s["x"], s["gate"], s["up"], s["down"], activation=s["activation"], keep=True)
            return (y, *e.feed_forward_gradient(s["grad"], s["x"], kept, s["gate"], s["up"], s["down"],
                                                activation=s["activation"]))
        if kind == "product8":
            return e.block_matmul(e.quantize_blocks(s["x"]), s["weight"], dtype=s["dtype"])
        if kind == "serve8":
            return e.block_feed_forward(s["x"], s["gate"], s["up"], s["down"], activation=s["activation"])
        if kind == "loss":
            return e.distillation_loss(s["logits"], s["values"], s["indices"], temperature=s["temperature"])
        if kind == "loss_gradient":
            return e.distillation_gradient(s["grad"], s["logits"], s["lse"], s["values"], s["indices"],
                                           temperature=s["temperature"])
        loss, lse = e.distillation_loss(s["logits"], s["values"], s["indices"], temperature=s["temperature"])
        return loss, lse, e.distillation_gradient(s["grad"], s["logits"], lse, s["values"], s["indices"],
                                                  temperature=s["temperature"])
    if kind == "forward":
        return _plain_forward(s)[0]
    if kind == "gradient":
        return _plain_gradient(s, s["kept"][:, 0], s["kept"][:, 1])
    if kind == "step":
        y, gate, up = _plain_forward(s)
        return (y, *_plain_gradient(s, gate, up))
    if kind == "product8":
        return (_plain_values(_plain_quantize(s["x"])) @ _plain_values(s["weight"]).t()).to(s["dtype"])
    if kind == "serve8":
        return _plain_serve8(s)
    if kind == "loss":
        return _plain_loss(s)
    if kind == "loss_gradient":
        return _plain_loss_gradient(s, s["lse"])
    loss, lse = _plain_loss(s)
    return loss, lse, _plain_loss_gradient(s, lse)


def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    rows = case["rows"]
    if kind.startswith("loss"):
        classes, top = case["classes"], case["top"]
        matrix, teacher = rows * classes * size, rows * top * (size + 8)
        forward = {"bytes": matrix + teacher + 8 * rows, "flops": 4 * rows * classes}
        backward = {"bytes": 2 * matrix + teacher + 8 * rows, "flops": 4 * rows * classes}
        if kind == "loss":
            return forward
        if kind == "loss_gradient":
            return backward
        # The logits are read for the loss and again for the gradient.
        return {key: forward[key] + backward[key] for key in forward}
    dim = case["dim"]
    if kind == "product8":
        kept = case["out"] * dim * (1 + 1 / _BLOCK)
        return {"bytes": rows * (dim + case["out"]) * size + kept, "flops": 2 * rows * dim * case["out"]}
    hidden = case["hidden"]
    weights = 3 * dim * hidden
    if kind == "serve8":
        return {"bytes": 2 * rows * dim * size + weights * (1 + 1 / _BLOCK), "flops": 2 * rows * weights}
    forward = {"bytes": (2 * rows * dim + weights) * size, "flops": 2 * rows * weights}
    # Two products a matrix; what was kept of the hidden values is read where it is given.
    backward = {"bytes": (3 * rows * dim + 2 * weights) * size, "flops": 4 * rows * weights}
    if kind == "forward":
        return forward
    if kind == "gradient":
        return {"bytes": backward["bytes"] + 8 * rows * hidden, "flops": backward["flops"]}
    return {"bytes": (4 * rows * dim + 2 * weights) * size, "flops": 6 * rows * weights}


def _exact_activation(g, activation):
    """The activation and its slope."""
    if activation == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * torch.sigmoid(-g)
    phi = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
    return g * phi, phi + g * torch.exp(-g.square() / 2.0) / math.sqrt(2.0 * math.pi)


def _exact_block(s, gate=None, up=None):
    x = s["x"].double()
    wg, wu, wd = (s[name].double() for name in ("gate", "up", "down"))
    if gate is None:
        gate, up = torch.mm(x, wg.T), torch.mm(x, wu.T)
    act, slope = _exact_activation(gate, s["activation"])
    y = torch.mm(act * up, wd.T)
    if "grad" not in s:
        return y, None
    grad = s["grad"].double()
    dh = torch.mm(grad, wd)
    dup, dgate = dh * act, dh * up * slope
    return y, (torch.mm(dgate, wg).addmm_(dup, wu), torch.mm(dgate.T, x), torch.mm(dup.T, x), torch.mm(grad.T, act * up))


def _exact_quantized(x):
    """The values that e4m3 with a power of two for each 128 stands for."""
    out = torch.empty_like(x, dtype=torch.float64)
    for begin in range(0, x.shape[1], _BLOCK):
        v = x[:, begin:begin + _BLOCK].double()
        largest = v.abs().max(1, keepdim=True).values
        scale = torch.exp2(torch.floor(torch.log2(torch.where(largest > 0, largest, 256.0))) - 8.0)
        scale = torch.where(largest > 448.0 * scale, 2.0 * scale, scale)
        scale = torch.where(largest < 224.0 * scale, 0.5 * scale, scale)
        scale = torch.where(largest > 0, scale.clamp(min=2.0 ** -127), 1.0)
        v = v / scale
        # Steps of 2^-3 of a value's power of two, from 2^-6 on.
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
        out[:, begin:begin + _BLOCK] = torch.round(v / step) * step * scale
    return out


def _exact_weight(case, seed, kind):
    """The matrices as they were before they were rounded, drawn as `prepare` does."""
    g = _generator(seed)
    rows, dim, dtype = case["rows"], case["dim"], _DTYPES[case["dtype"]]
    torch.randn(rows, dim, generator=g, device="cuda")
    torch.rand(dim, generator=g, device="cuda")
    shapes = [(case["out"], dim)] if kind == "product8" else [(case["hidden"], dim)] * 2 + [(dim, case["hidden"])]
    return [(torch.randn(*s, generator=g, device="cuda") * s[1] ** -0.5).to(dtype) for s in shapes]


def _exact_loss(s):
    t = s["temperature"]
    z = s["logits"].double() / t
    lse = torch.logsumexp(z, 1)
    loss = torch.zeros_like(lse)
    teach = torch.zeros_like(z) if "grad" in s else None
    present = (s["indices"] >= 0).all(1)
    at = s["indices"][present]
    log_p = torch.log_softmax(s["values"][present].double() / t, 1)
    loss[present] = t * t * (log_p.exp() * (log_p - z[present].gather(1, at) + lse[present, None])).sum(1)
    if teach is None:
        return loss, lse, None
    given = s["lse"].double() if "lse" in s else lse
    teach[present] = torch.exp(z[present] - given[present, None]).scatter_add(1, at, -log_p.exp())
    return loss, lse, teach * (t * s["grad"].double())[:, None]


def exact(case, seed):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind.startswith("loss"):
        loss, lse, gradient = _exact_loss(s)
        return {"loss": (loss, lse), "loss_gradient": gradient, "loss_step": (loss, lse, gradient)}[kind]
    if kind in ("product8", "serve8"):
        weights = [_exact_quantized(w) for w in _exact_weight(case, seed, kind)]
        x = _exact_quantized(s["x"])
        if kind == "product8":
            return torch.mm(x, weights[0].T)
        act, _ = _exact_activation(torch.mm(x, weights[0].T), case["activation"])
        return torch.mm(_exact_quantized(act * torch.mm(x, weights[1].T)), weights[2].T)
    if kind == "gradient":
        kept = s["kept"].double()
        return _exact_block(s, kept[:, 0], kept[:, 1])[1]
    y, gradients = _exact_block(s)
    return y if kind == "forward" else (y, *gradients)
