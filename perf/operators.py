"""Performance cases of the leaf encoder's operators: what turns the leaves of
a boosted model into vectors and trains the matrices behind them.

Each case is a dict of plain values; `kind` names the call:

- lookup: rows of an embedding table for tokens, scaled; with `trees` the sum
  of a row's tokens, one token per tree (`Booster.predict(pred_leaf=True)`);
- lookup_gradient: the table's gradient from the vectors' gradient;
- norm: layer norm over the last axis, with the statistics its gradient reads;
- norm_gradient: the gradients of layer norm's input, weight and bias;
- norm_step: both, as in a training step;
- orthogonalize: a matrix's update by Newton-Schulz products.

With `own` false the operators run in their plain form, elementary torch
operations in 32 bits; with `own` true as `xgboost.encoder` has them.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-5
_STEPS = 5
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_NORM_EPS = 1e-7
_package = None


def _encoder():
    global _package
    if _package is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "xgboost-metal_amd", "python"))
        from xgboost import encoder
        _package = encoder
    return _package


def _leaves(name, kind, rows, trees, leaves, dim, dtype):
    return {"name": name, "kind": kind, "rows": rows, "trees": trees, "vocabulary": trees * leaves, "dim": dim,
            "dtype": dtype}


def _tokens(name, kind, rows, vocabulary, dim, dtype, padding):
    return {"name": name, "kind": kind, "rows": rows, "trees": 0, "vocabulary": vocabulary, "dim": dim,
            "dtype": dtype, "padding": padding}


def _matrix(name, kind, rows, dim, dtype):
    return {"name": name, "kind": kind, "rows": rows, "dim": dim, "dtype": dtype}


def listed():
    return [
        # One request of a service: 16 rows through 100 trees of depth 6.
        _leaves("lookup_request_16x100", "lookup", 16, 100, 64, 32, "f32"),
        # Encoding a whole table: 262,144 rows through 100 trees of depth 8.
        _leaves("lookup_table_262k_x100", "lookup", 262144, 100, 256, 64, "bf16"),
        # Tokens one by one, wide vectors, padded sequences, an odd count.
        _tokens("lookup_tokens_8191_x1024", "lookup", 8191, 32768, 1024, "bf16", 0.05),
        # A mini-batch's gradient: launches count.
        _leaves("lookup_gradient_256x100", "lookup_gradient", 256, 100, 64, 32, "f32"),
        # A large batch through 100 trees of depth 8: many tokens a table row.
        _leaves("lookup_gradient_65k_x100", "lookup_gradient", 65536, 100, 256, 64, "bf16"),
        # Sequences of tokens with a few frequent ones, most table rows untouched.
        _tokens("lookup_gradient_tokens_16411_x1024", "lookup_gradient", 16411, 32768, 1024, "f16", 0.05),
        # The encoder's norm on one request.
        _matrix("norm_request_16x32", "norm", 16, 32, "f32"),
        # Backward pass at odd sizes.
        _matrix("norm_gradient_5003x1000", "norm_gradient", 5003, 1000, "f32"),
        # Forward and backward of a training step on a large batch.
        _matrix("norm_step_65k_x1024", "norm_step", 65536, 1024, "bf16"),
        # The update of a small encoder's projection.
        _matrix("orthogonalize_64x256", "orthogonalize", 64, 256, "f32"),
        # Odd sizes, taller than wide.
        _matrix("orthogonalize_1500x1001", "orthogonalize", 1500, 1001, "f32"),
        # A wide layer's update.
        _matrix("orthogonalize_2048x4096", "orthogonalize", 2048, 4096, "bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _dim(rng, high):
    # Mostly whole vectors of 8 values, sometimes any width.
    d = _log_int(rng, 8, high)
    return d if rng.random() < 0.3 else max(8, d // 8 * 8)


def draw(rng):
    kind = rng.choice(["lookup", "lookup", "lookup_gradient", "lookup_gradient", "norm", "norm_gradient", "norm_step",
                       "orthogonalize", "orthogonalize"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind.startswith("lookup"):
        if rng.random() < 0.5:
            # Tokens times width stay below the listed tables'.
            most = 262144 * 100 * 64 if kind == "lookup" else 65536 * 100 * 64
            if dtype == "f32":
                most //= 2
            trees, dim = rng.randint(10, 300), _dim(rng, 128)
            rows = _log_int(rng, 1, max(2, min(262144, most // (trees * dim))))
            case = {"kind": kind, "rows": rows, "trees": trees, "vocabulary": trees * rng.choice([16, 64, 200, 256]),
                    "dim": dim}
        else:
            case = {"kind": kind, "rows": _log_int(rng, 1, 16384), "trees": 0, "vocabulary": _log_int(rng, 100, 32768),
                    "dim": _dim(rng, 1024), "padding": rng.choice([0.0, 0.05, 0.5])}
    elif kind == "orthogonalize":
        case = {"kind": kind, "rows": _log_int(rng, 16, 2048), "dim": _log_int(rng, 16, 2048)}
    else:
        dim = _log_int(rng, 8, 8192)
        case = {"kind": kind, "rows": _log_int(rng, 1, 65536 * 512 // dim), "dim": dim}
    case["dtype"] = dtype
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _draw_tokens(case, g):
    rows, trees, vocabulary = case["rows"], case["trees"], case["vocabulary"]
    if trees:
        # Leaves hold unequal shares of the rows; tree t's tokens follow tree
        # t - 1's.
        leaves = vocabulary // trees
        u = torch.rand(rows, trees, generator=g, device="cuda")
        leaf = (u * u * leaves).to(torch.int32).clamp_(max=leaves - 1)
        return leaf + torch.arange(trees, dtype=torch.int32, device="cuda") * leaves
    u = torch.rand(rows, generator=g, device="cuda")
    rank = (u.pow(4) * vocabulary).long().clamp_(max=vocabulary - 1)
    tokens = torch.randperm(vocabulary, generator=g, device="cuda")[rank]
    return torch.where(torch.rand(rows, generator=g, device="cuda") < case["padding"], -torch.ones_like(tokens), tokens)


def prepare(case, seed):
    g = _generator(seed)
    kind, dtype = case["kind"], _DTYPES[case["dtype"]]
    rows, dim = case["rows"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = {"kind": kind}
    if kind.startswith("lookup"):
        state["pool"] = case["trees"] > 0
        state["scale"] = 1.0 / case["trees"] if case["trees"] else math.sqrt(dim)
        state["tokens"] = _draw_tokens(case, g)
        state["vocabulary"] = case["vocabulary"]
        if kind == "lookup":
            state["weight"] = normal(case["vocabulary"], dim).mul_(dim ** -0.5).to(dtype)
        else:
            state["grad"] = normal(rows, dim).to(dtype)
    elif kind == "orthogonalize":
        # Momentum of a few directions above noise.
        rank = max(1, min(rows, dim) // 8)
        update = normal(rows, rank) @ normal(rank, dim) / math.sqrt(rank) + 0.3 * normal(rows, dim)
        state["update"] = (update * 1e-2).to(dtype)
    else:
        # Some columns far from the others, rows off zero.
        x = normal(rows, dim) * (1.0 + 4.0 * (torch.rand(dim, generator=g, device="cuda") < 0.02)) + 0.5 * normal(rows, 1)
        state["x"] = x.to(dtype)
        state["weight"] = (1.0 + 0.1 * normal(dim)).to(dtype)
        state["bias"] = (0.1 * normal(dim)).to(dtype)
        if kind != "norm":
            state["grad"] = normal(rows, dim).to(dtype)
        if kind == "norm_gradient":
            x = state["x"].double()
            mean = x.mean(1)
            state["mean"] = mean.float()
            state["rstd"] = (((x - mean[:, None]) ** 2).mean(1) + _EPS).rsqrt().float()
    return state


def _plain_lookup(weight, tokens, scale, pool):
    present = (tokens >= 0) & (tokens < weight.shape[0])
    rows = weight[torch.where(present, tokens, 0).long()].float()
    rows = torch.where(present[..., None], rows, 0.0)
    if pool:
        rows = rows.sum(-2)
    return (rows * scale).to(weight.dtype)


def _plain_lookup_gradient(grad, tokens, vocabulary, scale, pool):
    present = (tokens >= 0) & (tokens < vocabulary)
    at = torch.where(present, tokens, vocabulary).long().reshape(-1)
    dim = grad.shape[-1]
    each = grad.float()
    if pool:
        each = each[:, None, :].expand(tokens.shape[0], tokens.shape[1], dim).reshape(-1, dim)
    total = torch.zeros(vocabulary + 1, dim, device=grad.device)
    total.index_add_(0, at, each)
    return (total[:vocabulary] * scale).to(grad.dtype)


def _plain_norm(x, weight, bias):
    v = x.float()
    mean = v.mean(-1)
    centred = v - mean[..., None]
    rstd = ((centred * centred).mean(-1) + _EPS).rsqrt()
    y = centred * rstd[..., None] * weight.float() + bias.float()
    return y.to(x.dtype), mean, rstd


def _plain_norm_gradient(grad, x, mean, rstd, weight):
    d = grad.float()
    hat = (x.float() - mean[..., None]) * rstd[..., None]
    dw, db = (d * hat).sum(0), d.sum(0)
    d = d * weight.float()
    dx = (d - d.mean(-1, keepdim=True) - hat * (d * hat).mean(-1, keepdim=True)) * rstd[..., None]
    return dx.to(x.dtype), dw.to(weight.dtype), db.to(weight.dtype)


def _plain_orthogonalize(update):
    a, b, c = _COEFFICIENTS
    x = update.float()
    x = x / ((x * x).sum().sqrt() + _NORM_EPS)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t()
    for _ in range(_STEPS):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.t() if tall else x).to(update.dtype)


def run(state):
    kind = state["kind"]
    if own:
        e = _encoder()
        if kind == "lookup":
            return e.embedding_lookup(state["weight"], state["tokens"], scale=state["scale"], pool=state["pool"])
        if kind == "lookup_gradient":
            return e.embedding_gradient(state["grad"], state["tokens"], state["vocabulary"], scale=state["scale"],
                                        pool=state["pool"])
        if kind == "norm":
            return e.layer_norm(state["x"], state["weight"], state["bias"], eps=_EPS)
        if kind == "norm_gradient":
            return e.layer_norm_gradient(state["grad"], state["x"], state["mean"], state["rstd"], state["weight"])
        if kind == "norm_step":
            y, mean, rstd = e.layer_norm(state["x"], state["weight"], state["bias"], eps=_EPS)
            return (y, *e.layer_norm_gradient(state["grad"], state["x"], mean, rstd, state["weight"]))
        return e.orthogonalize(state["update"], steps=_STEPS, coefficients=_COEFFICIENTS, eps=_NORM_EPS)
    if kind == "lookup":
        return _plain_lookup(state["weight"], state["tokens"], state["scale"], state["pool"])
    if kind == "lookup_gradient":
        return _plain_lookup_gradient(state["grad"], state["tokens"], state["vocabulary"], state["scale"], state["pool"])
    if kind == "norm":
        return _plain_norm(state["x"], state["weight"], state["bias"])
    if kind == "norm_gradient":
        return _plain_norm_gradient(state["grad"], state["x"], state["mean"], state["rstd"], state["weight"])
    if kind == "norm_step":
        y, mean, rstd = _plain_norm(state["x"], state["weight"], state["bias"])
        return (y, *_plain_norm_gradient(state["grad"], state["x"], mean, rstd, state["weight"]))
    return _plain_orthogonalize(state["update"])


def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    rows, dim = case["rows"], case["dim"]
    if kind.startswith("lookup"):
        trees, vocabulary = case["trees"], case["vocabulary"]
        count = rows * max(1, trees)
        ids = count * (4 if trees else 8)
        if kind == "lookup":
            # The table's rows that tokens name, at most one read each.
            return {"bytes": ids + (min(vocabulary, count) + rows) * dim * size, "flops": (count + rows) * dim}
        return {"bytes": ids + (rows + vocabulary) * dim * size, "flops": (count + vocabulary) * dim}
    if kind == "orthogonalize":
        # Each step is a polynomial in X X^T, symmetric: X X^T once, the steps'
        # products among m x m matrices, one product with X (multiplications
        # and additions, half of them where the result is symmetric).
        m, n = min(rows, dim), max(rows, dim)
        return {"bytes": 2 * m * n * size, "flops": 2 * m * m * (1.5 * n + (2 * _STEPS - 1.5) * m)}
    matrix = rows * dim * size
    forward = {"bytes": 2 * matrix + 2 * dim * size + 8 * rows, "flops": 8 * rows * dim}
    if kind == "norm":
        return forward
    backward = {"bytes": 3 * matrix + 3 * dim * size + 8 * rows, "flops": 14 * rows * dim}
    if kind == "norm_gradient":
        return backward
    # x is read for the forward pass and again for the backward.
    return {key: forward[key] + backward[key] for key in forward}


def _exact_lookup(weight, tokens, scale, pool):
    tokens = tokens if pool else tokens[:, None]
    table = torch.cat([weight.double() * scale, torch.zeros(1, weight.shape[1], dtype=torch.float64, device="cuda")])
    total = torch.zeros(tokens.shape[0], weight.shape[1], dtype=torch.float64, device="cuda")
    for column in tokens.long().unbind(1):
        total += table[torch.where((column < 0) | (column >= len(weight)), len(weight), column)]
    return total


def _exact_lookup_gradient(grad, tokens, vocabulary, scale, pool):
    tokens = tokens if pool else tokens[:, None]
    grad = grad.double() * scale
    total = torch.zeros(vocabulary, grad.shape[1], dtype=torch.float64, device="cuda")
    for column in tokens.long().unbind(1):
        keep = ((column >= 0) & (column < vocabulary)).nonzero()[:, 0]
        order = column[keep].argsort(stable=True)
        found, counts = column[keep][order].unique_consecutive(return_counts=True)
        # Sums of runs as differences of a running sum in 64 bits.
        running = torch.cat([torch.zeros(1, grad.shape[1], dtype=torch.float64, device="cuda"),
                             grad[keep[order]].cumsum(0)])
        ends = counts.cumsum(0)
        total[found] += running[ends] - running[ends - counts]
    return total


def _exact_norm(x, weight, bias):
    x = x.double()
    variance, mean = torch.var_mean(x, -1, correction=0)
    rstd = 1.0 / (variance + _EPS).sqrt()
    return (x - mean[:, None]) * (rstd[:, None] * weight.double()) + bias.double(), mean, rstd


def _exact_norm_gradient(grad, x, mean, rstd, weight):
    grad, rstd = grad.double(), rstd.double()[:, None]
    hat = (x.double() - mean.double()[:, None]) * rstd
    through = grad * weight.double()
    dim = x.shape[1]
    dx = rstd / dim * (dim * through - through.sum(1, keepdim=True) - hat * (through * hat).sum(1, keepdim=True))
    return dx, torch.einsum("rd,rd->d", grad, hat), torch.einsum("rd->d", grad)


def _exact_orthogonalize(update):
    a, b, c = _COEFFICIENTS
    y = update.double()
    y = y / (torch.linalg.vector_norm(y) + _NORM_EPS)
    if y.shape[0] < y.shape[1]:
        y = y.t()
    for _ in range(_STEPS):
        gram = y.t() @ y
        z = gram @ gram * c + gram * b
        z.diagonal().add_(a)
        y = y @ z
    return y.t() if update.shape[0] < update.shape[1] else y


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "lookup":
        return _exact_lookup(s["weight"], s["tokens"], s["scale"], s["pool"])
    if kind == "lookup_gradient":
        return _exact_lookup_gradient(s["grad"], s["tokens"], s["vocabulary"], s["scale"], s["pool"])
    if kind == "norm":
        return _exact_norm(s["x"], s["weight"], s["bias"])
    if kind == "norm_gradient":
        return _exact_norm_gradient(s["grad"], s["x"], s["mean"], s["rstd"], s["weight"])
    if kind == "norm_step":
        y, mean, rstd = _exact_norm(s["x"], s["weight"], s["bias"])
        return (y, *_exact_norm_gradient(s["grad"], s["x"], mean, rstd, s["weight"]))
    return _exact_orthogonalize(s["update"])
