"""Leaf encoder: vectors from a model's leaves, and what trains them, on torch tensors.

A boosted model sorts each row into one leaf per tree; as tokens of an
embedding table those leaves feed a small network.  This module has the
operators such an encoder runs on the GPU as hand-written gfx950 kernels:

- `embedding_lookup` / `embedding_gradient`: scaled table rows for tokens, one
  by one or summed over a row's tokens, and the table's gradient by sorted
  tokens;
- `layer_norm` / `layer_norm_gradient`;
- `orthogonalize`: a matrix's update by Newton-Schulz products;

and over them `LeafTokenizer`, the torch modules `Embedding` and `LayerNorm`
and the optimizer `Muon`.

Tensors are float32, float16 or bfloat16 on a GPU.  The operators run on the
current stream of the tensors' device, wait for nothing, and keep nothing
between calls; as with torch's own, a tensor that another stream still writes
has to be waited for first.  Sums are in 32 bits and rounded once; no result
depends on the order of atomics.  Derivatives are reverse-mode and of first order;
forward-mode (dual) tensors and traces (torch.jit.trace, make_fx, torch.export)
raise NotImplementedError.  The module needs torch, which the rest of the
package does not: import torch before xgboost, so that both use one HIP runtime,
then this module by name, `from xgboost import encoder`.
"""
from __future__ import annotations

from typing import Any, Optional, Sequence, Tuple

import numpy as np
import torch

from .core import Booster, DMatrix

__all__ = ["Embedding", "LayerNorm", "LeafTokenizer", "Muon", "embedding_gradient", "embedding_lookup", "layer_norm",
           "layer_norm_gradient", "orthogonalize"]


def _one_runtime() -> None:
    # torch brings a HIP runtime of its own.  Loaded first, it is the one
    # libxgboost.so takes too; loaded second, the process would hold two, of which
    # neither knows the other's streams.
    with open("/proc/self/maps", encoding="utf-8") as maps:
        runtimes = {line.split(maxsplit=5)[-1].strip() for line in maps if "/libamdhip64.so" in line}
    if len(runtimes) > 1:
        raise ImportError("xgboost was imported before torch, which loaded a second HIP runtime: import torch first "
                          f"(loaded: {', '.join(sorted(runtimes))})")


_one_runtime()
try:
    from . import _encoder
except ImportError as missing:
    raise ImportError("xgboost._encoder was not found; build it with "
                      "`python -c 'import __graft_entry__ as g; g.build()'`") from missing


class _NoDerivative(torch.autograd.Function):
    """An operator's results where an argument requires a gradient: one that would
    have to pass them is an error, not a graph that ends there unseen."""

    @staticmethod
    def forward(ctx, name, operator, *arguments):  # pylint: disable=arguments-differ
        ctx.name = name
        return operator(*arguments)

    @staticmethod
    def backward(ctx, *_):  # pylint: disable=arguments-differ
        raise NotImplementedError(f"{ctx.name} has no derivative")


def _without_derivative(name: str, operator: Any, *arguments: Any) -> Any:
    if torch.is_grad_enabled() and any(getattr(a, "requires_grad", False) for a in arguments):
        return _NoDerivative.apply(name, operator, *arguments)
    return operator(*arguments)


# ---- embedding ---------------------------------------------------------------

def embedding_gradient(grad: torch.Tensor, tokens: torch.Tensor, num_embeddings: int, *, scale: float = 1.0,
                       pool: bool = False) -> torch.Tensor:
    """The table's gradient, (num_embeddings, dim) in grad's type, from the
    gradient of `embedding_lookup`'s result: each table row's sum over the
    tokens that name it.  Fewer than 2^31 tokens.  Has no derivative itself: where
    grad requires one, a backward pass through the result is an error."""
    return _without_derivative("embedding_gradient", _encoder.lookup_gradient, grad, tokens, num_embeddings, scale, pool)


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale, pool):  # pylint: disable=arguments-differ
        ctx.save_for_backward(tokens)
        ctx.table, ctx.scale, ctx.pool = weight.shape[0], scale, pool
        return _encoder.lookup(weight, tokens, scale, pool)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):  # pylint: disable=arguments-differ
        tokens, = ctx.saved_tensors
        return embedding_gradient(grad, tokens, ctx.table, scale=ctx.scale, pool=ctx.pool), None, None, None


def embedding_lookup(weight: torch.Tensor, tokens: torch.Tensor, *, scale: float = 1.0,
                     pool: bool = False) -> torch.Tensor:
    """scale * weight[tokens]: one row of the table (num_embeddings, dim) per
    token (int32 or int64, any shape).  With `pool` the tokens' last axis is
    summed, one vector per row of tokens.  A token outside the table, -1 for
    padding, names no row and adds nothing.  Differentiable in weight."""
    if torch.is_grad_enabled() and getattr(weight, "requires_grad", False):
        return _EmbeddingLookup.apply(weight, tokens, scale, pool)
    return _encoder.lookup(weight, tokens, scale, pool)


# ---- layer norm --------------------------------------------------------------

def layer_norm_gradient(grad: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None
                        ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """The gradients of `layer_norm`'s x, weight and bias from its result's
    gradient and the statistics it returned; without a weight the last two are
    None.  Has no derivative itself, like `embedding_gradient`."""
    return _without_derivative("layer_norm_gradient", _encoder.norm_gradient, grad, x, mean, rstd, weight)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):  # pylint: disable=arguments-differ
        y, mean, rstd = _encoder.norm(x, weight, bias, eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.has_bias = bias is not None
        ctx.mark_non_differentiable(mean, rstd)
        ctx.set_materialize_grads(False)
        return y, mean, rstd

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, *_):  # pylint: disable=arguments-differ
        if grad is None:
            return None, None, None, None
        x, mean, rstd, weight = ctx.saved_tensors
        dx, dweight, dbias = layer_norm_gradient(grad, x, mean, rstd, weight)
        return dx, dweight, dbias if ctx.has_bias else None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): x's last axis normalised to mean 0 and variance 1, times
    weight plus bias, and the statistics (float32) that `layer_norm_gradient`
    reads.  y comes of the mean in more than 32 bits, the gradient of the one
    returned.  weight and bias are float32 or x's type; a bias needs a weight.
    Differentiable in x, weight and bias through y."""
    if torch.is_grad_enabled() and (getattr(x, "requires_grad", False) or getattr(weight, "requires_grad", False) or
                                    getattr(bias, "requires_grad", False)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _encoder.norm(x, weight, bias, eps)


# ---- orthogonalised updates ----------------------------------------------------

def orthogonalize(update: torch.Tensor, *, steps: int = 5,
                  coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315), eps: float = 1e-7) -> torch.Tensor:
    """The update with its singular values driven towards 1 (the Muon
    optimiser's): X = update / (norm + eps), then `steps` times
    X = (a I + b A + c A^2) X with A = X X^T, on the shorter side.  Leading axes
    are a batch of matrices.  Coefficients that could take a singular value of at
    most 1 beyond about 4 before the last step are refused.  Whatever the type, a
    value of X is kept to 22 bits, or to 2^-37 if it is below 2^-14 (X has norm 1
    at first), and the result is rounded to its type once.  Has no derivative:
    where the update requires one, a backward pass through the result is an error."""
    return _without_derivative("orthogonalize", _encoder.orthogonalize, update, steps, coefficients, eps)


class Muon(torch.optim.Optimizer):
    """Matrices by orthogonalised momentum: m = momentum m + grad, and
    w -= lr (sqrt(max(1, rows / columns)) orthogonalize(grad + momentum m) + weight_decay w)
    (without `nesterov` orthogonalize(m)).  For weights of two axes; biases,
    norms and embedding tables belong to another optimizer.

    The step is computed in float32.  Of a float16 or bfloat16 weight the state
    keeps the float32 value too (`weight`, beside `momentum`), of which the
    parameter is the rounding: steps and decays below half a unit of its type add
    up.  A parameter set from outside goes on from what it was set to."""

    def __init__(self, params: Any, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5,
                 coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315)) -> None:
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, coefficients=tuple(coefficients)))

    def add_param_group(self, param_group: Any) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2:
                self.param_groups.pop()
                raise ValueError(f"Muon takes matrices, got a parameter of shape {tuple(p.shape)}")

    def load_state_dict(self, state_dict: Any) -> None:
        super().load_state_dict(state_dict)
        # That rounds the state to the parameters' types.
        saved = [k for group in state_dict["param_groups"] for k in group["params"]]
        for k, p in zip(saved, (p for group in self.param_groups for p in group["params"])):
            for name, value in state_dict["state"].get(k, {}).items():
                self.state[p][name] = value.to(device=p.device, dtype=self._state_type(p), copy=True)

    @staticmethod
    def _state_type(p: torch.Tensor) -> torch.dtype:
        return torch.float32 if p.dtype in (torch.float16, torch.bfloat16) else p.dtype

    @torch.no_grad()
    def step(self, closure: Any = None) -> Any:  # pylint: disable=arguments-differ
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                short = p.dtype != self._state_type(p)
                weight, grad = p, p.grad
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(p, dtype=self._state_type(p))
                if short:
                    grad = grad.float()
                    if "weight" not in state:
                        state["weight"] = p.float()
                    weight = state["weight"]  # written in place: a captured step's replays go on from it
                    torch.where(weight.to(p.dtype) == p, weight, p.float(), out=weight)
                m = state["momentum"].mul_(group["momentum"]).add_(grad)
                update = torch.add(grad, m, alpha=group["momentum"]) if group["nesterov"] else m
                update = orthogonalize(update, steps=group["steps"], coefficients=group["coefficients"])
                if group["weight_decay"]:
                    weight.mul_(1.0 - group["lr"] * group["weight_decay"])
                weight.add_(update, alpha=-group["lr"] * max(1.0, p.shape[0] / p.shape[1]) ** 0.5)
                if short:
                    p.copy_(weight)
        return loss


# ---- modules -------------------------------------------------------------------

class Embedding(torch.nn.Module):
    """`embedding_lookup` with a table of its own, drawn from a normal
    distribution of variance 1 / dim."""

    def __init__(self, num_embeddings: int, dim: int, *, scale: float = 1.0, pool: bool = False,
                 device: Any = "cuda", dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        self.scale, self.pool = scale, pool
        self.weight = torch.nn.Parameter(torch.randn(num_embeddings, dim, device=device, dtype=dtype) * dim ** -0.5)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return embedding_lookup(self.weight, tokens, scale=self.scale, pool=self.pool)


class LayerNorm(torch.nn.Module):
    """`layer_norm` with a weight of ones and a bias of zeros."""

    def __init__(self, dim: int, *, eps: float = 1e-5, device: Any = "cuda",
                 dtype: torch.dtype = torch.float32) -> None:
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(dim, device=device, dtype=dtype))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, eps=self.eps)[0]


class LeafTokenizer:
    """A model's leaves as tokens: every leaf of every tree of `iteration_range`
    has a number of its own below `vocabulary`, tree by tree in the order of the
    node ids.  Calling it with a DMatrix gives int32 tokens (rows, trees) on the
    GPU."""

    def __init__(self, booster: Booster, iteration_range: Tuple[int, int] = (0, 0), device: Any = "cuda") -> None:
        if not isinstance(booster, Booster):
            raise TypeError("`booster` must be an xgboost.Booster")
        begin, end = (int(v) for v in iteration_range)
        if begin != 0:
            raise ValueError("leaves are of the rounds [0, end)")
        trees = booster.trees_to_json()
        trees = trees[:end] if end > 0 else trees
        if not trees:
            raise ValueError("the model has no trees")
        nodes = max(len(t["left_children"]) for t in trees)
        table = np.full((len(trees), nodes), -1, np.int32)
        self.vocabulary = 0
        for row, tree in zip(table, trees):
            leaves = np.flatnonzero(np.asarray(tree["left_children"]) == -1)
            row[leaves] = np.arange(self.vocabulary, self.vocabulary + len(leaves), dtype=np.int32)
            self.vocabulary += len(leaves)
        self._booster, self._rounds = booster, (0, len(trees))
        self.trees = len(trees)
        self._table = torch.from_numpy(table).to(device)

    def __call__(self, data: DMatrix) -> torch.Tensor:
        leaves = self._booster.predict(data, pred_leaf=True, iteration_range=self._rounds)
        leaves = torch.from_numpy(leaves.reshape(-1, self.trees)).to(self._table.device).long()
        return self._table.gather(1, leaves.t()).t().contiguous()
