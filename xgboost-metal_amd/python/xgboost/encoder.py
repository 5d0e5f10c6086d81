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
depends on the order of atomics.  The module needs torch, which the rest of the
package does not: import torch before xgboost, so that both use one HIP runtime,
then this module by name, `from xgboost import encoder`.
"""
from __future__ import annotations

import ctypes
from typing import Any, Optional, Sequence, Tuple

import numpy as np
import torch

from .core import _LIB as _CORE
from .core import Booster, DMatrix, XGBoostError

__all__ = ["Embedding", "LayerNorm", "LeafTokenizer", "Muon", "embedding_gradient", "embedding_lookup", "layer_norm",
           "layer_norm_gradient", "orthogonalize"]


def _bind_lib():
    # torch brings a HIP runtime of its own.  Loaded first, it is the one the
    # library takes too; loaded second, the process would hold two, of which
    # only one can have the GPU's queues and neither knows the other's streams.
    with open("/proc/self/maps", encoding="utf-8") as maps:
        runtimes = {line.split(maxsplit=5)[-1].strip() for line in maps if "/libamdhip64.so" in line}
    if len(runtimes) > 1:
        raise ImportError("xgboost was imported before torch, which loaded a second HIP runtime: import torch first "
                          f"(loaded: {', '.join(sorted(runtimes))})")
    lib = _CORE
    pointer, size, integer, real = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
    lib.mgb_last_error.restype = ctypes.c_char_p
    lib.mgb_embedding_lookup.argtypes = [pointer] * 3 + [size] * 5 + [real, integer, integer, pointer]
    lib.mgb_embedding_gradient_workspace_bytes.argtypes = [size] * 3 + [integer]
    lib.mgb_embedding_gradient_workspace_bytes.restype = ctypes.c_size_t
    lib.mgb_embedding_gradient.argtypes = ([pointer] * 3 + [size] * 5 + [real, integer, integer, pointer,
                                                                         ctypes.c_size_t, pointer])
    lib.mgb_layer_norm.argtypes = [pointer] * 6 + [size] * 3 + [real, integer, integer, pointer]
    lib.mgb_layer_norm_gradient_workspace_bytes.argtypes = [size, size, integer]
    lib.mgb_layer_norm_gradient_workspace_bytes.restype = ctypes.c_size_t
    lib.mgb_layer_norm_gradient.argtypes = ([pointer] * 8 + [size] * 4 + [integer, integer, pointer, ctypes.c_size_t,
                                                                          pointer])
    lib.mgb_orthogonalize_workspace_bytes.argtypes = [size] * 3
    lib.mgb_orthogonalize_workspace_bytes.restype = ctypes.c_size_t
    lib.mgb_orthogonalize.argtypes = ([pointer] * 2 + [size] * 5 + [integer, pointer, real, integer, pointer,
                                                                    ctypes.c_size_t, pointer])
    return lib


_LIB = _bind_lib()
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TOKEN_BYTES = {torch.int32: 4, torch.int64: 8}


def _check_call(ret: int) -> None:
    if ret != 0:
        raise XGBoostError(_LIB.mgb_last_error().decode())


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class _on:
    """Makes a tensor's device the current one for a call, where it is not."""

    __slots__ = ("_index", "_before")

    def __init__(self, device: torch.device) -> None:
        self._index = device.index

    def __enter__(self) -> None:
        self._before = torch.cuda.current_device()
        if self._before != self._index:
            torch.cuda.set_device(self._index)

    def __exit__(self, *exc: Any) -> None:
        if self._before != self._index:
            torch.cuda.set_device(self._before)


def _dtype(name: str, t: torch.Tensor) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU, is on {t.device}")
    return code


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """t, or a copy of it, as rows of its last axis at one distance, and that distance."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] == 1):
        return t, t.stride(0)
    return t.contiguous(), t.shape[-1]


def _same_device(t: torch.Tensor, **others: Optional[torch.Tensor]) -> None:
    for name, other in others.items():
        if other is not None and other.device != t.device:
            raise ValueError(f"{name} must be on {t.device}, is on {other.device}")


# ---- embedding ---------------------------------------------------------------

def _tokens(tokens: torch.Tensor, pool: bool) -> Tuple[torch.Tensor, int]:
    if not isinstance(tokens, torch.Tensor):
        raise TypeError(f"tokens must be a torch.Tensor, got {type(tokens).__name__}")
    size = _TOKEN_BYTES.get(tokens.dtype)
    if size is None:
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    if pool and tokens.dim() == 0:
        raise ValueError("pool needs tokens with an axis to sum over")
    return tokens.contiguous(), size


def _lookup(weight: torch.Tensor, tokens: torch.Tensor, scale: float, pool: bool) -> torch.Tensor:
    dtype = _dtype("weight", weight)
    if weight.dim() != 2:
        raise ValueError(f"weight must be a table of rows, has shape {tuple(weight.shape)}")
    tokens, size = _tokens(tokens, pool)
    _same_device(weight, tokens=tokens)
    weight, stride = _rows(weight)
    vocabulary, dim = weight.shape
    shape = tokens.shape[:-1] if pool else tokens.shape
    bag = tokens.shape[-1] if pool else 1
    out = torch.empty((*shape, dim), dtype=weight.dtype, device=weight.device)
    with _on(weight.device):
        _check_call(_LIB.mgb_embedding_lookup(out.data_ptr(), weight.data_ptr(), tokens.data_ptr(),
                                              shape.numel(), bag, vocabulary, dim, stride, scale, dtype, size,
                                              _stream(weight.device)))
    return out


def embedding_gradient(grad: torch.Tensor, tokens: torch.Tensor, num_embeddings: int, *, scale: float = 1.0,
                       pool: bool = False) -> torch.Tensor:
    """The table's gradient, (num_embeddings, dim) in grad's type, from the
    gradient of `embedding_lookup`'s result: each table row's sum over the
    tokens that name it.  Fewer than 2^31 tokens."""
    dtype = _dtype("grad", grad)
    tokens, size = _tokens(tokens, pool)
    _same_device(grad, tokens=tokens)
    shape = tokens.shape[:-1] if pool else tokens.shape
    if grad.dim() < 1 or grad.shape[:-1] != shape:
        raise ValueError(f"grad must have shape {(*shape, 'dim')} for these tokens, has {tuple(grad.shape)}")
    if num_embeddings < 1:
        raise ValueError(f"num_embeddings must be at least 1, is {num_embeddings}")
    dim = grad.shape[-1]
    grad, stride = _rows(grad)
    bag = tokens.shape[-1] if pool else 1
    out = torch.empty((num_embeddings, dim), dtype=grad.dtype, device=grad.device)
    need = _LIB.mgb_embedding_gradient_workspace_bytes(tokens.numel(), num_embeddings, dim, dtype)
    workspace = torch.empty(need, dtype=torch.uint8, device=grad.device)
    with _on(grad.device):
        _check_call(_LIB.mgb_embedding_gradient(out.data_ptr(), grad.data_ptr(), tokens.data_ptr(), shape.numel(), bag,
                                                num_embeddings, dim, stride, scale, dtype, size,
                                                workspace.data_ptr(), need, _stream(grad.device)))
    return out


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tokens, scale, pool):  # pylint: disable=arguments-differ
        ctx.save_for_backward(tokens)
        ctx.table, ctx.scale, ctx.pool = weight.shape[0], scale, pool
        return _lookup(weight, tokens, scale, pool)

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
    if isinstance(weight, torch.Tensor) and weight.requires_grad and torch.is_grad_enabled():
        return _EmbeddingLookup.apply(weight, tokens, scale, pool)
    return _lookup(weight, tokens, scale, pool)


# ---- layer norm --------------------------------------------------------------

def _norm_weight(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor]) -> int:
    if weight is None:
        if bias is not None:
            raise ValueError("a bias needs a weight")
        return 0
    dtype = _dtype("weight", weight)
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"weight must be {x.dtype} or float32, is {weight.dtype}")
    if bias is not None and bias.dtype != weight.dtype:
        raise TypeError(f"bias must be {weight.dtype} as the weight, is {bias.dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != x.shape[-1:]:
            raise ValueError(f"{name} must have shape {tuple(x.shape[-1:])}, has {tuple(t.shape)}")
    _same_device(x, weight=weight, bias=bias)
    return dtype


def _norm(x, weight, bias, eps):
    dtype = _dtype("x", x)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last axis to normalise, has shape {tuple(x.shape)}")
    weight_dtype = _norm_weight(x, weight, bias) if weight is not None or bias is not None else dtype
    x, stride = _rows(x)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    shape = x.shape[:-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = torch.empty(shape, dtype=torch.float32, device=x.device)
    rstd = torch.empty(shape, dtype=torch.float32, device=x.device)
    with _on(x.device):
        _check_call(_LIB.mgb_layer_norm(y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), x.data_ptr(),
                                        None if weight is None else weight.data_ptr(),
                                        None if bias is None else bias.data_ptr(), shape.numel(), x.shape[-1], stride,
                                        eps, dtype, weight_dtype, _stream(x.device)))
    return y, mean, rstd


def layer_norm_gradient(grad: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: Optional[torch.Tensor] = None
                        ) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """The gradients of `layer_norm`'s x, weight and bias from its result's
    gradient and the statistics it returned; without a weight the last two are
    None."""
    dtype = _dtype("x", x)
    if _dtype("grad", grad) != dtype or grad.shape != x.shape:
        raise ValueError(f"grad must be like x, {x.dtype} {tuple(x.shape)}, is {grad.dtype} {tuple(grad.shape)}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last axis to normalise, has shape {tuple(x.shape)}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype != torch.float32 or t.shape != x.shape[:-1]:
            raise ValueError(f"{name} must be float32 {tuple(x.shape[:-1])}, is {t.dtype} {tuple(t.shape)}")
    _same_device(x, grad=grad, mean=mean, rstd=rstd)
    weight_dtype = _norm_weight(x, weight, None) if weight is not None else dtype
    x, stride = _rows(x)
    grad, grad_stride = _rows(grad)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    rows, dim = x.shape[:-1].numel(), x.shape[-1]
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dweight = dbias = workspace = None
    need = 0
    if weight is not None:
        weight = weight.contiguous()
        dweight = torch.empty_like(weight)
        dbias = torch.empty_like(weight)
        need = _LIB.mgb_layer_norm_gradient_workspace_bytes(rows, dim, dtype)
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    with _on(x.device):
        _check_call(_LIB.mgb_layer_norm_gradient(
            dx.data_ptr(), None if weight is None else dweight.data_ptr(), None if weight is None else dbias.data_ptr(),
            grad.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
            None if weight is None else weight.data_ptr(), rows, dim, grad_stride, stride, dtype, weight_dtype,
            None if weight is None else workspace.data_ptr(), need, _stream(x.device)))
    return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):  # pylint: disable=arguments-differ
        y, mean, rstd = _norm(x, weight, bias, eps)
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
    reads.  weight and bias are float32 or x's type; a bias needs a weight.
    Differentiable in x, weight and bias through y."""
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm(x, weight, bias, eps)


# ---- orthogonalised updates ----------------------------------------------------

def orthogonalize(update: torch.Tensor, *, steps: int = 5,
                  coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315), eps: float = 1e-7) -> torch.Tensor:
    """The update with its singular values driven towards 1 (the Muon
    optimiser's): X = update / (norm + eps), then `steps` times
    X = (a I + b A + c A^2) X with A = X X^T, on the shorter side.  Leading axes
    are a batch of matrices.  Works with 22 bits of each value whatever the
    type; the result is rounded to it once."""
    dtype = _dtype("update", update)
    if update.dim() < 2:
        raise ValueError(f"update must be a matrix, has shape {tuple(update.shape)}")
    if len(coefficients) != 3:
        raise ValueError("coefficients must be three numbers")
    update = update.detach()
    rows, columns = update.shape[-2:]
    batch = update.shape[:-2].numel()
    if update.dim() == 2 and (update.stride(1) == 1 or columns == 1):
        stride, batch_stride = update.stride(0), 0
    else:
        update = update.contiguous()
        stride, batch_stride = columns, rows * columns
    out = torch.empty(update.shape, dtype=update.dtype, device=update.device)
    need = _LIB.mgb_orthogonalize_workspace_bytes(batch, rows, columns)
    workspace = torch.empty(need, dtype=torch.uint8, device=update.device)
    with _on(update.device):
        _check_call(_LIB.mgb_orthogonalize(out.data_ptr(), update.data_ptr(), batch, rows, columns, stride,
                                           batch_stride, steps, (ctypes.c_float * 3)(*coefficients), eps, dtype,
                                           workspace.data_ptr(), need, _stream(update.device)))
    return out


class Muon(torch.optim.Optimizer):
    """Matrices by orthogonalised momentum: m = momentum m + grad, and
    w -= lr (sqrt(max(1, rows / columns)) orthogonalize(grad + momentum m) + weight_decay w)
    (without `nesterov` orthogonalize(m)).  For weights of two axes; biases,
    norms and embedding tables belong to another optimizer."""

    def __init__(self, params: Any, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5,
                 coefficients: Sequence[float] = (3.4445, -4.7750, 2.0315)) -> None:
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, coefficients=tuple(coefficients)))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"Muon takes matrices, got a parameter of shape {tuple(p.shape)}")

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
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(p)
                m = state["momentum"].mul_(group["momentum"]).add_(p.grad)
                update = torch.add(p.grad, m, alpha=group["momentum"]) if group["nesterov"] else m
                update = orthogonalize(update, steps=group["steps"], coefficients=group["coefficients"])
                if group["weight_decay"]:
                    p.mul_(1.0 - group["lr"] * group["weight_decay"])
                p.add_(update, alpha=-group["lr"] * max(1.0, p.shape[0] / p.shape[1]) ** 0.5)
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
        trees = trees[:end] if end else trees
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
