"""The encoder's products at sizes whose tiles, shares of the depth and ends the other
tests do not reach (xgboost.encoder): tiles of 256 x 256 of every form, whole, in equal
shares and with a longer first one, hidden values rounded to blocks where they are made,
rows of more blocks than 64 shares of 64.

Tolerances element by element are those of test_gpu_block.py and test_gpu_block8.py;
of many terms they leave room for a wrong step.  The norms do not: a result's own
rounding and those of up to three inner factors are each at most u of the norm and
independent of each other, so 2 u together; float32 sums of n terms (of three parts
each, six products) go 2^-23 a term astray at random, sqrt(6 n) 2^-23 and twice
that at most.  One step of 32 among the depths below is 3 % of a norm or more.
"""
import pytest
import torch

from test_gpu_block import (E, NAMES, TYPES, U, _act, _case, _forward64, _gen, _gradient64, _inner64, _near, _randn)
from test_gpu_block8 import _blocks64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


def _norm_near(got, want, terms, what):
    bound = 2 * U[got.dtype] if got.dtype != torch.float32 else 2 * E * (6 * terms) ** 0.5
    off = (got.double() - want).norm() / want.norm()
    assert off <= bound, f"{what}: {off:.2e} of the norm, {bound:.2e} allowed"


TRAINED = [
    # rows, dim, hidden; t: with a transposed operand
    (101, 1000, 3001),     # matrices' gradients in large tiles, two steps of rows
    (1031, 500, 3001),     # f32: matrices' gradients in large tiles, shares
    (2051, 2000, 2051),    # 16 bits: the input's gradient in large tiles (t), shares
    (2051, 4000, 2051),    # f32: the input's gradient in large tiles, a longer first share; 16 bits: whole (t)
    (4001, 500, 3001),     # 16 bits: the first gradient product in large tiles (t); matrices' gradients, shares
    (4001, 1000, 3001),    # f32: matrices' gradients in large tiles, a longer first share
    (3001, 4000, 5000),    # f32: both outer products with a longer first share; 16 bits: the input's gradient so (t)
    (5001, 1544, 1001),    # 16 bits: y and the input's gradient in large tiles, whole
    (8001, 1032, 8200),    # 16 bits: y in large tiles, a longer first share
    (12001, 1000, 8201),   # 16 bits: the input's gradient in large tiles, a longer first share
    (12001, 1544, 2051),   # 16 bits: matrices' gradients in large tiles, a longer first share
]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,dim,hidden", TRAINED)
def test_block_and_gradient(enc, rows, dim, hidden, dtype):
    g = _gen(rows + dim + hidden)
    activation = "gelu" if (dim // 4 + hidden) % 2 else "silu"
    x, gate, up, down, grad = _case(g, rows, dim, hidden, dtype)
    y, kept = enc.feed_forward(x, gate, up, down, activation=activation, keep=True)
    want, error = _forward64(x, gate, up, down, activation)
    _near(y, want, error, "y")
    _norm_near(y, want, hidden, "y")
    assert torch.equal(y, enc.feed_forward(x, gate, up, down, activation=activation))
    for k, (want, error) in enumerate(_inner64(x, gate, up, dtype)):
        _near(kept[:, k], want, error, "kept")
        _norm_near(kept[:, k], want, dim, "kept")
    del want, error
    got = enc.feed_forward_gradient(grad, x, kept, gate, up, down, activation=activation)
    wants = _gradient64(grad, x, kept, gate, up, down, activation)
    for name, out, terms, (want, error) in zip(("dx", "dgate", "dup", "ddown"), got, (2 * hidden, rows, rows, rows), wants):
        _near(out, want, error, name)
        _norm_near(out, want, terms, name)


SERVED = [
    (101, 500, 8201),      # widened, medium tiles
    (2051, 500, 2051),     # hidden values rounded in large tiles
    (2051, 500, 5001),     # the last product in medium tiles, shares
    (2051, 2000, 8200),    # in large tiles, shares
    (2051, 8320, 2000),    # rows of more than 64 blocks: widened, large tiles
    (5001, 1544, 1001),    # the last product in large tiles, whole
    (8001, 1032, 8200),    # with a longer first share
]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,dim,hidden", SERVED)
def test_block_feed_forward(enc, rows, dim, hidden, dtype):
    """Against the 64-bit form that rounds the hidden values so.  Those that lie next to a
    border of e4m3 fall on either side, a sixteenth of themselves apart: with products off by
    2^-12 of sums like a norm's, up to 1 in 50 of them, 0.9 % of the norm.  One block of the
    depths is 12 %."""
    g = _gen(rows + dim + hidden)
    activation = "gelu" if hidden % 2 else "silu"
    x = _randn(g, rows, dim, dtype=dtype)
    x[5] = 0
    gate, up = (enc.quantize_blocks(_randn(g, hidden, dim, scale=dim ** -0.5)) for _ in range(2))
    down = enc.quantize_blocks(_randn(g, dim, hidden, scale=hidden ** -0.5))
    got = enc.block_feed_forward(x, gate, up, down, activation=activation)
    v = enc.quantize_blocks(x).dequantize().double()
    h = _act(v @ gate.dequantize().double().t(), activation)[0] * (v @ up.dequantize().double().t())
    values, exponent = _blocks64(h)
    h = (values.view(rows, -1, 128) * torch.exp2(exponent)[..., None]).flatten(1)[:, :hidden]
    want = h @ down.dequantize().double().t()
    off = (got.double() - want).norm(dim=1)
    assert (off <= 0.03 * want.norm(dim=1)).all() and off.norm() <= 0.01 * want.norm()
    assert (got[5] == 0).all()
    assert torch.equal(got, enc.block_feed_forward(x, gate, up, down, activation=activation))
    other = x.clone()
    other[7] = float("nan")
    again = enc.block_feed_forward(other, gate, up, down, activation=activation)
    there = torch.arange(rows, device="cuda") != 7
    assert torch.equal(again[there], got[there]) and torch.isnan(again[7]).all()


PRODUCTS = [(4001, 500, 2051), (2051, 8200, 2000), (8001, 8200, 1032), (5001, 1001, 1544)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,dim,out", PRODUCTS)
def test_block_matmul(enc, rows, dim, out, dtype):
    """Large tiles, whole, in shares and with a longer first one; each block's scale its own."""
    g = _gen(rows + 3 * dim + out)
    grow = torch.exp2(torch.randint(-5, 6, (rows + out, (dim + 127) // 128), generator=g, device="cuda").float())
    both = _randn(g, rows + out, dim, scale=2.0 ** -6) * grow.repeat_interleave(128, 1)[:, :dim]
    x, w = enc.quantize_blocks(both[:rows]), enc.quantize_blocks(both[rows:])
    got = enc.block_matmul(x, w, dtype=dtype)
    a, b = x.dequantize().double(), w.dequantize().double()
    want, size = a @ b.t(), a.abs() @ b.t().abs()
    _near(got, want, size * ((dim + 2) * E if dtype == torch.float32 else 2.0 ** -12 + dim * E))
    _norm_near(got, want, dim, "product")
    assert torch.equal(got, enc.block_matmul(x, w, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,blocks", [(3, 8192), (40, 4096), (40, 4097), (70, 8192), (300, 5003)])
def test_rows_of_very_many_blocks(enc, rows, blocks, dtype):
    """Up to 2^20 values a row, more than 64 shares of 64 blocks.  One value of x for each
    16 blocks is 1 or -1 and the rest zeros, so that sums are whole numbers of at most 512
    terms, below 256, which every form has exactly, bfloat16 results too."""
    out, dim = 70, blocks * 128 - 5
    g = _gen(rows + blocks)
    x = torch.zeros(rows, dim, device="cuda")
    every = torch.arange(0, dim - 2048, 2048, device="cuda")
    at = every + torch.randint(0, 2048, (rows, len(every)), generator=g, device="cuda")
    x.scatter_(1, at, torch.where(torch.rand(rows, len(every), generator=g, device="cuda") < 0.2, -1.0, 1.0))
    w = torch.randint(-1, 2, (out, dim), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    got = enc.block_matmul(enc.quantize_blocks(x), enc.quantize_blocks(w), dtype=dtype)
    want = torch.stack([(x[k, at[k]].double() * w[:, at[k]].double()).sum(1) for k in range(rows)])
    assert want.abs().max() < 256
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("dtype", TYPES[1:], ids=NAMES[1:])
def test_hidden_values_of_very_many_blocks(enc, dtype):
    """A hidden side above 2^19: one hidden value of each 16 blocks is not zero, and equal
    to a whole number that all roundings keep."""
    rows, dim, hidden = 40, 64, 524_289
    g = _gen(7)
    x = torch.zeros(rows, dim, device="cuda", dtype=dtype)
    at = torch.arange(rows, device="cuda") % dim
    x[torch.arange(rows), at] = 1.0
    some = torch.arange(0, hidden, 2048, device="cuda")
    gate, up = torch.zeros(hidden, dim, device="cuda"), torch.zeros(hidden, dim, device="cuda")
    gate[some] = 64.0  # silu(64) is 64 in binary32
    up[some] = torch.randint(0, 3, (len(some), dim), generator=g, device="cuda").float() / 64
    down = torch.randint(-1, 2, (dim, hidden), generator=g, device="cuda").float()
    got = enc.block_feed_forward(x, *(enc.quantize_blocks(w) for w in (gate, up, down)))
    want = (64.0 * up[some].double()[:, at]).t() @ down[:, some].double().t()
    assert want.abs().max() < 256
    assert torch.equal(got.double(), want)
