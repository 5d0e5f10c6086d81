"""The leaf encoder's operators (xgboost.encoder) against plain 64-bit forms.

Tolerances: a sum of n binary32 terms is off by at most n 2^-24 of the terms'
absolute sum, whatever the order, and a result's rounding to its type by u
(2^-24, 2^-11 or 2^-8) of its value; `_near` adds both.  The pieces are
derived at each test.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = ["f32", "f16", "bf16"]
E32 = 2.0 ** -24


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _near(got, want, slack, what=""):
    """|got - want| <= slack + the rounding of want to got's type, everywhere."""
    dtype = got.dtype
    bound = slack + (want.abs() + slack) * U[dtype] + TINY[dtype]
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"


# ---- embedding -------------------------------------------------------------

def _lookup64(weight, tokens, scale, pool):
    """The sum in 64 bits and the absolute sum of its terms."""
    w = torch.cat([weight.double(), torch.zeros(1, weight.shape[1], dtype=torch.float64, device="cuda")])
    at = torch.where((tokens < 0) | (tokens >= len(weight)), len(weight), tokens.long())
    if not pool:
        return w[at] * scale, (w[at] * scale).abs()
    total = torch.zeros(*tokens.shape[:-1], weight.shape[1], dtype=torch.float64, device="cuda")
    size = total.clone()
    for j in range(tokens.shape[-1]):
        total += w[at[..., j]]
        size += w[at[..., j]].abs()
    return total * scale, size * abs(scale)


def _gradient64(grad, tokens, table, scale, pool):
    t = tokens if pool else tokens[..., None]
    t = t.reshape(-1, t.shape[-1])
    g = grad.double().reshape(len(t), -1) * scale
    total = torch.zeros(table + 1, g.shape[1], dtype=torch.float64, device="cuda")
    size, count = total.clone(), torch.zeros(table + 1, 1, dtype=torch.float64, device="cuda")
    for j in range(t.shape[1]):
        at = torch.where((t[:, j] < 0) | (t[:, j] >= table), table, t[:, j].long())
        total.index_add_(0, at, g)
        size.index_add_(0, at, g.abs())
        count.index_add_(0, at, torch.ones(len(t), 1, dtype=torch.float64, device="cuda"))
    return total[:table], size[:table], count[:table]


def _tokens(g, shape, table, dtype, absent):
    t = torch.randint(0, table, shape, generator=g, device="cuda", dtype=torch.int64)
    # Some frequent tokens, some outside the table on either side.
    t = torch.where(torch.rand(shape, generator=g, device="cuda") < 0.2, t % 3 % table, t)
    r = torch.rand(shape, generator=g, device="cuda")
    t = torch.where(r < absent / 2, torch.full_like(t, -1), t)
    t = torch.where((r >= absent / 2) & (r < absent), torch.full_like(t, table + 5), t)
    return t.to(dtype)


LOOKUPS = [
    # rows, bag (0: not pooled), table, dim
    (1, 0, 1, 1), (1, 0, 7, 64), (7, 0, 300, 33), (513, 0, 70000, 8), (100, 0, 50, 1024), (33, 0, 1000, 1001),
    (1, 1, 5, 3), (1, 100, 640, 32), (16, 100, 6400, 32), (3, 7, 20, 5), (257, 13, 130, 64), (1000, 9, 90, 100),
    (5, 3000, 100, 16), (4099, 30, 66000, 24), (50, 64, 640, 520), (2, 17, 17, 2),
]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,bag,table,dim", LOOKUPS)
def test_lookup_and_gradient(enc, rows, bag, table, dim, dtype):
    g = _gen(rows * 31 + bag * 7 + table + dim)
    token_type = torch.int32 if (rows + dim) % 2 else torch.int64
    pool = bag > 0
    tokens = _tokens(g, (rows, bag) if pool else (rows,), table, token_type, 0.1)
    weight = _randn(g, table, dim, dtype=dtype)
    scale = 1.0 / bag if pool else math.sqrt(dim)
    out = enc.embedding_lookup(weight, tokens, scale=scale, pool=pool)
    assert out.shape == (rows, dim) and out.dtype == dtype
    # `scale` itself is rounded to binary32: one more relative 2^-24, the product another.
    want, size = _lookup64(weight, tokens, scale, pool)
    _near(out, want, size * ((bag or 1) + 2) * E32, "lookup")
    grad = _randn(g, rows, dim, dtype=dtype)
    dw = enc.embedding_gradient(grad, tokens, table, scale=scale, pool=pool)
    assert dw.shape == (table, dim) and dw.dtype == dtype
    want, size, count = _gradient64(grad, tokens, table, scale, pool)
    _near(dw, want, size * (count + 2) * E32, "gradient")
    assert torch.equal(dw, enc.embedding_gradient(grad, tokens, table, scale=scale, pool=pool))


@pytest.mark.parametrize("tokens,table", [(100000, 1), (70001, 3), (40000, 40000), (5000, 16777300),
                                          (32768, 1), (30001, 3), (32768, 60000), (9, 300), (32769, 500)])
def test_gradient_of_frequent_and_rare_tokens(enc, tokens, table):
    """One token for everything (its sum crosses every group), few, each once,
    and keys of four digits."""
    g = _gen(tokens)
    t = torch.randperm(table, generator=g, device="cuda")[:tokens] if table >= tokens else \
        torch.randint(0, table, (tokens,), generator=g, device="cuda")
    grad = _randn(g, tokens, 12)
    dw = enc.embedding_gradient(grad, t, table)
    want, size, count = _gradient64(grad, t, table, 1.0, False)
    _near(dw, want, size * count * E32)


@pytest.mark.parametrize("rows,bag,table,dim,dtype", [
    (20011, 60, 900, 128, torch.bfloat16),   # windows of 32-bit entries, the last one short
    (9, 4000, 3, 500000, torch.float32),     # wide rows: more windows than rows
    (40000, 60, 50, 64, torch.float32),      # long tiles
    (3_000_000, 1, 2000, 8, torch.float16),  # windows of single tokens
    (70000, 1, 1 << 21, 4, torch.float32),   # 64-bit entries, three digits
    (300, 20, 1 << 26, 2, torch.float16),    # 64-bit entries in one workgroup
])
def test_gradient_sorts(enc, rows, bag, table, dim, dtype):
    """Each way the tokens are sorted and the windows summed, with tokens outside the table."""
    g = _gen(rows)
    tokens = _tokens(g, (rows, bag), table, torch.int32, 0.05)
    grad = _randn(g, rows, dim, dtype=dtype)
    dw = enc.embedding_gradient(grad, tokens, table, scale=0.5, pool=True)
    want, size, count = _gradient64(grad, tokens, table, 0.5, True)
    _near(dw, want, size * (count + 1) * E32)
    assert torch.equal(dw, enc.embedding_gradient(grad, tokens, table, scale=0.5, pool=True))


# Many rows: a column's tokens from a narrow range of the table, from all of it,
# or narrow ones followed by wide ones and narrow ones again; absent tokens among
# them and a column of nothing else; infinities in the table.
@pytest.mark.parametrize("wide", [(), (0,), (13,), (11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 21, 22)], ids=["narrow", "first", "one", "late"])
@pytest.mark.parametrize("rows,bag,leaves,dim,dtype,ids", [
    (131072, 23, 256, 64, torch.bfloat16, torch.int32),
    (140001, 23, 200, 32, torch.float32, torch.int64),
    (131100, 25, 250, 96, torch.float16, torch.int32),
    (131075, 24, 100, 128, torch.bfloat16, torch.int32),
])
def test_lookup_of_many_rows(enc, rows, bag, leaves, dim, dtype, ids, wide):
    g = _gen(rows + bag + len(wide))
    table = leaves * bag
    tokens = torch.randint(0, leaves, (rows, bag), generator=g, device="cuda") + leaves * torch.arange(bag, device="cuda")
    for c in wide:
        tokens[:, c] = torch.randint(0, table, (rows,), generator=g, device="cuda")
    gone = torch.rand(rows, bag, generator=g, device="cuda") < 0.01
    tokens = torch.where(gone, torch.where(tokens % 2 == 0, -1, table), tokens)
    tokens[:, 5] = -7
    tokens[rows - 3] = table + 1
    tokens = tokens.to(ids)
    weight = _randn(g, table, dim, dtype=dtype)
    weight[leaves * 2 + 1, 3] = float("inf")
    got = enc.embedding_lookup(weight, tokens, scale=0.25, pool=True)
    want, slack = torch.zeros(rows, dim, dtype=torch.float64, device="cuda"), torch.zeros(rows, dim, dtype=torch.float64, device="cuda")
    padded = torch.cat([weight.double(), torch.zeros(1, dim, dtype=torch.float64, device="cuda")])
    for column in tokens.long().unbind(1):
        each = padded[torch.where((column < 0) | (column >= table), table, column)] * 0.25
        want += each
        slack += each.abs()
    infinite = torch.isinf(want)
    assert torch.equal(infinite, torch.isinf(got)) and bool(infinite.any())
    # A sum of `bag` terms in binary32, then one rounding of the result.
    bound = slack * (bag + 2) * 2.0 ** -24 + want.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny
    assert bool(((got.double() - want).abs() <= bound)[~infinite].all())
    assert bool((got[rows - 3] == 0).all())


def test_lookup_leaves_unnamed_rows_alone(enc):
    """NaN and infinity in rows that no token names, row 0 among them, stay there."""
    weight = torch.ones(10, 40, device="cuda")
    weight[0] = float("nan")
    weight[9] = float("inf")
    tokens = torch.tensor([[1, -1, 10], [-1, -7, 2 ** 31 - 1], [3, 4, 5]], device="cuda", dtype=torch.int32)
    out = enc.embedding_lookup(weight, tokens, pool=True)
    assert out[:, 0].tolist() == [1.0, 0.0, 3.0] and torch.isfinite(out).all()
    assert torch.equal(enc.embedding_lookup(weight, tokens)[1], torch.zeros(3, 40, device="cuda"))
    grad = torch.full((3, 40), float("nan"), device="cuda")
    grad[0] = 1.0
    dw = enc.embedding_gradient(grad, tokens, 10, pool=True)
    assert dw[1].tolist() == [1.0] * 40 and torch.isnan(dw[3:6]).all()
    assert not dw[[0, 2, 6, 7, 8, 9]].any()


def test_lookup_empty_and_shaped(enc):
    weight = _randn(_gen(0), 20, 6)
    for shape in ((0,), (0, 5), (4, 0, 3)):
        t = torch.zeros(shape, dtype=torch.int64, device="cuda")
        assert enc.embedding_lookup(weight, t).shape == (*shape, 6)
        assert not enc.embedding_gradient(torch.zeros(*shape, 6, device="cuda"), t, 20).any()
    t = torch.zeros((3, 0), dtype=torch.int64, device="cuda")
    assert not enc.embedding_lookup(weight, t, pool=True).any()
    assert not enc.embedding_gradient(torch.ones(3, 6, device="cuda"), t, 20, pool=True).any()
    t = torch.arange(12, device="cuda").reshape(2, 3, 2)
    assert torch.equal(enc.embedding_lookup(weight, t), weight[t])
    assert torch.equal(enc.embedding_lookup(weight, t[..., 0]), weight[t[..., 0]])
    pooled = enc.embedding_lookup(weight, t, pool=True)
    assert pooled.shape == (2, 3, 6) and torch.equal(pooled, weight[t[..., 0]] + weight[t[..., 1]])
    assert torch.equal(enc.embedding_lookup(weight, torch.tensor(3, device="cuda")), weight[3])


def test_lookup_strides(enc):
    """Rows at a distance, backwards in columns (copied), at odd addresses, one row for all."""
    g = _gen(5)
    big = _randn(g, 50, 77, dtype=torch.float16)
    tokens = torch.randint(0, 50, (30, 4), generator=g, device="cuda")
    for weight in (big[:, 1:40], big[:, ::2], big[1:, 3:4], big.t()[:50, :44], big[::3]):
        t = tokens % len(weight)
        want, size = _lookup64(weight, t, 0.5, True)
        _near(enc.embedding_lookup(weight, t, scale=0.5, pool=True), want, size * 6 * E32)
    assert torch.equal(enc.embedding_lookup(big, tokens.t()), big[tokens.t()])
    for grad in (_randn(g, 30, 99)[:, 5:38], _randn(g, 33, 30).t(), _randn(g, 1, 33).expand(30, 33)):
        want, size, count = _gradient64(grad, tokens, 50, 2.0, True)
        _near(enc.embedding_gradient(grad, tokens, 50, scale=2.0, pool=True), want, size * (count + 1) * E32)


def test_embedding_beyond_32_bit_offsets(enc):
    table, dim = 35_000_000, 64
    weight = torch.zeros(table, dim, device="cuda", dtype=torch.float16)
    weight[-1], weight[table // 2] = 3.0, 2.0
    tokens = torch.tensor([table - 1, 0, table // 2, table], device="cuda")
    assert enc.embedding_lookup(weight, tokens)[:, 7].tolist() == [3.0, 0.0, 2.0, 0.0]
    del weight
    dw = enc.embedding_gradient(torch.ones(4, dim, device="cuda", dtype=torch.float16), tokens, table)
    assert dw[[table - 1, 0, table // 2, 5]].sum(1).tolist() == [64.0, 64.0, 64.0, 0.0]
    assert dw.view(torch.int32).count_nonzero().item() == 3 * 32


# ---- layer norm --------------------------------------------------------------

def _norm64(x, weight, bias, eps):
    """y, mean, rstd in 64 bits and how far the kernel's may be: the mean off by
    d = (D + 1) 2^-24 of the values' mean size; the variance relatively by
    (D + 4) 2^-24 and d^2 / (variance + eps); y by both, times the weight."""
    x = x.double()
    dim = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    variance = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = (variance + eps) ** -0.5
    d = (dim + 2) * E32 * x.abs().mean(-1, keepdim=True)
    relative = 0.5 * ((dim + 6) * E32 + d * d * rstd * rstd) + 4 * E32
    h = (x - mean) * rstd
    slack = h.abs() * (relative + 4 * E32) + d * rstd * (1 + relative)
    w = weight.double() if weight is not None else torch.ones(dim, dtype=torch.float64, device="cuda")
    b = bias.double() if bias is not None else torch.zeros(dim, dtype=torch.float64, device="cuda")
    return h * w + b, mean[..., 0], rstd[..., 0], slack * w.abs() + (h * w).abs() * E32, d[..., 0], relative[..., 0]


NORMS = [(1, 1), (3, 2), (16, 32), (5, 31), (1, 64), (65, 100), (1000, 129), (7, 1000), (33, 1024), (10, 1025), (4, 2048),
         (3, 4097), (9, 8192), (2, 8200), (3, 20000), (2, 32768), (2, 40001), (600, 17), (4500, 264)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,dim", NORMS)
def test_norm_and_gradient(enc, rows, dim, dtype):
    g = _gen(rows * 3 + dim)
    x = (_randn(g, rows, dim) + 3 * _randn(g, rows, 1)).to(dtype)
    wtype = torch.float32 if rows % 2 else dtype
    weight, bias = _randn(g, dim, dtype=wtype), _randn(g, dim, dtype=wtype)
    if dim % 5 == 0:
        bias = None
    eps = 1e-5
    y, mean, rstd = enc.layer_norm(x, weight, bias, eps=eps)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == torch.float32 and mean.shape == rstd.shape == (rows,)
    want, wmean, wrstd, slack, d, relative = _norm64(x, weight, bias, eps)
    _near(y, want, slack, "y")
    _near(mean, wmean, d, "mean")
    _near(rstd, wrstd, wrstd * relative, "rstd")
    grad = _randn(g, rows, dim, dtype=dtype)
    dx, dw, db = enc.layer_norm_gradient(grad, x, mean, rstd, weight)
    assert dx.dtype == dtype and dw.dtype == db.dtype == wtype and dw.shape == db.shape == (dim,)
    # From the same statistics: h is off by 3 roundings, g by one, the row's two
    # means by (D + 4) 2^-24 of their terms' mean size, dx by a few roundings of
    # its three terms.
    m, r, dy = mean.double()[:, None], rstd.double()[:, None], grad.double()
    h = (x.double() - m) * r
    gw = dy * weight.double()
    s1, s2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    a1, a2 = gw.abs().mean(1, keepdim=True), (gw * h).abs().mean(1, keepdim=True)
    want = r * (gw - s1 - h * s2)
    slack = r * ((dim + 8) * E32 * (a1 + h.abs() * a2) + 8 * E32 * (gw.abs() + s1.abs() + (h * s2).abs()))
    _near(dx, want, slack, "dx")
    _near(dw, (dy * h).sum(0), (rows + 6) * E32 * (dy * h).abs().sum(0), "dweight")
    _near(db, dy.sum(0), (rows + 2) * E32 * dy.abs().sum(0), "dbias")
    again = enc.layer_norm_gradient(grad, x, mean, rstd, weight)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))
    plain, dwn, dbn = enc.layer_norm_gradient(grad, x, mean, rstd)
    assert dwn is None and dbn is None
    gw = dy
    s1, s2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    a1, a2 = gw.abs().mean(1, keepdim=True), (gw * h).abs().mean(1, keepdim=True)
    slack = r * ((dim + 8) * E32 * (a1 + h.abs() * a2) + 8 * E32 * (gw.abs() + s1.abs() + (h * s2).abs()))
    _near(plain, r * (gw - s1 - h * s2), slack, "dx without a weight")


def test_norm_far_from_zero_and_constant_rows(enc):
    """A row of one value has variance 0: y is the bias, rstd 1 / sqrt(eps).
    Rows at 1e4 keep their spread of 1."""
    x = torch.full((3, 256), 1.0, device="cuda")
    bias = _randn(_gen(1), 256)
    y, mean, rstd = enc.layer_norm(x, torch.ones(256, device="cuda"), bias)
    assert torch.equal(y, bias.expand(3, 256)) and mean.tolist() == [1.0] * 3
    assert torch.allclose(rstd.double(), torch.full((3,), 1e-5 ** -0.5, dtype=torch.float64, device="cuda"), rtol=2 ** -22, atol=0)
    x = _randn(_gen(2), 40, 512) + 1e4
    y, mean, rstd = enc.layer_norm(x)
    want, _, _, slack, _, _ = _norm64(x, None, None, 1e-5)
    _near(y, want, slack)


def test_norm_infinities_stay_in_their_row(enc):
    x = _randn(_gen(3), 5, 100)
    x[1, 7], x[3, 99] = float("inf"), float("nan")
    y, mean, rstd = enc.layer_norm(x)
    assert torch.isnan(y[1]).any() and torch.isnan(y[3]).all()
    assert torch.isfinite(y[[0, 2, 4]]).all() and torch.isfinite(mean[[0, 2, 4]]).all()


def test_norm_strides_and_empty(enc):
    g = _gen(9)
    big = _randn(g, 40, 90, dtype=torch.bfloat16)
    grad_big = _randn(g, 40, 120, dtype=torch.bfloat16)
    w = _randn(g, 90, dtype=torch.bfloat16)
    for x, grad in ((big[:, 3:60], grad_big[:, 7:64]), (big[::3, :33], grad_big[::3, :33]),
                    (big.t()[:33, :40], grad_big.t()[:33, :40]), (big[:1].expand(7, 90), grad_big[:7, :90])):
        weight = w[:x.shape[1]]
        y, mean, rstd = enc.layer_norm(x, weight, weight)
        same = enc.layer_norm(x.contiguous(), weight.clone(), weight.clone())
        assert all(torch.equal(p, q) for p, q in zip((y, mean, rstd), same))
        got = enc.layer_norm_gradient(grad, x, mean, rstd, weight)
        same = enc.layer_norm_gradient(grad.contiguous(), x.contiguous(), mean, rstd, weight)
        assert all(torch.equal(p, q) for p, q in zip(got, same))
    x = torch.zeros(0, 70, device="cuda")
    y, mean, rstd = enc.layer_norm(x)
    assert y.shape == (0, 70) and mean.shape == (0,)
    for dim in (70, 50000):
        x = torch.zeros(0, dim, device="cuda")
        dx, dw, db = enc.layer_norm_gradient(x, x, mean, rstd, torch.ones(dim, device="cuda"))
        assert dx.shape == (0, dim) and not dw.any() and not db.any()
    x = _randn(g, 2, 3, 4, 20)
    y, mean, rstd = enc.layer_norm(x)
    assert y.shape == x.shape and mean.shape == (2, 3, 4)
    one = enc.layer_norm(x[0, 0, 0])
    assert torch.equal(one[0], y[0, 0, 0]) and one[1].shape == ()


def test_norm_beyond_32_bit_offsets(enc):
    rows, dim = 4_300_000, 512
    x = torch.zeros(rows, dim, device="cuda", dtype=torch.float16)
    x[-3:] = _randn(_gen(4), 3, dim, dtype=torch.float16)
    y, mean, rstd = enc.layer_norm(x)
    tail = enc.layer_norm(x[-3:].clone())
    assert torch.equal(y[-3:], tail[0]) and torch.equal(mean[-3:], tail[1])
    dx, _, _ = enc.layer_norm_gradient(x, x, mean, rstd)
    assert torch.equal(dx[-3:], enc.layer_norm_gradient(x[-3:].clone(), x[-3:].clone(), *tail[1:])[0])


# ---- orthogonalize -------------------------------------------------------------

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _orthogonal64(update, steps, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = update.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    for _ in range(steps):
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT.contiguous() if tall else x


def _close_matrix(got, want, dtype, steps):
    """An operand's rounding, 2^-22 of X's size, grows a-fold a step where X is
    small, and a^2-fold in A inside a segment of three: at most
    (a^steps + 5 a^4) 2^-22 of the norm, and the type's rounding of each entry."""
    a = COEFFICIENTS[0]
    bound = (a ** min(steps, 5) + 5 * a ** 4) * 2.0 ** -22 + U[dtype]
    off = (got.double() - want).norm() / want.norm()
    assert off <= bound, f"{off:.2e} of the norm, bound {bound:.2e}"


MATRICES = [(1, 1), (1, 9), (9, 1), (3, 7), (16, 16), (64, 64), (64, 256), (65, 129), (200, 64), (130, 1000), (1000, 131),
            (300, 301), (512, 512)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,columns", MATRICES)
def test_orthogonalize(enc, rows, columns, dtype):
    g = _gen(rows + columns)
    update = (_randn(g, rows, columns) * 0.01).to(dtype)
    got = enc.orthogonalize(update)
    assert got.shape == update.shape and got.dtype == dtype
    _close_matrix(got, _orthogonal64(update, 5), dtype, 5)
    assert torch.equal(got, enc.orthogonalize(update))


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7])
def test_orthogonalize_steps_and_low_rank(enc, steps):
    """Few directions above noise a thousand times smaller."""
    g = _gen(steps)
    update = _randn(g, 96, 4) @ _randn(g, 4, 300) + 1e-3 * _randn(g, 96, 300)
    got = enc.orthogonalize(update, steps=steps)
    _close_matrix(got, _orthogonal64(update, steps), torch.float32, steps)
    got = enc.orthogonalize(update.t(), steps=steps)
    _close_matrix(got, _orthogonal64(update.t(), steps), torch.float32, steps)


def test_orthogonalize_singular_values(enc):
    """The result has the update's singular vectors and the polynomial of its singular values."""
    g = _gen(77)
    update = _randn(g, 80, 120)
    u, s, vt = np.linalg.svd(update.double().cpu().numpy(), full_matrices=False)
    s = s / np.linalg.norm(s)
    for _ in range(5):
        s = COEFFICIENTS[0] * s + COEFFICIENTS[1] * s ** 3 + COEFFICIENTS[2] * s ** 5
    want = torch.from_numpy(u * s @ vt).cuda()
    _close_matrix(enc.orthogonalize(update), want, torch.float32, 5)
    assert 0.5 < s.min() and s.max() < 1.3


def test_orthogonalize_other_coefficients(enc):
    g = _gen(78)
    update = _randn(g, 70, 90)
    for coefficients in ((2.0, -1.5, 0.5), (1.5, -0.5, 0.0)):
        got = enc.orthogonalize(update, steps=4, coefficients=coefficients)
        _close_matrix(got, _orthogonal64(update, 4, coefficients), torch.float32, 4)


def test_orthogonalize_batch_and_strides(enc):
    g = _gen(80)
    batch = _randn(g, 2, 3, 50, 70)
    got = enc.orthogonalize(batch)
    for i in range(2):
        for j in range(3):
            assert torch.equal(got[i, j], enc.orthogonalize(batch[i, j]))
    big = _randn(g, 90, 200)
    for update in (big[3:80, 5:105], big.t(), big[::2, 1::2], big[:, :1]):
        assert torch.equal(enc.orthogonalize(update), enc.orthogonalize(update.clone(memory_format=torch.contiguous_format)))


def test_orthogonalize_zero_and_not_finite(enc):
    assert not enc.orthogonalize(torch.zeros(30, 40, device="cuda")).any()
    for shape in ((0, 5), (5, 0), (0, 4, 4)):
        assert enc.orthogonalize(torch.zeros(shape, device="cuda")).shape == shape
    bad = _randn(_gen(1), 20, 30)
    bad[2, 3] = float("nan")
    assert torch.isnan(enc.orthogonalize(bad)).all()
    # One value far above the others.
    peak = _randn(_gen(2), 40, 40) * 1e-4
    peak[5, 6] = 50.0
    _close_matrix(enc.orthogonalize(peak), _orthogonal64(peak, 5), torch.float32, 5)


# ---- gradients against differences ---------------------------------------------

def test_gradients_against_differences(enc):
    """Central differences of the 64-bit forms along random directions, step 1e-4:
    off by the third derivative's 1e-8 and 1e-16 / 1e-4; binary32's own 1e-5."""
    g = _gen(100)
    x, w, b, dy = (_randn(g, *s) for s in ((6, 50), (50,), (50,), (6, 50)))
    _, mean, rstd = enc.layer_norm(x, w, b)
    grads = enc.layer_norm_gradient(dy, x, mean, rstd, w)
    values = [x.double(), w.double(), b.double()]
    for k in range(3):
        v = torch.randn(values[k].shape, generator=g, device="cuda", dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = [t + (sign * 1e-4 * v if i == k else 0) for i, t in enumerate(values)]
            ends.append((_norm64(moved[0], moved[1], moved[2], 1e-5)[0] * dy.double()).sum().item())
        slope = (ends[0] - ends[1]) / 2e-4
        got = (grads[k].double() * v).sum().item()
        assert abs(got - slope) <= 1e-5 * (grads[k].double() * v).abs().sum().item() + 1e-6
    weight, tokens, dy = _randn(g, 20, 9), torch.randint(-1, 20, (8, 5), generator=g, device="cuda"), _randn(g, 8, 9)
    dw = enc.embedding_gradient(dy, tokens, 20, scale=0.3, pool=True)
    v = _randn(g, 20, 9).double()
    slope = sum(s * (_lookup64(weight.double() + s * 1e-2 * v, tokens, 0.3, True)[0] * dy.double()).sum().item()
                for s in (1, -1)) / 2e-2
    assert abs((dw.double() * v).sum().item() - slope) <= 1e-5 * (dw.double() * v).abs().sum().item()


def test_autograd(enc):
    """The modules' gradients are the operators'; what needs none gets none."""
    g = _gen(101)
    emb, norm = enc.Embedding(30, 16, scale=0.25, pool=True), enc.LayerNorm(16)
    tokens = torch.randint(0, 30, (12, 6), generator=g, device="cuda")
    dy = _randn(g, 12, 16)
    pooled = emb(tokens)
    pooled.retain_grad()
    y = norm(pooled)
    y.backward(dy)
    _, mean, rstd = enc.layer_norm(pooled.detach(), norm.weight.detach(), norm.bias.detach())
    dx, dw, db = enc.layer_norm_gradient(dy, pooled.detach(), mean, rstd, norm.weight.detach())
    assert torch.equal(pooled.grad, dx) and torch.equal(norm.weight.grad, dw) and torch.equal(norm.bias.grad, db)
    assert torch.equal(emb.weight.grad, enc.embedding_gradient(dx, tokens, 30, scale=0.25, pool=True))
    x = _randn(g, 4, 16).requires_grad_()
    y, mean, rstd = enc.layer_norm(x)
    assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
    y.sum().backward()
    assert x.grad is not None
    with torch.no_grad():
        assert not enc.layer_norm(x)[0].requires_grad and not emb(tokens).requires_grad


# ---- streams and graphs ----------------------------------------------------------

def _everything(enc, s):
    y, mean, rstd = enc.layer_norm(s["x"], s["w"], s["b"])
    return (enc.embedding_lookup(s["table"], s["tokens"], pool=True),
            enc.embedding_gradient(s["x"], s["tokens"], len(s["table"]), pool=True), y, mean, rstd,
            *enc.layer_norm_gradient(s["x"], y, mean, rstd, s["w"]), enc.orthogonalize(s["x"]))


def _state(seed):
    g = _gen(seed)
    return {"x": _randn(g, 300, 96), "w": _randn(g, 96), "b": _randn(g, 96), "table": _randn(g, 500, 96),
            "tokens": torch.randint(0, 500, (300, 40), generator=g, device="cuda")}


def test_other_stream(enc):
    """Inputs made on a side stream that is still busy, used there."""
    want = _everything(enc, _state(1))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            a = a @ a * 1e-4
        state = _state(1)
        got = _everything(enc, state)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_graph_replays(enc):
    """Captured once, replayed over other inputs, with eager calls between."""
    state = _state(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _everything(enc, state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _everything(enc, state)
    for seed in (3, 4, 2, 5):
        new = _state(seed)
        for k, t in state.items():
            t.copy_(new[k])
        graph.replay()
        torch.cuda.synchronize()
        want = _everything(enc, new)
        assert all(torch.equal(p, q) for p, q in zip(out, want)), seed


# ---- from trees to a trained encoder ---------------------------------------------

def test_leaf_tokens_and_training(enc, xgb):
    """Tokens are the leaves pred_leaf gives; a small encoder on them learns."""
    rng = np.random.default_rng(3)
    X = rng.normal(size=(2000, 6)).astype(np.float32)
    y = (X[:, 0] * X[:, 1] + np.abs(X[:, 2])).astype(np.float32)
    d = xgb.DMatrix(X, label=y)
    bst = xgb.train({"max_depth": 4, "objective": "reg:squarederror"}, d, 20)
    tok = enc.LeafTokenizer(bst)
    tokens = tok(d)
    assert tokens.shape == (2000, 20) and tokens.dtype == torch.int32 and tokens.is_cuda
    leaves = bst.predict(d, pred_leaf=True).astype(np.int64)
    trees = bst.trees_to_json()
    first, t = 0, tokens.cpu().numpy()
    for k, tree in enumerate(trees):
        ids = np.flatnonzero(np.asarray(tree["left_children"]) == -1)
        np.testing.assert_array_equal(ids[t[:, k] - first], leaves[:, k])
        first += len(ids)
    assert tok.vocabulary == first
    assert torch.equal(enc.LeafTokenizer(bst, (0, 5))(d), tokens[:, :5])
    torch.manual_seed(0)
    emb, norm = enc.Embedding(tok.vocabulary, 32, scale=20 ** -0.5, pool=True), enc.LayerNorm(32)
    inner = torch.nn.Linear(32, 32, device="cuda")
    head = torch.nn.Linear(32, 1, device="cuda")
    muon = enc.Muon([inner.weight], lr=0.02)
    adam = torch.optim.Adam([emb.weight, norm.weight, norm.bias, inner.bias, *head.parameters()], lr=0.01)
    target = torch.from_numpy(y - y.mean()).cuda()
    losses = []
    for _ in range(60):
        out = head(torch.relu(inner(norm(emb(tokens)))))[:, 0]
        loss = (out - target).square().mean()
        muon.zero_grad()
        adam.zero_grad()
        loss.backward()
        muon.step()
        adam.step()
        losses.append(loss.item())
    assert losses[-1] < 0.25 * losses[0]


def test_example():
    """The example trains an encoder on the leaves that predicts what the trees do, about as well."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parents[1] / "examples" / "leaf_encoder.py"
    spec = importlib.util.spec_from_file_location("leaf_encoder", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    trees, leaves = example.main(rows=8000, rounds=20, dim=32, hidden=64, batch=1000, epochs=15)
    assert leaves < 1.5 * trees


def test_negated_views(enc):
    """A view that torch negates on reading is read negated, as what it stands for."""
    g = _gen(31)
    x, dy, table, w, update = (_randn(g, *s) for s in ((6, 40), (6, 40), (9, 40), (40,), (20, 30)))
    tokens = torch.randint(0, 9, (6, 5), generator=g, device="cuda")
    y, mean, rstd = enc.layer_norm(x, w, w)
    for call, values in ((lambda t: enc.embedding_lookup(t, tokens, pool=True), (table,)),
                         (lambda t: enc.embedding_gradient(t, tokens, 9, pool=True), (dy,)),
                         (lambda t: enc.embedding_lookup(table, t), (tokens,)),
                         (lambda t: enc.orthogonalize(t), (update,)),
                         (lambda t: enc.layer_norm(t, w, w), (x,)), (lambda t: enc.layer_norm(x, t, w), (w,)),
                         (lambda t: enc.layer_norm(x, w, t), (w,)),
                         (lambda t: enc.layer_norm_gradient(t, x, mean, rstd, w), (dy,)),
                         (lambda t: enc.layer_norm_gradient(dy, t, mean, rstd, w), (x,)),
                         (lambda t: enc.layer_norm_gradient(dy, x, t, rstd, w), (mean,)),
                         (lambda t: enc.layer_norm_gradient(dy, x, mean, t, w), (rstd,)),
                         (lambda t: enc.layer_norm_gradient(dy, x, mean, rstd, t), (w,))):
        value, = values
        got, want = call(torch._neg_view(-value)), call(value)
        if isinstance(got, torch.Tensor):
            got, want = (got,), (want,)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        got = call(torch._neg_view(value))
        got = (got,) if isinstance(got, torch.Tensor) else got
        want = call(-value)
        want = (want,) if isinstance(want, torch.Tensor) else want
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_results_without_a_derivative_say_so(enc):
    """What has no derivative gives values as ever, and an error where a gradient
    would have to pass it, not a graph that ends there without a word."""
    g = _gen(41)
    x, dy, w = (_randn(g, *s) for s in ((6, 20), (6, 20), (20,)))
    tokens = torch.randint(0, 5, (6,), generator=g, device="cuda")
    _, mean, rstd = enc.layer_norm(x, w)
    for call, given in ((lambda t: enc.orthogonalize(t), x), (lambda t: enc.embedding_gradient(t, tokens, 5), dy),
                        (lambda t: enc.layer_norm_gradient(t, x, mean, rstd, w), dy),
                        (lambda t: enc.layer_norm_gradient(dy, t, mean, rstd), x),
                        (lambda t: enc.layer_norm_gradient(dy, x, mean, rstd, t), w)):
        leaf = given.clone().requires_grad_()
        want, got = call(given), call(leaf)
        want, got = ((want,), (got,)) if isinstance(want, torch.Tensor) else (want, got)
        for p, q in zip(want, got):
            assert (p is None) == (q is None)
            if p is not None:
                assert torch.equal(p, q.detach()) and q.requires_grad and not p.requires_grad
        with pytest.raises(NotImplementedError, match="derivative"):
            got[0].sum().backward()
        with torch.no_grad():
            out = call(leaf)
            assert not (out if isinstance(out, torch.Tensor) else out[0]).requires_grad
    # Twice through the differentiable ones is an error as before.
    x = x.requires_grad_()
    once, = torch.autograd.grad(enc.layer_norm(x)[0].square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        once.sum().backward()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("dim", [2, 33, 512, 768, 777, 1000, 4100, 8192, 20000, 33000, 40001])
def test_norm_far_from_zero(enc, dim, dtype):
    """Rows of one value (y 0, the mean the value), and rows whose spread is small
    against their mean.  No value takes part in more than 80 additions of a sum
    (40 of a lane, 6 steps in a wave, 16 waves, and a few roundings), so a sum is
    off by 80 2^-24 of its terms' sizes: the first mean by d of the row's, what is
    left of it after centring by 80 2^-24 of the centred sizes, s at most, and y by
    that and a few roundings of a centred value, times rstd; the variance by its
    sum's and the square of that."""
    g = _gen(dim)
    rows = [torch.full((dim,), v, device="cuda") for v in (10000.1, 100000.3, 1234.567, -777.77, 3.0e-3)]
    rows += [_randn(g, dim) * spread + at for spread, at in ((1.0, 1e4), (1e-2, 300.0), (1.0, -6e4), (1e-3, 0.1))]
    x = torch.stack(rows).clamp(-65000, 65000).to(dtype)
    y, mean, rstd = enc.layer_norm(x)
    v = x.double()
    wmean = v.mean(1)
    centred = v - wmean[:, None]
    wrstd = (centred.square().mean(1) + 1e-5) ** -0.5
    d = 80 * E32 * v.abs().mean(1)
    s = centred.abs().mean(1) + d
    off = 80 * E32 * s + 4 * E32 * d
    relative = 0.5 * (84 * E32 + off ** 2 * wrstd ** 2) + 4 * E32
    h = centred * wrstd[:, None]
    slack = wrstd[:, None] * (off[:, None] + 4 * E32 * centred.abs()) + h.abs() * relative[:, None]
    _near(y, h, slack, "y")
    _near(mean, wmean, off, "mean")
    _near(rstd, wrstd, wrstd * relative, "rstd")
    # The rows of one value have that mean, and so gradients without h.
    assert torch.equal(mean[:5], x[:5, 0].float())
    grad = _randn(g, len(x), dim, dtype=dtype)
    dx, dw, db = enc.layer_norm_gradient(grad[:5], x[:5], mean[:5], rstd[:5], torch.ones(dim, device="cuda"))
    assert not dw.any()
    g64 = grad[:5].double()
    want = wrstd[:5, None] * (g64 - g64.mean(1, keepdim=True))
    _near(dx, want, wrstd[:5, None] * (relative[:5, None] + (dim + 8) * E32) * (g64.abs() + g64.abs().mean(1, keepdim=True)), "dx")


def test_leaf_tokens_of_rounds(enc, xgb):
    """An end below 1 means all rounds and one beyond them the last, as in Booster.predict."""
    rng = np.random.default_rng(5)
    X = rng.normal(size=(300, 4)).astype(np.float32)
    d = xgb.DMatrix(X, label=X[:, 0])
    bst = xgb.train({"max_depth": 3}, d, 4)
    whole = enc.LeafTokenizer(bst)(d)
    for end in (0, -1, -3, 4, 9, 2):
        tok = enc.LeafTokenizer(bst, (0, end))
        leaves = bst.predict(d, pred_leaf=True, iteration_range=(0, end)).reshape(300, -1)
        assert tok.trees == leaves.shape[1] and torch.equal(tok(d), whole[:, :tok.trees])


def test_pooled_beyond_32_bit_offsets(enc):
    """Rows of the table, and of the gradient, more than 4 GB apart."""
    rows, stride = 1100, 2_000_000
    big = torch.zeros(rows, stride, device="cuda", dtype=torch.float16)  # 4.4 GB
    g = _gen(11)
    big[:, 5:45] = _randn(g, rows, 40, dtype=torch.float16)
    weight = big[:, 5:45]
    tokens = torch.randint(-1, rows + 1, (300, 17), generator=g, device="cuda")
    tokens[0, 0] = rows - 1
    want, size = _lookup64(weight, tokens, 0.5, True)
    _near(enc.embedding_lookup(weight, tokens, scale=0.5, pool=True), want, size * 19 * E32)
    # 200 tokens a row: more than one launch takes; and fewer, which one does.
    for bag in (200, 10):
        tokens = _tokens(g, (rows, bag), 700, torch.int32, 0.1)
        want, size, count = _gradient64(weight, tokens, 700, 2.0, True)
        _near(enc.embedding_gradient(weight, tokens, 700, scale=2.0, pool=True), want, size * (count + 1) * E32)


@pytest.mark.parametrize("dim", [3, 100, 5000, 40001])
def test_norm_statistics_of_infinite_rows(enc, dim):
    """The mean of a row with infinities is what their sum is; rstd is not a number, nor is y."""
    x = _randn(_gen(6), 5, dim)
    inf = float("inf")
    x[0, 1], x[1, 0], x[2, dim - 1] = inf, -inf, float("nan")
    x[3, 0], x[3, 2] = inf, -inf
    y, mean, rstd = enc.layer_norm(x)
    assert mean[0].item() == inf and mean[1].item() == -inf and torch.isnan(mean[2:4]).all()
    assert torch.isnan(rstd[:4]).all() and torch.isnan(y[:4]).all()
    assert torch.isfinite(mean[4]) and torch.isfinite(y[4]).all()
