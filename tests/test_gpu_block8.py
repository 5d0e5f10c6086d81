"""Products in 8 bits and distillation (xgboost.encoder) against plain 64-bit forms.

Rounding to blocks is exact arithmetic, so it is compared bit for bit.  Of 16-bit
results the 8-bit instructions keep about 16 bits of a few products' sums; each
product counts with 2^-12 of its size here, eight times what was seen of them.
Float32 results are sums of exact products: n 2^-23 of the absolute sum.  The
logarithm's and the exponential's arguments are off by a few 2^-24 of their size,
which is what their results are off by, relative.
"""
import math

import pytest
import torch

from test_gpu_block import E, NAMES, TINY, TYPES, U, _act, _gen, _near, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


def _blocks64(x):
    """Values and exponents of x's rows as blocks, in 64 bits (finite x)."""
    rows, dim = x.shape
    n = (dim + 127) // 128
    v = torch.zeros(rows, n * 128, dtype=torch.float64, device=x.device)
    v[:, :dim] = x.double()
    v = v.view(rows, n, 128)
    most = v.abs().amax(2)
    e = torch.ceil(torch.log2(torch.where(most > 0, most, 448.0) / 448.0))
    e = torch.where(most > 448.0 * torch.exp2(e), e + 1, e)       # log2's rounding
    e = torch.where(most <= 448.0 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(most > 0, e.clamp(min=-127), 0.0)
    s = v / torch.exp2(e)[..., None]
    step = torch.exp2(torch.floor(torch.log2(s.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(s / step) * step).flatten(1), e


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 127), (3, 128), (2, 129), (5, 640), (70, 1000), (1000, 257), (4099, 128), (2, 70000)])
def test_quantize(enc, rows, dim, dtype):
    g = _gen(rows + dim)
    # Blocks of very different sizes, some of zeros.
    size = torch.exp2(torch.randint(-12, 10, (rows, (dim + 127) // 128), generator=g, device="cuda").double())
    x = (_randn(g, rows, dim).double() * size.repeat_interleave(128, 1)[:, :dim]).to(dtype)
    x[rows // 2, :128] = 0
    got = enc.quantize_blocks(x)
    assert got.values.dtype == torch.float8_e4m3fn and got.scales.dtype == torch.float8_e8m0fnu and got.dim == dim
    values, exponent = _blocks64(x)
    assert torch.equal(got.values.double(), values)
    assert torch.equal(got.scales.view(torch.uint8).double(), exponent + 127)
    want = (values.view(rows, -1, 128) * torch.exp2(exponent)[..., None]).flatten(1)[:, :dim]
    assert torch.equal(got.dequantize().double(), want)
    wide = torch.full((rows + 1, dim + 5), float("nan"), device="cuda", dtype=dtype)
    wide[1:, 3:3 + dim] = x
    for view in (wide[1:, 3:3 + dim], x.t().contiguous().t(), x[None]):
        again = enc.quantize_blocks(view)
        assert torch.equal(again.values.view(torch.uint8).view(rows, -1), got.values.view(torch.uint8))
        assert torch.equal(again.scales.view(torch.uint8).reshape(rows, -1), got.scales.view(torch.uint8))


def test_quantize_borders(enc):
    """Ties, the largest value on either side of a power of two, subnormal blocks,
    binary32's ends, and what is not finite."""
    steps = torch.arange(0, 256, device="cuda", dtype=torch.float32)
    for top in (448.0, 449.0, 256.0, 255.9, 447.99, 224.0, 224.01, 1.0, 1.75, 1.7500001):
        for scale in (2.0 ** -149, 2.0 ** -140, 2.0 ** -126, 2.0 ** -60, 1.0, 2.0 ** 60, 2.0 ** 118):
            x = torch.cat([steps / 128 * top / 2, -steps / 3]).clamp(-top, top) * scale
            x[0] = top * scale
            x = x.view(4, 128)
            values, exponent = _blocks64(x)
            got = enc.quantize_blocks(x)
            assert torch.equal(got.values.double(), values), (top, scale)
            assert torch.equal(got.scales.view(torch.uint8).double(), exponent + 127), (top, scale)
    x = torch.linspace(-3, 3, 384, device="cuda").view(1, 384).repeat(3, 1)
    want = enc.quantize_blocks(x)
    bad = x.clone()
    bad[0, 5], bad[1, 200], bad[2, 300] = float("inf"), float("nan"), -float("inf")
    got = enc.quantize_blocks(bad)
    there = torch.isfinite(bad)
    assert torch.equal(got.values.float()[there], want.values.float()[there]) and torch.isnan(got.values.float()[~there]).all()
    assert torch.equal(got.scales.float(), want.scales.float())
    got = enc.quantize_blocks(torch.full((1, 128), float("inf"), device="cuda"))
    assert torch.isnan(got.values.float()).all() and got.scales.float().item() == 1.0
    got = enc.quantize_blocks(torch.full((2, 130), 3.4028234e38, device="cuda"))
    assert torch.equal(got.values.float()[:, :130], torch.full((2, 130), 256.0, device="cuda"))
    assert (got.values.float()[:, 130:] == 0).all()
    assert enc.quantize_blocks(torch.zeros(0, 5, device="cuda")).values.shape == (0, 128)


PRODUCTS = [(1, 1, 1), (1, 128, 16), (1, 4096, 1000), (2, 300, 7), (15, 129, 65), (16, 1024, 64), (33, 640, 129), (100, 257, 300),
            (300, 1000, 777), (1030, 384, 513), (2049, 1500, 1025), (5, 9000, 70), (300, 20000, 200)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,dim,out", PRODUCTS)
def test_block_matmul(enc, rows, dim, out, dtype):
    g = _gen(rows + 3 * dim + out)
    # Scales of every block of every row their own.
    blocks = (dim + 127) // 128
    grow = torch.exp2(torch.randint(-5, 6, (rows + out, blocks), generator=g, device="cuda").float())
    both = _randn(g, rows + out, dim) * grow.repeat_interleave(128, 1)[:, :dim]
    x, w = enc.quantize_blocks(both[:rows].contiguous()), enc.quantize_blocks(both[rows:].contiguous())
    got = enc.block_matmul(x, w, dtype=dtype)
    assert got.shape == (rows, out) and got.dtype == dtype
    a, b = x.dequantize().double(), w.dequantize().double()
    if dtype == torch.float16:  # keep within its range
        shrink = 2.0 ** -12
        x = enc.quantize_blocks(both[:rows] * shrink)
        a = x.dequantize().double()
        got = enc.block_matmul(x, w, dtype=dtype)
    want, size = a @ b.t(), a.abs() @ b.t().abs()
    _near(got, want, size * ((dim + 2) * E if dtype == torch.float32 else 2.0 ** -12 + dim * E))
    assert torch.equal(got, enc.block_matmul(x, w, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_block_matmul_exact_sums(enc, dtype):
    """Small whole numbers, whose sums every form has exactly: a row and a column of
    each tile and of each block, one at a time."""
    g = _gen(1)
    for rows, dim, out in ((1, 512, 40), (20, 260, 300), (200, 384, 700), (600, 256, 1100)):
        x = torch.zeros(rows, dim, device="cuda")
        x[torch.arange(rows), torch.randint(0, dim, (rows,), generator=g, device="cuda")] = torch.randint(1, 8, (rows,), generator=g, device="cuda").float()
        w = torch.randint(-8, 9, (out, dim), generator=g, device="cuda").float()
        got = enc.block_matmul(enc.quantize_blocks(x), enc.quantize_blocks(w), dtype=dtype)
        assert torch.equal(got.double(), x.double() @ w.double().t())


def test_blocks_that_a_program_made(enc):
    """Values and scales in other places than quantize_blocks puts them, more axes, no rows."""
    g = _gen(9)
    x, w = enc.quantize_blocks(_randn(g, 6, 5, 300)), enc.quantize_blocks(_randn(g, 50, 300))
    want = enc.block_matmul(x, w, dtype=torch.float32)
    assert want.shape == (6, 5, 50)
    wide = torch.zeros(50, 384 + 8, device="cuda", dtype=torch.uint8)
    wide[:, 4:388] = w.values.view(torch.uint8)
    values = wide[:, 4:388].view(torch.float8_e4m3fn)
    scales = w.scales.view(torch.uint8).contiguous().view(torch.float8_e8m0fnu)   # three bytes a row
    for v, s in ((values, w.scales), (w.values, scales), (values, scales)):
        assert torch.equal(enc.block_matmul(x, enc.BlockScaled(v, s, 300), dtype=torch.float32), want)
        assert torch.equal(enc.block_matmul(x, enc.BlockScaled(v, s, 300)), enc.block_matmul(x, w))
    tail = enc.BlockScaled(w.values[-1:], w.scales[-1:], 300)  # the last row of its storage
    assert torch.equal(enc.block_matmul(x, tail, dtype=torch.float32), want[..., -1:])
    assert enc.block_matmul(enc.BlockScaled(x.values[:0], x.scales[:0], 300), w).shape == (0, 5, 50)
    assert enc.block_matmul(x, enc.BlockScaled(w.values[:0], w.scales[:0], 300)).shape == (6, 5, 0)


SERVED = [(1, 1, 1), (1, 1024, 2048), (2, 100, 130), (16, 64, 256), (17, 129, 65), (130, 200, 777), (300, 640, 129), (1030, 256, 512),
          (2500, 512, 1100)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,dim,hidden", SERVED)
def test_block_feed_forward(enc, rows, dim, hidden, dtype):
    """Hidden values next to a border of e4m3 may fall on either side: a fraction of
    them by half a step or less each.  The bound takes every hidden value whose own
    error reaches a border as one whole step off."""
    g = _gen(rows + dim + hidden)
    activation = "gelu" if hidden % 2 else "silu"
    x = _randn(g, rows, dim, dtype=dtype)
    gate, up = (enc.quantize_blocks(_randn(g, hidden, dim, scale=dim ** -0.5)) for _ in range(2))
    down = enc.quantize_blocks(_randn(g, dim, hidden, scale=hidden ** -0.5))
    got = enc.block_feed_forward(x, gate, up, down, activation=activation)
    assert got.shape == x.shape and got.dtype == dtype
    v = enc.quantize_blocks(x).dequantize().double()
    wg, wu, wd = (m.dequantize().double() for m in (gate, up, down))
    each = 2.0 ** -12 if dtype == torch.bfloat16 else 0.0
    a, u = v @ wg.t(), v @ wu.t()
    ea, eu = ((v.abs() @ w.t().abs()) * (each + (dim + 2) * E) for w in (wg, wu))
    act, _ = _act(a, activation)
    h = act * u
    eh = (1.13 * ea + act.abs() * (a.abs() + 4) * E + a.abs() * 1e-6) * u.abs() + act.abs() * eu + h.abs() * E

    def kept(t):
        values, exponent = _blocks64(t)
        return (values.view(rows, -1, 128) * torch.exp2(exponent)[..., None]).flatten(1)[:, :hidden]

    # A block whose largest value may cross a power of two has the other scale as well.
    low, high = kept(h - eh), kept(h + eh)
    most = torch.stack([kept(h), low, high])
    moved = (most - most[0]).abs().amax(0) + eh * 0
    pad = torch.zeros(rows, (hidden + 127) // 128 * 128, device="cuda", dtype=torch.float64)
    pad[:, :hidden] = h.abs()
    top = pad.view(rows, -1, 128).amax(2)
    pad[:, :hidden] = eh
    reach = pad.view(rows, -1, 128).amax(2)
    edge = 448.0 * torch.exp2(torch.round(torch.log2(top.clamp(min=1e-300) / 448.0)))
    crossing = ((top - edge).abs() <= reach).repeat_interleave(128, 1)[:, :hidden]
    moved = torch.where(crossing, moved + h.abs() * 2.0 ** -3 + top.repeat_interleave(128, 1)[:, :hidden] * 2.0 ** -16, moved)
    want = kept(h) @ wd.t()
    size = (kept(h).abs() + moved) @ wd.t().abs()
    last = (hidden + 2) * E + (0.0 if dtype == torch.float32 else 2.0 ** -12)
    _near(got, want, moved @ wd.t().abs() + size * last)
    assert torch.equal(got, enc.block_feed_forward(x, gate, up, down, activation=activation))
    if rows > 2:
        wide = torch.full((rows, dim + 3), float("nan"), device="cuda", dtype=dtype)
        wide[:, 1:1 + dim] = x
        assert torch.equal(enc.block_feed_forward(wide[:, 1:1 + dim], gate, up, down, activation=activation), got)
        other = x.clone()
        other[1] = float("nan")
        again = enc.block_feed_forward(other, gate, up, down, activation=activation)
        assert torch.equal(again[2:], got[2:]) and torch.isnan(again[1]).all()


def test_quantized_module(enc):
    block = enc.FeedForward(100, 200)
    served = block.quantized()
    x = torch.randn(7, 100, device="cuda")
    want = served(x)
    assert torch.equal(want, enc.block_feed_forward(x, *(enc.quantize_blocks(w.detach()) for w in (block.gate, block.up, block.down))))
    other = enc.FeedForward(100, 200).quantized()
    other.load_state_dict(served.state_dict())
    assert torch.equal(other(x), want)
    assert enc.block_feed_forward(x[:0], *(enc.quantize_blocks(w.detach()) for w in (block.gate, block.up, block.down))).shape == (0, 100)


# ---- distillation ------------------------------------------------------------------

def _distil64(logits, values, indices, temperature):
    """loss, lse, the gradient for a loss's gradient of 1, and the errors of the first two and
    (relative to q + p) of the last."""
    classes = logits.shape[-1]
    z = logits.double() / temperature
    lse = z.logsumexp(-1)
    there = (indices >= 0) & (indices < classes) & (values != -math.inf)
    t = torch.where(there, values.double() / temperature, -math.inf)
    some = there.any(-1)
    log_p = torch.where(some[..., None], t - t.logsumexp(-1, keepdim=True), -math.inf)
    p = log_p.exp()
    at = torch.where(there, indices.long(), 0)
    log_q = z.gather(-1, at) - lse[..., None]
    each = torch.where(p > 0, p * (log_p - log_q), 0.0)
    finite_z = torch.where(torch.isfinite(z), z, 0.0).abs().amax(-1)
    lse_error = 2.0 ** -20 + (classes / 64 + 16) * E + 4 * E * finite_z
    finite_t = torch.where(there, t, 0.0).abs().amax(-1) if t.shape[-1] else finite_z * 0
    entry = lse_error + 2.0 ** -20 + 8 * E * (finite_z + finite_t) + indices.shape[-1] * E
    error = temperature ** 2 * (entry + torch.where(p > 0, p * (log_p - log_q).abs(), 0.0).sum(-1) * entry)
    d = torch.zeros(*logits.shape[:-1], classes, dtype=torch.float64, device="cuda").scatter_add(-1, at, -p)
    size = -d
    q = torch.where(some[..., None], (z - lse[..., None]).exp(), 0.0)
    return torch.where(some, each.sum(-1), 0.0) * temperature ** 2, lse, (d + q) * temperature, \
        torch.where(some, error, 0.0), lse_error, (q + size) * temperature * entry[..., None]


def _check(enc, logits, values, indices, temperature, grad=None):
    loss, lse = enc.distillation_loss(logits, values, indices, temperature=temperature)
    assert loss.dtype == lse.dtype == torch.float32 and loss.shape == lse.shape == logits.shape[:-1]
    want, want_lse, slope, error, lse_error, slope_error = _distil64(logits, values, indices, temperature)
    _near(loss, want, error, "loss")
    _near(lse, want_lse, lse_error, "lse")
    if grad is None:
        grad = torch.ones_like(loss)
    d = enc.distillation_gradient(grad, logits, want_lse.float(), values, indices, temperature=temperature)
    assert d.dtype == logits.dtype and d.shape == logits.shape
    g = grad.double()[..., None]
    _near(d, slope * g, slope_error * g.abs(), "gradient")
    return loss, lse, d


def _teacher(g, rows, classes, top, dtype, index_type, absent=0.1):
    teacher = _randn(g, rows, classes) * 3
    values, indices = teacher.topk(top, 1)
    indices = torch.where(torch.rand(rows, top, generator=g, device="cuda") < absent, -1, indices)
    indices = torch.where(torch.rand(rows, top, generator=g, device="cuda") < absent / 4, classes + 3, indices)
    if rows > 2:
        indices[1] = -1  # a row without entries
    return (0.5 * teacher + _randn(g, rows, classes)).to(dtype), values.to(dtype), indices.to(index_type)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,classes,top", [
    (1, 1, 1), (3, 2, 2), (64, 1000, 10), (5, 63, 63), (7, 65, 1), (1, 2048, 16), (33, 2049, 20), (2, 8191, 300), (9, 50001, 64),
    (1100, 4097, 8), (5000, 130, 5), (3, 262145, 1024), (1, 100003, 3), (1025, 30011, 32)])
def test_distillation(enc, rows, classes, top, dtype):
    g = _gen(rows + classes + top)
    index_type = torch.int32 if rows % 2 else torch.int64
    temperature = (1.0, 2.0, 0.5)[classes % 3]
    logits, values, indices = _teacher(g, rows, classes, top, dtype, index_type)
    grad = torch.rand(rows, generator=g, device="cuda") + 0.5
    loss, lse, d = _check(enc, logits, values, indices, temperature, grad)
    assert torch.equal(loss, enc.distillation_loss(logits, values, indices, temperature=temperature)[0])
    if rows > 2:
        assert loss[1] == 0 and (d[1] == 0).all()
    # values in binary32 beside logits of another type, and index types
    if dtype != torch.float32:
        _check(enc, logits, values.float() + 0.01, indices.long(), temperature, grad)


def test_distillation_entries(enc):
    """The same column twice and more, entries of -inf, the type's lowest value, rows
    of them alone, no entries at all, and logits of -inf."""
    g = _gen(2)
    for classes in (40, 5000):
        for dtype in TYPES:
            logits, values, indices = _teacher(g, 6, classes, 12, dtype, torch.int64, absent=0.0)
            indices[0] = indices[0, 3]
            indices[2, 4:9] = indices[2, 0]
            values[3, 2:] = -math.inf
            values[4] = -math.inf
            values[5, 1:] = torch.finfo(dtype).min
            loss, _, d = _check(enc, logits, values, indices, 1.5)
            assert loss[4] == 0 and (d[4] == 0).all()
            _check(enc, logits, values[:, :0], indices[:, :0], 1.0)
            values = torch.full_like(values, torch.finfo(dtype).min)
            _check(enc, logits, values, indices, 1.0)  # as likely as each other
            masked = logits.clone()
            masked[:, 7::3] = -math.inf
            keep = torch.where(indices % 3 == 1, 0, indices)  # the teacher names none of them
            _check(enc, masked, torch.zeros_like(values), keep, 1.0)
            masked[:, 7::3] = torch.finfo(dtype).min
            _check(enc, masked, torch.zeros_like(values), keep, 1.0)
            masked[2, 8] = -math.inf
            at = torch.full((6, 1), 8, device="cuda")
            loss, lse = enc.distillation_loss(masked, values[:, :1] * 0, at)
            assert loss[2] == math.inf
            d = enc.distillation_gradient(torch.ones(6, device="cuda"), masked, lse, values[:, :1] * 0, at)
            assert d[2, 8] == -1.0
            masked[3, 5] = math.nan
            loss, lse = enc.distillation_loss(masked, values[:, :1] * 0, at)
            assert torch.isnan(loss[3]) and torch.isfinite(loss[[0, 4, 5]]).all()


def test_distillation_strides_and_autograd(enc):
    g = _gen(6)
    logits, values, indices = _teacher(g, 30, 700, 9, torch.bfloat16, torch.int64)
    want, lse, d = _check(enc, logits, values, indices, 2.0)
    wide = torch.full((30, 705), math.nan, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:703] = logits
    wide_values, wide_indices = torch.zeros(30, 20, device="cuda"), torch.zeros(30, 20, device="cuda", dtype=torch.int32)
    wide_values[:, 5:14], wide_indices[:, 5:14] = values.float(), indices.int()
    args = wide[:, 3:703], wide_values[:, 5:14], wide_indices[:, 5:14]
    got = enc.distillation_loss(*args, temperature=2.0)
    assert torch.equal(got[0], want) and torch.equal(got[1], lse)
    ones = torch.ones((), device="cuda").expand(30)  # of a sum: one value for all rows
    exact_lse = (logits.double() / 2).logsumexp(1).float()
    assert torch.equal(enc.distillation_gradient(ones, args[0], exact_lse, *args[1:], temperature=2.0), d)
    shaped = logits.view(5, 6, 700).clone().requires_grad_()
    loss, _ = enc.distillation_loss(shaped, values.view(5, 6, 9), indices.view(5, 6, 9), temperature=2.0)
    assert torch.equal(loss.view(30), want)
    loss.sum().backward()
    assert torch.equal(shaped.grad.view(30, 700), enc.distillation_gradient(ones, logits, lse, values, indices, temperature=2.0))
    weights = torch.rand(5, 6, device="cuda")
    shaped.grad = None
    (enc.distillation_loss(shaped, values.view(5, 6, 9), indices.view(5, 6, 9))[0] * weights).sum().backward()
    lse1 = enc.distillation_loss(logits, values, indices)[1]
    assert torch.equal(shaped.grad.view(30, 700), enc.distillation_gradient(weights.view(30), logits, lse1, values, indices))
    empty = enc.distillation_loss(logits[:0], values[:0], indices[:0])
    assert empty[0].shape == (0,)
    assert enc.distillation_gradient(empty[0], logits[:0], empty[1], values[:0], indices[:0]).shape == (0, 700)
    one = enc.distillation_loss(logits[3], values[3], indices[3], temperature=2.0)
    assert one[0].shape == () and torch.equal(one[0], want[3])
    assert torch.equal(enc.distillation_gradient(torch.ones((), device="cuda"), logits[3], exact_lse[3], values[3], indices[3],
                                                 temperature=2.0), d[3])


def test_distillation_against_differences(enc):
    """The gradient along a direction against the 64-bit loss's difference quotient."""
    g = _gen(12)
    logits, values, indices = _teacher(g, 20, 300, 6, torch.float32, torch.int64)
    lse = enc.distillation_loss(logits, values, indices, temperature=1.7)[1]
    d = enc.distillation_gradient(torch.ones(20, device="cuda"), logits, lse, values, indices, temperature=1.7).double()
    v = torch.randn(20, 300, generator=g, device="cuda", dtype=torch.float64)
    moved = [_distil64(logits.double() + s * 1e-5 * v, values, indices, 1.7)[0].sum() for s in (1, -1)]
    want = (moved[0] - moved[1]) / 2e-5
    assert abs((d * v).sum() - want) <= 2e-5 * (d.abs() * v.abs()).sum() + 1e-6


def test_distillation_captured(enc):
    """A step captured and replayed; a row's parts join through the workspace."""
    g = _gen(14)
    logits, values, indices = _teacher(g, 4, 60000, 10, torch.float16, torch.int32)
    grad = torch.ones(4, device="cuda")

    def work():
        loss, lse = enc.distillation_loss(logits, values, indices)
        return loss, lse, enc.distillation_gradient(grad, logits, lse, values, indices)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for seed in range(4):
        logits.copy_(_teacher(_gen(50 + seed), 4, 60000, 10, torch.float16, torch.int32)[0])
        want = work()
        for out in captured:
            out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), seed


def test_distillation_rows_beyond_4_gb(enc):
    rows, classes = 70_000, 32_768
    g = _gen(16)
    logits = torch.empty(rows, classes, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    indices = torch.randint(0, classes, (rows, 4), generator=g, device="cuda")
    values = torch.randn(rows, 4, generator=g, device="cuda")
    loss, lse = enc.distillation_loss(logits, values, indices)
    d = enc.distillation_gradient(torch.ones(rows, device="cuda"), logits, lse, values, indices)
    for part in (slice(0, 50), slice(65_500, 65_560), slice(rows - 50, rows)):
        want, want_lse, slope, error, lse_error, slope_error = _distil64(logits[part], values[part], indices[part], 1.0)
        _near(loss[part], want, error)
        _near(lse[part], want_lse, lse_error)
        _near(d[part], slope, slope_error + (slope.abs() + slope_error) * lse_error[:, None] * 4)
