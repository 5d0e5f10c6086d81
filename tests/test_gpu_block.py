"""The gated feed-forward block (xgboost.encoder) against plain 64-bit forms.

Tolerances, element by element.  A sum of n binary32 terms is off by at most
n 2^-23 of the terms' absolute sum, whatever the order (2^-24 a rounding; the
matrix instructions may cut instead of rounding, hence twice that).  Float32
operands are three bfloat16 each: six products a value, and what is left out or
rounded away is below 4 2^-24 of it.  The inner matrices are rounded to the type
once, u of their value (2^-24 for float32, whose three parts hold 24 bits).
Errors of factors go through the formulas to first order, with the activation's
slope at most 1.13 and its slope's slope at most 1; activations are off by
(|g| + 4) 2^-23 of themselves, gelu of 16-bit results by 8e-6 more.
"""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = ["f32", "f16", "bf16"]
E = 2.0 ** -23


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _near(got, want, slack, what=""):
    dtype = got.dtype
    bound = slack + (want.abs() + slack) * U[dtype] + TINY[dtype]
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound"


def _terms(n, dtype):
    """What a product over n is off by, of its absolute sum."""
    return (6 * n + 12) * E if dtype == torch.float32 else (n + 2) * E


def _act(g, activation):
    if activation == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * torch.sigmoid(-g))
    phi = 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
    return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def _act_error(g, activation, dtype):
    """Of act(g) and of its slope."""
    near = (g.abs() + 4) * E
    extra = 8e-6 if activation == "gelu" and dtype != torch.float32 else 1e-6 if activation == "gelu" else 0.0
    a, s = _act(g, activation)
    return a.abs() * near + g.abs() * extra, (s.abs() + 1) * near + extra


def _inner64(x, gate, up, dtype):
    """gate and up's products and what they are off by."""
    x, n = x.double(), _terms(x.shape[-1], dtype)
    return [(x @ w.double().t(), (x.abs() @ w.double().t().abs()) * n) for w in (gate, up)]


def _forward64(x, gate, up, down, activation):
    dtype = x.dtype
    (g, eg), (u, eu) = _inner64(x, gate, up, dtype)
    a, _ = _act(g, activation)
    ea = 1.13 * eg + _act_error(g, activation, dtype)[0]
    h = a * u
    eh = ea * u.abs() + (a.abs() + ea) * eu
    eh = eh + (h.abs() + eh) * (U[dtype] + E) + TINY[dtype]
    w = down.double()
    return h @ w.t(), eh @ w.t().abs() + ((h.abs() + eh) @ w.t().abs()) * _terms(w.shape[1], dtype)


def _gradient64(grad, x, kept, gate, up, down, activation):
    dtype = x.dtype
    dy, x64, n = grad.double(), x.double(), _terms
    g, u = kept[:, 0].double(), kept[:, 1].double()
    wg, wu, wd = gate.double(), up.double(), down.double()
    a, s = _act(g, activation)
    ea, es = _act_error(g, activation, dtype)
    dh = dy @ wd
    edh = (dy.abs() @ wd.abs()) * n(wd.shape[0], dtype)
    tiny = TINY[dtype]

    def rounded(value, error):
        return error + (value.abs() + error) * (U[dtype] + 2 * E) + tiny

    h, eh = a * u, rounded(a * u, ea * u.abs())
    dg, edg = dh * u * s, rounded(dh * u * s, edh * (u * s).abs() + (dh.abs() + edh) * u.abs() * es)
    du, edu = dh * a, rounded(dh * a, edh * a.abs() + (dh.abs() + edh) * ea)
    rows, hidden = x.shape[0], wg.shape[0]
    dx = dg @ wg + du @ wu
    edx = edg @ wg.abs() + edu @ wu.abs() + ((dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs()) * n(2 * hidden, dtype)

    def weight(d, ed, b):
        return d.t() @ b, ed.t() @ b.abs() + ((d.abs() + ed).t() @ b.abs()) * n(rows, dtype)

    dd = dy.t() @ h, dy.t().abs() @ eh + (dy.t().abs() @ (h.abs() + eh)) * n(rows, dtype)
    return (dx, edx), weight(dg, edg, x64), weight(du, edu, x64), dd


def _case(g, rows, dim, hidden, dtype):
    x = _randn(g, rows, dim, dtype=dtype)
    gate, up = (_randn(g, hidden, dim, dtype=dtype, scale=dim ** -0.5) for _ in range(2))
    return x, gate, up, _randn(g, dim, hidden, dtype=dtype, scale=hidden ** -0.5), _randn(g, rows, dim, dtype=dtype)


SIZES = [
    # rows, dim, hidden: single rows and values, odd ones, tiles' edges of every size, shares of the depth
    (1, 1, 1), (1, 8, 8), (2, 1, 5), (3, 7, 9), (1, 1024, 2048), (16, 64, 256), (17, 65, 33), (32, 128, 64), (33, 24, 520),
    (64, 64, 64), (65, 72, 136), (127, 200, 255), (130, 257, 129), (255, 320, 96), (300, 96, 777), (513, 40, 1000),
    (1000, 333, 500), (2049, 512, 264), (4100, 24, 40), (20011, 16, 8), (700, 1000, 1501), (1500, 2048, 1032), (6000, 512, 2056),
]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows,dim,hidden", SIZES)
def test_block_and_gradient(enc, rows, dim, hidden, dtype):
    g = _gen(rows * 7 + dim * 3 + hidden)
    activation = "gelu" if (rows + hidden) % 2 else "silu"
    x, gate, up, down, grad = _case(g, rows, dim, hidden, dtype)
    y = enc.feed_forward(x, gate, up, down, activation=activation)
    assert y.shape == x.shape and y.dtype == dtype
    _near(y, *_forward64(x, gate, up, down, activation), "y")
    again, kept = enc.feed_forward(x, gate, up, down, activation=activation, keep=True)
    assert kept.shape == (rows, 2, hidden) and kept.dtype == torch.float32
    _near(again, *_forward64(x, gate, up, down, activation), "y, kept")
    for k, (want, error) in enumerate(_inner64(x, gate, up, dtype)):
        _near(kept[:, k], want, error, "kept")
    got = enc.feed_forward_gradient(grad, x, kept, gate, up, down, activation=activation)
    names = ("dx", "dgate", "dup", "ddown")
    for name, out, like, (want, error) in zip(names, got, (x, gate, up, down),
                                              _gradient64(grad, x, kept, gate, up, down, activation)):
        assert out.shape == like.shape and out.dtype == dtype
        _near(out, want, error, name)
    for out, again in zip(got, enc.feed_forward_gradient(grad, x, kept, gate, up, down, activation=activation)):
        assert torch.equal(out, again)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_formula_against_differences(enc, activation):
    """The gradients' sum along a direction against the 64-bit forward pass's
    difference quotient: cut off at 1e-10 of the third derivative, rounded to 1e-11."""
    g = _gen(5)
    x, gate, up, down, grad = _case(g, 37, 24, 56, torch.float32)
    got = enc.feed_forward_gradient(grad, x, enc.feed_forward(x, gate, up, down, activation=activation, keep=True)[1], gate, up,
                                    down, activation=activation)

    def loss(values):
        x, gate, up, down = values
        return ((_act(x @ gate.t(), activation)[0] * (x @ up.t())) @ down.t() * grad.double()).sum()

    point = [t.double() for t in (x, gate, up, down)]
    for k, out in enumerate(got):
        v = torch.randn(out.shape, generator=g, device="cuda", dtype=torch.float64)
        moved = [[t + s * 1e-5 * v if j == k else t for j, t in enumerate(point)] for s in (1, -1)]
        want = (loss(moved[0]) - loss(moved[1])) / 2e-5
        size = (out.double().abs() * v.abs()).sum()
        assert abs((out.double() * v).sum() - want) <= 2e-5 * size + 1e-6


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_values_where_activations_end(enc, dtype):
    """Gates far from zero on both sides, zeros, and rows of zeros."""
    gate_values = torch.tensor([0.0, -0.0, 1e-6, -1e-6, 0.5, -0.5, 3.0, -3.0, 8.0, -8.0, 20.0, -20.0, 60.0, -60.0, 200.0, -200.0],
                               device="cuda", dtype=dtype)
    dim = len(gate_values)
    x = torch.eye(dim, device="cuda", dtype=dtype)
    x[-1] = 0
    gate, up = gate_values[:, None].expand(dim, dim).contiguous(), torch.ones(dim, dim, device="cuda", dtype=dtype)
    down = torch.eye(dim, device="cuda", dtype=dtype)
    for activation in ("silu", "gelu"):
        y, kept = enc.feed_forward(x, gate, up, down, activation=activation, keep=True)
        _near(y, *_forward64(x, gate, up, down, activation), activation)
        assert (y[-1] == 0).all()
        got = enc.feed_forward_gradient(torch.ones_like(x), x, kept, gate, up, down, activation=activation)
        for out, (want, error) in zip(got, _gradient64(torch.ones_like(x), x, kept, gate, up, down, activation)):
            _near(out, want, error, activation)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_strides_and_shapes(enc, dtype):
    g = _gen(11)
    rows, dim, hidden = 70, 48, 88
    x, gate, up, down, grad = _case(g, rows, dim, hidden, dtype)
    want, kept = enc.feed_forward(x, gate, up, down, keep=True)
    want_gradient = enc.feed_forward_gradient(grad, x, kept, gate, up, down)

    def inside(t, before, after):  # a view with other values around
        wide = torch.full((t.shape[0] + 2, t.shape[1] + before + after), float("nan"), device="cuda", dtype=dtype)
        view = wide[1:-1, before:before + t.shape[1]]
        view.copy_(t)
        return view

    for before, after in ((8, 8), (3, 2), (0, 16), (1, 0)):
        views = [inside(t, before, after) for t in (x, gate, up, down)]
        assert torch.equal(enc.feed_forward(*views), want)
        got = enc.feed_forward_gradient(inside(grad, before, after), views[0], kept, *views[1:])
        assert all(torch.equal(a, b) for a, b in zip(got, want_gradient))
    # gate and up of one matrix, rows in turn, and at unlike distances
    both = torch.stack([gate, up], 1).reshape(2 * hidden, dim)
    assert torch.equal(enc.feed_forward(x, both[::2], both[1::2], down), want)
    assert torch.equal(enc.feed_forward(x, both[::2], up, down), want)
    assert all(torch.equal(a, b) for a, b in zip(enc.feed_forward_gradient(grad, x, kept, both[::2], up, down), want_gradient))
    # transposed storage, more axes, one axis, broadcast rows
    assert torch.equal(enc.feed_forward(x.t().contiguous().t(), gate, up, down.t().contiguous().t()), want)
    y, k = enc.feed_forward(x.view(7, 10, dim), gate, up, down, keep=True)
    assert torch.equal(y.view(rows, dim), want) and k.shape == (7, 10, 2, hidden)
    got = enc.feed_forward_gradient(grad.view(7, 10, dim), x.view(7, 10, dim), k, gate, up, down)
    assert got[0].shape == (7, 10, dim) and all(torch.equal(a.view(b.shape), b) for a, b in zip(got, want_gradient))
    y, k = enc.feed_forward(x[5], gate, up, down, keep=True)
    assert y.shape == (dim,) and k.shape == (2, hidden)
    _near(y[None], *_forward64(x[5:6], gate, up, down, "silu"))
    same = x[:1].expand(rows, dim)
    assert torch.equal(enc.feed_forward(same, gate, up, down), enc.feed_forward(same.contiguous(), gate, up, down))
    ones = torch.ones((), device="cuda", dtype=dtype).expand(rows, dim)
    got = enc.feed_forward_gradient(ones, same, kept, gate, up, down)
    for a, b in zip(got, enc.feed_forward_gradient(ones.contiguous(), same.contiguous(), kept, gate, up, down)):
        assert torch.equal(a, b)
    kept_wide = torch.zeros(rows, 2, hidden + 3, device="cuda")[:, :, :hidden].copy_(kept)
    assert all(torch.equal(a, b) for a, b in zip(enc.feed_forward_gradient(grad, x, kept_wide, gate, up, down), want_gradient))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_no_rows(enc, dtype):
    g = _gen(3)
    x, gate, up, down, grad = _case(g, 5, 12, 20, dtype)
    y, kept = enc.feed_forward(x[:0], gate, up, down, keep=True)
    assert y.shape == (0, 12) and kept.shape == (0, 2, 20)
    dx, *matrices = enc.feed_forward_gradient(grad[:0], x[:0], kept, gate, up, down)
    assert dx.shape == (0, 12)
    for out, like in zip(matrices, (gate, up, down)):
        assert out.shape == like.shape and (out == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("dim,hidden", [(24, 40), (23, 41)])
def test_a_row_with_nan_is_alone(enc, dim, hidden, dtype):
    """What one row holds reaches no other row of y and dx."""
    g = _gen(dim)
    x, gate, up, down, grad = _case(g, 150, dim, hidden, dtype)
    want, kept = enc.feed_forward(x, gate, up, down, keep=True)
    want_dx = enc.feed_forward_gradient(grad, x, kept, gate, up, down)[0]
    others = torch.arange(150, device="cuda") != 77
    for bad in (float("nan"), float("inf"), -float("inf")):
        x2, grad2 = x.clone(), grad.clone()
        x2[77, 3], grad2[77, 5] = bad, bad
        y, kept2 = enc.feed_forward(x2, gate, up, down, keep=True)
        assert torch.equal(y[others], want[others]) and not torch.isfinite(y[77]).all()
        dx = enc.feed_forward_gradient(grad2, x, kept, gate, up, down)[0]
        assert torch.equal(dx[others], want_dx[others]) and not torch.isfinite(dx[77]).all()
        dx = enc.feed_forward_gradient(grad, x2, kept2, gate, up, down)[0]
        assert torch.equal(dx[others], want_dx[others])
    # NaN in a matrix' row reaches the hidden value it makes, and through it all of y.
    gate2 = gate.clone()
    gate2[hidden - 1] = float("nan")
    _, kept2 = enc.feed_forward(x, gate2, up, down, keep=True)
    assert torch.equal(kept2[:, 0, :-1], kept[:, 0, :-1]) and torch.isnan(kept2[:, 0, -1]).all()
    assert torch.equal(kept2[:, 1], kept[:, 1])


def test_binary32_range(enc):
    """Values near both ends of binary32, whose parts bfloat16 has to hold."""
    big = torch.tensor([[3.402823e38, -3.39e38, 1e-30, 2e38]], device="cuda")
    gate = torch.zeros(8, 4, device="cuda")
    gate[0, 0], gate[1, 1], gate[2, 2], gate[3, 3] = 1e-38, 1e-38, 1e30, -1e-38
    up = torch.zeros(8, 4, device="cuda")
    up[:, 2] = 1e30
    _, kept = enc.feed_forward(big, gate, up, torch.ones(4, 8, device="cuda"), keep=True)
    want = big.double() @ gate.double().t()
    assert torch.isfinite(kept).all()
    # bfloat16's last step is 2^-133, so the parts of a value end there: 1e-38, of which
    # binary32 has 2^-149 steps itself, is off by up to 2^-134, here times 3.4e38.
    parts = big.double().abs() @ (gate != 0).double().t() * 2.0 ** -134
    assert ((kept[0, 0].double() - want[0]).abs() <= want[0].abs() * 2.0 ** -20 + parts).all()
    assert ((kept[0, 1].double() - 1.0).abs() <= 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_modules_and_autograd(enc, dtype):
    """The module, leaf gradients, those that are not wanted, two calls' sum, a
    broadcast gradient and one of nothing."""
    torch.manual_seed(2)
    block = enc.FeedForward(40, 72, activation="gelu", dtype=dtype)
    x = torch.randn(9, 11, 40, device="cuda").to(dtype).requires_grad_()
    block(x).sum().backward()
    ones = torch.ones_like(x)
    kept = enc.feed_forward(x.detach(), block.gate.detach(), block.up.detach(), block.down.detach(), activation="gelu", keep=True)[1]
    want = enc.feed_forward_gradient(ones, x.detach(), kept, block.gate.detach(), block.up.detach(), block.down.detach(),
                                     activation="gelu")
    leaves = (x, block.gate, block.up, block.down)
    for leaf, w in zip(leaves, want):
        assert torch.equal(leaf.grad, w)
    assert torch.equal(block(x).detach(), enc.feed_forward(x.detach(), *(p.detach() for p in leaves[1:]), activation="gelu"))
    for k in range(4):  # one wanted at a time
        args = [t.detach().clone().requires_grad_(j == k) for j, t in enumerate(leaves)]
        enc.feed_forward(*args, activation="gelu").sum().backward()
        assert torch.equal(args[k].grad, want[k]) and all(a.grad is None for j, a in enumerate(args) if j != k)
    y, kept = enc.feed_forward(x, *leaves[1:], keep=True)
    assert y.requires_grad and not kept.requires_grad
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.float().square().sum(), x, create_graph=True)[0].float().sum().backward()


def test_served_and_trained_together(enc):
    """Leaves to vectors, norm, block, a teacher's logits, optimizer steps, and the
    block in 8 bits."""
    torch.manual_seed(4)
    leaves, norm = enc.Embedding(300, 64, pool=True), enc.LayerNorm(64)
    block, head = enc.FeedForward(64, 128), torch.nn.Linear(64, 50, device="cuda")
    tokens = torch.randint(0, 300, (200, 12), device="cuda", dtype=torch.int32)
    values, indices = torch.randn(200, 50, device="cuda").topk(5)
    muon = enc.Muon([block.gate, block.up, block.down], lr=0.01)

    def loss():
        return enc.distillation_loss(head(block(norm(leaves(tokens)))), values, indices, temperature=2.0)[0].mean()

    first = loss()
    first.backward()
    parameters = [*leaves.parameters(), *norm.parameters(), *block.parameters(), *head.parameters()]
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and (p.grad != 0).any() for p in parameters)
    # Along the gradient by a small step the loss falls by step |gradient|^2, to second order.
    with torch.no_grad():
        square = sum(p.grad.double().square().sum() for p in parameters).item()
        before = [p.detach().clone() for p in parameters]
        step = 1e-3 / math.sqrt(square)
        for p in parameters:
            p -= step * p.grad
        fall = (first - loss()).item()
        for p, b in zip(parameters, before):
            p.copy_(b)
    assert abs(fall / (step * square) - 1.0) < 0.05
    muon.step()
    x = norm(leaves(tokens)).detach()
    served, plain = block.quantized()(x), block(x).detach()
    # e4m3 rounds by 2^-4 at most, three factors of a sum of independent terms: below 3 2^-4 of the norm.
    assert (served - plain).norm() < 3 * 2.0 ** -4 * plain.norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_captured_and_replayed(enc, dtype):
    """A graph of a training step and a served call, replayed between eager work."""
    g = _gen(8)
    x, gate, up, down, grad = _case(g, 200, 72, 136, dtype)
    matrices = [enc.quantize_blocks(w) for w in (gate, up, down)]

    def work():
        y, kept = enc.feed_forward(x, gate, up, down, keep=True)
        return (y, *enc.feed_forward_gradient(grad, x, kept, gate, up, down), enc.block_feed_forward(x, *matrices))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for seed in range(4):
        fresh = _case(_gen(100 + seed), 200, 72, 136, dtype)
        x.copy_(fresh[0])
        grad.copy_(fresh[4])
        want = work()
        for out in captured:
            out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b), seed


def test_on_other_streams(enc):
    """Calls run on the current stream: two at once, each behind its own slow work."""
    g = _gen(21)
    cases = [_case(g, 500, 256, 512, torch.bfloat16) for _ in range(2)]
    want = [enc.feed_forward(*c[:4]) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    busy = torch.randn(2048, 2048, device="cuda")
    out, late = [None, None], [None, None]
    torch.cuda.synchronize()
    for _ in range(3):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                slow = busy
                for _ in range(4):
                    slow = slow @ busy * 1e-2
                late[k] = cases[k][0] + (slow[0, 0] * 0).to(torch.bfloat16)
                out[k] = enc.feed_forward(late[k], *cases[k][1:4])
    torch.cuda.synchronize()
    for a, b in zip(out, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [0, 2], ids=["f32", "bf16"])
def test_nothing_is_written_around_results(enc, dtype):
    """The C entries with results inside larger buffers, which keep what they held."""
    from test_arguments_block import Forward, Gradient, P
    import xgboost.core as core
    lib = ctypes.CDLL(core._LIB.path)
    kind = torch.float32 if dtype == 0 else torch.bfloat16
    for name in ("feed_forward", "feed_forward_gradient"):
        getattr(lib, f"mgb_{name}_workspace_bytes").restype = ctypes.c_size_t
    for rows, dim, hidden in ((1, 5, 3), (67, 33, 129), (130, 64, 72)):
        x, gate, up, down, grad = _case(_gen(rows), rows, dim, hidden, kind)
        want, want_kept = enc.feed_forward(x, gate, up, down, keep=True)
        want_gradient = enc.feed_forward_gradient(grad, x, want_kept, gate, up, down)

        def framed(like):
            room = torch.full((like.numel() + 512,), 7.0, device="cuda", dtype=like.dtype)
            return room, room.data_ptr() + 256 * room.element_size()

        def unframed(room, like, what):
            assert torch.equal(room[256:256 + like.numel()].view(like.shape), like), what
            assert (room[:256] == 7).all() and (room[256 + like.numel():] == 7).all(), what

        stream = P(torch.cuda.current_stream().cuda_stream)
        y, kept = framed(want), framed(want_kept)
        p = Forward(y[1], kept[1], x.data_ptr(), gate.data_ptr(), up.data_ptr(), down.data_ptr(), rows, dim, hidden, dim, dim, dim,
                    hidden, 0, dtype)
        need = lib.mgb_feed_forward_workspace_bytes(ctypes.byref(p))
        space = torch.full((need + 4096,), 7, device="cuda", dtype=torch.uint8)
        assert space.data_ptr() % 256 == 0
        assert lib.mgb_feed_forward(ctypes.byref(p), P(space.data_ptr()), ctypes.c_size_t(need), stream) == 0
        torch.cuda.synchronize()
        unframed(y[0], want, "y")
        unframed(kept[0], want_kept, "kept")
        assert (space[need:] == 7).all()
        rooms = [framed(w) for w in want_gradient]
        q = Gradient(*(r[1] for r in rooms), grad.data_ptr(), x.data_ptr(), want_kept.data_ptr(), gate.data_ptr(), up.data_ptr(),
                     down.data_ptr(), rows, dim, hidden, dim, dim, dim, dim, hidden, 0, dtype)
        need = lib.mgb_feed_forward_gradient_workspace_bytes(ctypes.byref(q))
        space = torch.full((need + 4096,), 7, device="cuda", dtype=torch.uint8)
        assert lib.mgb_feed_forward_gradient(ctypes.byref(q), P(space.data_ptr()), ctypes.c_size_t(need), stream) == 0
        torch.cuda.synchronize()
        for (room, _), w in zip(rooms, want_gradient):
            unframed(room, w, "gradient")
        assert (space[need:] == 7).all()


def test_rows_beyond_4_gb(enc):
    """1.1 million rows of 2,048: the last ones lie more than 4 GB from the first."""
    rows, dim, hidden = 1_100_000, 2048, 16
    g = _gen(31)
    gate, up = (_randn(g, hidden, dim, dtype=torch.bfloat16, scale=dim ** -0.5) for _ in range(2))
    down = _randn(g, dim, hidden, dtype=torch.bfloat16, scale=0.25)
    x = torch.empty(rows, dim, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    y, kept = enc.feed_forward(x, gate, up, down, keep=True)
    for part in (slice(0, 300), slice(1_048_500, 1_048_700), slice(rows - 300, rows)):
        _near(y[part], *_forward64(x[part], gate, up, down, "silu"), "y")
    del y
    dx, dgate, _, ddown = enc.feed_forward_gradient(x, x, kept, gate, up, down)
    for part in (slice(0, 100), slice(rows - 100, rows)):
        want, error = _gradient64(x[part], x[part], kept[part], gate, up, down, "silu")[0]
        _near(dx[part], want, error, "dx")
    want = [torch.zeros(hidden, dim, device="cuda", dtype=torch.float64), torch.zeros(dim, hidden, device="cuda", dtype=torch.float64)]
    error = [torch.zeros_like(w) for w in want]
    for begin in range(0, rows, 50_000):
        part = slice(begin, begin + 50_000)
        _, (dg, edg), _, (dd, edd) = _gradient64(x[part], x[part], kept[part], gate, up, down, "silu")
        # (a part's sums stand for 50,000 terms of 1.1 million: 22 times their roundings)
        for k, (value, off) in enumerate(((dg, edg), (dd, edd))):
            want[k] += value
            error[k] += 22 * off
    _near(dgate, want[0], error[0], "dgate")
    _near(ddown, want[1], error[1], "ddown")
