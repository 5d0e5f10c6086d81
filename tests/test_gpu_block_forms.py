"""The feed-forward block, its 8-bit form and distillation where their forms meet:
rows that go in slices, whole or as tiles, rows of more than one workgroup's scales,
scales at their ends, captured training, and the example that runs them together.
Tolerances are those of test_gpu_block.py and test_gpu_block8.py."""
import importlib.util
from pathlib import Path

import pytest
import torch

from test_gpu_block import E, NAMES, TYPES, _act, _case, _forward64, _gen, _gradient64, _inner64, _near, _randn
from test_gpu_block8 import _blocks64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("dim,hidden", [(37, 61), (130, 777), (1000, 300), (2056, 40), (8200, 24), (24, 8200), (64, 4112)])
def test_few_rows(enc, dim, hidden, dtype):
    """Every number of rows at which the few rows' form changes, on both sides of it."""
    g = _gen(dim + hidden)
    x, gate, up, down, _ = _case(g, 33, dim, hidden, dtype)
    wide = torch.full((33, dim + 3), float("nan"), device="cuda", dtype=dtype)
    wide[:, 2:2 + dim] = x
    for rows in (1, 2, 4, 5, 8, 9, 16, 17, 32, 33):
        y, kept = enc.feed_forward(x[:rows], gate, up, down, keep=True)
        _near(y, *_forward64(x[:rows], gate, up, down, "silu"), f"{rows} rows")
        for k, (want, error) in enumerate(_inner64(x[:rows], gate, up, dtype)):
            _near(kept[:, k], want, error, f"{rows} rows, kept")
        assert torch.equal(enc.feed_forward(wide[:rows, 2:2 + dim], gate, up, down), y), rows
        assert torch.equal(enc.feed_forward(x[:1].expand(rows, dim), gate, up, down),
                           enc.feed_forward(x[:1].repeat(rows, 1), gate, up, down)), rows


@pytest.mark.parametrize("dtype", TYPES[1:], ids=NAMES[1:])
@pytest.mark.parametrize("rows,dim,hidden", [(1, 16, 64), (3, 200, 500), (31, 250, 333), (40, 24, 700), (33, 248, 1000), (500, 16, 3000),
                                             (5000, 8, 40)])
def test_few_results_are_rounded_once(enc, rows, dim, hidden, dtype, monkeypatch):
    """Up to 8,192 of them: inner values count as two of the type, off by u^2, and their
    products are twice as many terms."""
    import test_gpu_block
    g = _gen(rows + dim + hidden)
    x, gate, up, down, grad = _case(g, rows, dim, hidden, dtype)
    y, kept = enc.feed_forward(x, gate, up, down, keep=True)
    got = (y, *enc.feed_forward_gradient(grad, x, kept, gate, up, down))
    with monkeypatch.context() as m:
        m.setattr(test_gpu_block, "U", {t: u * u for t, u in test_gpu_block.U.items()})
        wants = (_forward64(x, gate, up, down, "silu"), *_gradient64(grad, x, kept, gate, up, down, "silu"))
    for name, out, (want, error) in zip(("y", "dx", "dgate", "dup", "ddown"), got, wants):
        few = rows * dim if name == "y" else min(rows, hidden) * dim
        if few <= 8192:
            _near(out, want, 2 * error, name)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("dim,out", [(100, 61), (700, 300), (2100, 40), (8400, 24), (300, 4112)])
def test_few_rows_of_blocks(enc, dim, out, dtype):
    g = _gen(dim + out)
    x, w = enc.quantize_blocks(_randn(g, 33, dim)), enc.quantize_blocks(_randn(g, out, dim))
    a, b = x.dequantize().double(), w.dequantize().double()
    size = a.abs() @ b.t().abs()
    slack = size * ((dim + 2) * E if dtype == torch.float32 else 2.0 ** -12 + dim * E)
    for rows in (1, 4, 5, 8, 9, 16, 17, 32, 33):
        part = enc.BlockScaled(x.values[:rows], x.scales[:rows], dim)
        _near(enc.block_matmul(part, w, dtype=dtype), (a @ b.t())[:rows], slack[:rows], f"{rows} rows")


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("rows", [1, 5, 12, 30, 50])
def test_rows_beyond_a_workgroups_scales(enc, rows, dtype):
    """More than 64 blocks a row: whole numbers that all roundings keep.  One hidden value
    a block of 128 is not zero, and it is a product of whole numbers below 16."""
    dim, hidden = 8192 + 384, 8192 + 200
    x = torch.zeros(rows, dim, device="cuda", dtype=dtype)
    at = torch.arange(rows, device="cuda") * 171 % dim
    x[torch.arange(rows), at] = 1.0
    gate, up = torch.zeros(hidden, dim, device="cuda"), torch.zeros(hidden, dim, device="cuda")
    some = torch.arange(0, hidden, 128, device="cuda")
    gate[some] = 64.0  # silu(64) is 64 in binary32
    up[some] = (torch.arange(dim, device="cuda") % 3 + 1).float()
    g = _gen(rows)
    down = torch.randint(-2, 3, (dim, hidden), generator=g, device="cuda").float()
    got = enc.block_feed_forward(x, *(enc.quantize_blocks(w) for w in (gate, up, down)))
    h = torch.zeros(rows, hidden, device="cuda", dtype=torch.float64)
    h[:, some] = 64.0 * up[0][at].double()[:, None]
    want = h @ down.double().t()
    # float16 and bfloat16 round the sum, a whole number of 64s, once.
    _near(got, want, want.abs() * 2.0 ** -16 if dtype == torch.bfloat16 else want * 0)


@pytest.mark.parametrize("rows,dim,hidden", [(40, 256, 512), (130, 200, 777), (300, 512, 1024)])
def test_served_few_hidden_values(enc, rows, dim, hidden):
    """Bfloat16 rows of up to 2 million hidden values are served as the 64-bit form
    rounds, but for values that lie next to a border to its last bits: the result is off
    by its own rounding, u / sqrt(3) of its norm, and at most a tenth of that."""
    g = _gen(rows)
    x = _randn(g, rows, dim, dtype=torch.bfloat16)
    gate, up = (enc.quantize_blocks(_randn(g, hidden, dim, scale=dim ** -0.5)) for _ in range(2))
    down = enc.quantize_blocks(_randn(g, dim, hidden, scale=hidden ** -0.5))
    v = enc.quantize_blocks(x).dequantize().double()
    h = _act(v @ gate.dequantize().double().t(), "silu")[0] * (v @ up.dequantize().double().t())
    values, exponent = _blocks64(h)
    kept = (values.view(rows, -1, 128) * torch.exp2(exponent)[..., None]).flatten(1)[:, :hidden]
    want = kept @ down.dequantize().double().t()
    got = enc.block_feed_forward(x, gate, up, down)
    rounding = (want.bfloat16().double() - want).norm()
    assert (got.double() - want).norm() <= 1.1 * rounding


def test_scales_at_their_ends(enc):
    """Scale 255 stands for NaN in every form, scale 0 for 2^-127."""
    g = _gen(17)
    w = enc.quantize_blocks(_randn(g, 70, 256))
    for rows in (3, 6, 12, 20, 40):
        x = enc.quantize_blocks(_randn(g, rows, 256))
        want = [enc.block_matmul(x, w, dtype=t) for t in TYPES]
        scales = x.scales.view(torch.uint8).clone()
        scales[1, 0] = 255
        bad = enc.BlockScaled(x.values, scales.view(torch.float8_e8m0fnu), 256)
        assert torch.isnan(bad.dequantize()[1, :128]).all() and torch.isfinite(bad.dequantize()[1, 128:]).all()
        others = torch.arange(rows, device="cuda") != 1
        for t, sound in zip(TYPES, want):
            got = enc.block_matmul(bad, w, dtype=t)
            assert torch.isnan(got[1]).all() and torch.equal(got[others], sound[others])
        scales[1] = 0
        tiny = enc.BlockScaled(x.values, scales.view(torch.float8_e8m0fnu), 256)
        big = w.scales.view(torch.uint8) + 100
        grown = enc.BlockScaled(w.values, big.view(torch.float8_e8m0fnu), 256)
        a, b = tiny.values.double(), grown.dequantize().double()
        sizes = torch.exp2(scales.double() - 127).repeat_interleave(128, 1)
        got = enc.block_matmul(tiny, grown, dtype=torch.float32)[1]
        exact = ((a * sizes)[1:2] @ b.t())[0]
        # bfloat16's steps end at 2^-133: half of one for each value of x.
        slack = b.abs().sum(1) * 2.0 ** -134 + ((a * sizes)[1:2].abs() @ b.t().abs())[0] * 258 * E
        _near(got, exact, slack)


@pytest.mark.parametrize("rows,dim,hidden", [(700, 296, 1000), (1500, 520, 1304), (300, 1032, 2050), (4096, 130, 260)])
def test_binary32_in_tiles(enc, rows, dim, hidden):
    """Sizes between the ones where one tile size serves all products."""
    g = _gen(rows + hidden)
    x, gate, up, down, grad = _case(g, rows, dim, hidden, torch.float32)
    y, kept = enc.feed_forward(x, gate, up, down, activation="gelu", keep=True)
    _near(y, *_forward64(x, gate, up, down, "gelu"), "y")
    got = enc.feed_forward_gradient(grad, x, kept, gate, up, down, activation="gelu")
    for name, out, (want, error) in zip(("dx", "dgate", "dup", "ddown"), got, _gradient64(grad, x, kept, gate, up, down, "gelu")):
        _near(out, want, error, name)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_training_captured(enc, dtype):
    """Forward and backward passes of the modules in one graph, whose leaves no eager graph
    holds then; replays give the eager passes' gradients."""
    torch.manual_seed(3)
    block = enc.FeedForward(72, 136, dtype=dtype)
    x = torch.randn(150, 72, device="cuda").to(dtype)
    values, indices = torch.randn(150, 72, device="cuda").topk(6)
    leaves = [block.gate, block.up, block.down]

    def step():
        loss = enc.distillation_loss(block(x), values, indices, temperature=1.5)[0].sum()
        return loss.detach(), torch.autograd.grad(loss, leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    for seed in range(3):
        x.copy_(_randn(_gen(70 + seed), 150, 72, dtype=dtype))
        want_loss, want = step()
        for out in (loss, *grads):
            out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want_loss)
        assert all(torch.equal(a, b) for a, b in zip(grads, want)), seed


def test_capture_while_an_eager_graph_lives(enc):
    """Refused where the leaves' gradients would be added up on the default stream; once
    the eager results are gone, or were made on another stream, it is captured."""
    block = enc.FeedForward(24, 40)
    x = torch.randn(50, 24, device="cuda")
    leaves = list(block.parameters())
    values, indices = torch.randn(50, 40, device="cuda").topk(4)
    logits = torch.randn(50, 40, device="cuda", requires_grad=True)

    def refused(work):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="default stream"):
            with torch.cuda.graph(graph):
                work()

    y = block(x)
    refused(lambda: block(x))
    loss = enc.distillation_loss(logits, values, indices)[0]
    refused(lambda: enc.distillation_loss(logits, values, indices))
    want = torch.autograd.grad(y.sum(), leaves)
    del y, loss
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(block(x).sum(), leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(block(x).sum(), leaves)
    for _ in range(2):
        for g in got:
            g.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():  # without gradients nothing is held
        y = block(x)
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            block(x)
    assert torch.equal(y, enc.feed_forward(x, *(p.detach() for p in leaves)))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_matrices_that_lie_across(enc, dtype):
    """Parameters as transposed views, frozen ones, and a gradient that is one value."""
    g = _gen(31)
    x, gate, up, down, _ = _case(g, 90, 56, 104, dtype)
    across = [w.t().contiguous().t().requires_grad_(k != 1) for k, w in enumerate((gate, up, down))]
    straight = [w.clone().requires_grad_(k != 1) for k, w in enumerate((gate, up, down))]
    for matrices in (across, straight):
        enc.feed_forward(x, *matrices, activation="gelu").sum().backward()
    assert across[1].grad is None
    assert torch.equal(across[0].grad, straight[0].grad) and torch.equal(across[2].grad, straight[2].grad)


def test_two_calls_of_one_block_on_two_streams(enc):
    """Forward and backward passes with one block's parameters at once."""
    torch.manual_seed(5)
    block = enc.FeedForward(64, 160, dtype=torch.bfloat16)
    served = block.quantized()
    xs = [torch.randn(n, 64, device="cuda").bfloat16() for n in (400, 3)]

    def work(x):
        y, kept = enc.feed_forward(x, *(p.detach() for p in block.parameters()), keep=True)
        return (y, served(x), *enc.feed_forward_gradient(x, x, kept, *(p.detach() for p in block.parameters())))

    want = [work(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(10):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(work(xs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for outs in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[k]))


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "distilled_encoder.py"
    spec = importlib.util.spec_from_file_location("distilled_encoder", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_runs():
    shares = _example().main(rows=1500, classes=5, rounds=4, dim=32, hidden=48, top=3, batch=500, epochs=1)
    assert len(shares) == 3 and all(0.0 <= s <= 1.0 for s in shares)


def test_example_gradients(enc):
    """The student's gradients against 64-bit autograd of the same formulas.  A few
    products of at most 100 binary32 terms each, and their inverse norms: 1e-5 of the
    largest entry would be eight times their roundings; 1e-4 is allowed."""
    torch.manual_seed(1)
    student = _example().Student(90, 7, 32, 48, 5)
    tokens = torch.randint(0, 90, (60, 7), device="cuda", dtype=torch.int32)
    values, indices = torch.randn(60, 5, device="cuda").topk(3)
    enc.distillation_loss(student(tokens), values, indices, temperature=2.0)[0].mean().backward()
    names = dict(student.named_parameters())
    p = {name: w.detach().double().requires_grad_() for name, w in names.items()}

    def norm(x, name):
        return torch.nn.functional.layer_norm(x, (32,), p[name + ".weight"], p[name + ".bias"], getattr(student, name).eps)

    x = norm(p["leaves.weight"][tokens.long()].sum(1) * 7 ** -0.5, "norm")
    block = (_act(x @ p["block.gate"].t(), "silu")[0] * (x @ p["block.up"].t())) @ p["block.down"].t()
    z = norm(x + block, "last_norm") @ p["head.weight"].t() + p["head.bias"]
    log_q, log_p = (z / 2).log_softmax(1), (values.double() / 2).log_softmax(1)
    (4 * (log_p.exp() * (log_p - log_q.gather(1, indices))).sum(1)).mean().backward()
    for name, w in names.items():
        want = p[name].grad
        assert ((w.grad.double() - want).abs().max() <= 1e-4 * want.abs().max()), name
