"""The block, its 8-bit form and distillation at the ends of what they accept
(xgboost.encoder): more rows than a launch holds, infinities, types that modules are
cast to.  Tolerances are those of test_gpu_block.py and test_gpu_block8.py."""
import math

import pytest
import torch

from test_gpu_block import _forward64, _gen, _gradient64, _near, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


def test_distillation_of_more_rows_than_a_launch_holds(enc):
    """2^26 rows and a few, 64 lanes each: every part of them as in a call of its own."""
    rows, classes = (1 << 26) + 5, 10
    g = _gen(3)
    logits = torch.empty(rows, classes, device="cuda", dtype=torch.float16).normal_(generator=g)
    indices = torch.randint(-1, classes, (rows, 2), generator=g, device="cuda", dtype=torch.int32)
    values = torch.empty(rows, 2, device="cuda", dtype=torch.float16).normal_(generator=g)
    grad = torch.rand(rows, generator=g, device="cuda")
    loss, lse = enc.distillation_loss(logits, values, indices, temperature=1.5)
    d = enc.distillation_gradient(grad, logits, lse, values, indices, temperature=1.5)
    assert torch.isfinite(loss).all() and torch.isfinite(d).all()
    for begin in (0, 1 << 24, (1 << 25) - 500, (1 << 26) - 500):
        part = slice(begin, begin + 1000)
        want, want_lse = enc.distillation_loss(logits[part], values[part], indices[part], temperature=1.5)
        assert torch.equal(loss[part], want) and torch.equal(lse[part], want_lse)
        assert torch.equal(d[part], enc.distillation_gradient(grad[part], logits[part], want_lse, values[part], indices[part],
                                                              temperature=1.5))
    # One gradient for all rows, and teachers' rows that are one row.
    d = enc.distillation_gradient(grad[:1].expand(rows), logits, lse, values[:1].expand(rows, 2), indices[:1].expand(rows, 2))
    part = slice(rows - 1000, rows)
    assert torch.equal(d[part], enc.distillation_gradient(grad[:1].expand(1000), logits[part], lse[part],
                                                          values[:1].expand(1000, 2), indices[:1].expand(1000, 2)))


def test_distillation_of_more_wide_rows_than_a_launch_holds(enc):
    """2^24 rows and a few, 256 lanes each, of one row of logits: the loss at one entry of
    each row is that of the entry's column."""
    rows, classes = (1 << 24) + 3, 2100
    g = _gen(4)
    row = _randn(g, 1, classes)
    indices = torch.randint(0, classes, (rows, 1), generator=g, device="cuda", dtype=torch.int32)
    one = torch.zeros(1, 1, device="cuda")
    loss, lse = enc.distillation_loss(row.expand(rows, classes), one.expand(rows, 1), indices)
    each, each_lse = enc.distillation_loss(row.expand(classes, classes), one.expand(classes, 1),
                                           torch.arange(classes, device="cuda")[:, None])
    assert torch.equal(loss, each[indices[:, 0].long()]) and (lse == each_lse[0]).all()


def test_block_of_more_rows_than_small_tiles_launch(enc):
    """2^30 rows and a few of three values: smaller tiles would be 2^32 lanes.  Gradients come
    of rows at the beginning, where the small tiles would end, and at the end."""
    rows, dim, hidden = (1 << 30) + 300, 3, 5
    g = _gen(5)
    gate, up = (_randn(g, hidden, dim, dtype=torch.bfloat16) for _ in range(2))
    down = _randn(g, dim, hidden, dtype=torch.bfloat16)
    x = torch.empty(rows, dim, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    y, kept = enc.feed_forward(x, gate, up, down, keep=True)
    parts = [slice(0, 3000), slice((1 << 29) - 1500, (1 << 29) + 1500), slice((1 << 30) - 3000, (1 << 30)), slice(1 << 30, rows)]
    for part in parts:
        _near(y[part], *_forward64(x[part], gate, up, down, "silu"), "y")
    del y
    grad = torch.zeros(rows, dim, device="cuda", dtype=torch.bfloat16)
    for part in parts:
        grad[part] = _randn(g, part.stop - part.start, dim, dtype=torch.bfloat16)
    got = enc.feed_forward_gradient(grad, x, kept, gate, up, down)
    some = [torch.cat([t[part] for part in parts]) for t in (grad, x, kept)]
    wants = _gradient64(*some, gate, up, down, "silu")
    dx = torch.cat([got[0][part] for part in parts])
    for name, out, (want, error) in zip(("dx", "dgate", "dup", "ddown"), (dx, *got[1:]), wants):
        _near(out, want, error, name)
    assert not got[0][3000:4000].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows,dim,hidden", [(5, 24, 41), (40, 24, 41), (700, 24, 41), (700, 24, 40), (300, 64, 1003), (5000, 512, 1027)])
def test_infinities_stay_infinite(enc, rows, dim, hidden, dtype):
    """An infinity times positive factors, whatever pads the hidden values' rows, and
    rows beside it as they are without it."""
    g = _gen(rows + hidden)
    x, gate, up = (_randn(g, n, dim, dtype=dtype) for n in (rows, hidden, hidden))
    down = _randn(g, dim, hidden, dtype=dtype)
    gate[:, 5], up[:, 5] = gate[:, 5].abs() + 0.5, up[:, 5].abs() + 0.5
    down[7] = down[7].abs() + 0.5
    want = enc.feed_forward(x, gate, up, down)
    x[2, 5] = float("inf")
    got = enc.feed_forward(x, gate, up, down)
    assert got[2, 7] == float("inf")
    there = torch.arange(rows, device="cuda") != 2
    assert torch.equal(got[there], want[there])


@pytest.mark.parametrize("classes", [40, 5000])
def test_teachers_that_are_not_finite(enc, classes):
    """NaN or +inf among a row's values: its loss and all of its gradient are NaN, the other
    rows' as they are; in an absent entry they do not count."""
    g = _gen(classes)
    logits, values = _randn(g, 6, classes), _randn(g, 6, 3)
    indices = torch.tensor([[1, 7, 30]], device="cuda").repeat(6, 1)
    grad = torch.ones(6, device="cuda")
    bad, at = values.clone(), indices.clone()
    bad[1, 2], bad[3, 0], bad[4, 1] = float("nan"), float("inf"), float("nan")
    at[4, 1] = -1
    loss, lse = enc.distillation_loss(logits, bad, at)
    d = enc.distillation_gradient(grad, logits, lse, bad, at)
    want, want_lse = enc.distillation_loss(logits, values, at)
    want_d = enc.distillation_gradient(grad, logits, want_lse, values, at)
    spoilt = torch.tensor([False, True, False, True, False, False], device="cuda")
    assert torch.isnan(loss[spoilt]).all() and torch.isnan(d[spoilt]).all()
    assert torch.equal(loss[~spoilt], want[~spoilt]) and torch.equal(d[~spoilt], want_d[~spoilt]) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("classes", [12, 3000, 40000])
@pytest.mark.parametrize("offset", [0.0, 3000.0, -3000.0])
def test_loss_of_logits_far_from_zero(enc, classes, offset):
    """What all of a row's logits have in common does not count: its loss is off by 2^-23 of
    the differences' sizes (below 30 / T), of the sum (classes / 64 terms a lane, and 16) and
    of the entries' products, not of the logits' 12,000 / T."""
    temperature = 0.25
    g = _gen(classes)
    logits = _randn(g, 20, classes) + offset
    values, indices = (_randn(g, 20, classes) + 50).topk(8, 1)
    loss, lse = enc.distillation_loss(logits, values, indices, temperature=temperature)
    log_q = (logits.double() / temperature).log_softmax(1).gather(1, indices)
    log_p = (values.double() / temperature).log_softmax(1)
    want = temperature ** 2 * (log_p.exp() * (log_p - log_q)).sum(1)
    size = temperature ** 2 * (log_p.exp() * (log_p.abs() + log_q.abs() + 1)).sum(1)
    _near(loss, want, size * (30 / temperature + classes / 64 + 16) * 2.0 ** -23)
    z = logits.double() / temperature
    _near(lse, z.logsumexp(1), z.abs().amax(1) * 2.0 ** -23 + (classes / 64 + 32 + 30 / temperature) * 2.0 ** -23)


def test_loss_between_the_largest_values(enc):
    """A difference that passes binary32 before it is divided by the temperature: an entry of
    probability e^-3 that the logits hold for impossible, T^2 p 2 top / T = 0.38 top."""
    top = torch.finfo(torch.float32).max
    logits = torch.tensor([[top, -top, 0.0]], device="cuda")
    loss, _ = enc.distillation_loss(logits, torch.tensor([[0.0, -12.0]], device="cuda"), torch.tensor([[0, 1]], device="cuda"),
                                    temperature=4.0)
    want = 8.0 * top * math.exp(-3.0) / (1.0 + math.exp(-3.0))
    assert abs(loss.item() / want - 1) < 1e-6


def test_capture_while_a_graph_of_torchs_lives(enc):
    """Refused too where what holds the leaves on the default stream are torch's operators;
    once their results are gone, it is captured."""
    block = enc.FeedForward(24, 40)
    x = torch.randn(50, 24, device="cuda")
    values, indices = torch.randn(50, 24, device="cuda").topk(4)
    logits = torch.randn(50, 24, device="cuda", requires_grad=True)
    leaves = [*block.parameters(), logits]

    def refused(work):
        with pytest.raises(RuntimeError, match="default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                work()

    held = block.down * 2
    refused(lambda: block(x))
    held = logits.exp()
    refused(lambda: enc.distillation_loss(logits, values, indices))
    del held

    def step():
        loss = enc.distillation_loss(block(x) + logits, values, indices)[0] + enc.distillation_loss(logits, values, indices)[0]
        return torch.autograd.grad(loss.sum(), leaves)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for g in got:
            g.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
