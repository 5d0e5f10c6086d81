"""Orthogonalised updates at every form their products take, and the optimizer
over them, against 64-bit forms.

LARGE has what the products come in: tiles of 128, of 64 and of 32 with the depth
in 1, 4 and 16 parts, single and by twos, symmetric or not, operands with and
without low parts, segments of one step and of several, batches.
"""
import copy

import pytest
import torch
from test_gpu_encoder import COEFFICIENTS, U, _gen, _orthogonal64, _randn, enc  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = ["f32", "f16", "bf16"]


def _plain32(update, steps, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = update.float()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    for _ in range(steps):
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT.contiguous() if tall else x


def _near_plain(got, update, steps, segmented):
    """Against 64 bits, by the error that plain binary32 makes of the same input.
    Operands of 22 bits where that has 24 are rounded four times as coarsely, and
    the product of the two low parts, left out, is as much again: 8.  In a segment
    of several steps A is carried on instead of taken from X, which adds
    b a^2 / a^3 of a step's error to it, below 2: 16.  A result x of fewer bits:
    |round(x) - want| <= |round(want) - want| + 2 |x - want|, as no number of the
    type is nearer to x than round(x)."""
    want = _orthogonal64(update, steps)
    norm = want.norm()
    error = ((_plain32(update, steps).double() - want).norm() / norm).item()
    bound = (16 if segmented else 8) * error
    if got.dtype != torch.float32:
        bound = 2 * bound + ((want.to(got.dtype).double() - want).norm() / norm).item()
    off = ((got.double() - want).norm() / norm).item()
    assert off <= bound, f"{off:.2e} of the norm, bound {bound:.2e}, binary32 {error:.2e}"


# shape, bits of the types it is for.  Tiles of 128: 2,048 x 4,096 (segments), 1,930 x
# 2,100, the batches; of 64: 700 x 1,400 and 500 x 1,100 (segments), 1,500 x 1,100;
# of 32: 400 x 2,500 and 128 x 2,048 (segments).
LARGE = [((2048, 4096), (16,)), ((1930, 2100), (16, 32)), ((2100, 1930), (32,)), ((700, 1400), (16, 32)),
         ((1500, 1100), (16, 32)), ((1100, 1500), (16, 32)), ((500, 1100), (16, 32)), ((400, 2500), (16, 32)),
         ((2500, 450), (16,)), ((128, 2048), (16, 32)), ((2, 7, 512, 512), (16, 32)), ((14, 450, 900), (16, 32)),
         ((3, 900, 450), (16,))]
LARGE = [pytest.param(shape, dtype, id="x".join(map(str, shape)) + "-" + name) for shape, bits in LARGE
         for dtype, name in zip(TYPES, NAMES) if (32 if dtype == torch.float32 else 16) in bits]


@pytest.mark.parametrize("steps", [5, 1])
@pytest.mark.parametrize("low_rank", [False, True], ids=["random", "low_rank"])
@pytest.mark.parametrize("shape,dtype", LARGE)
def test_products(enc, shape, dtype, low_rank, steps):  # noqa: F811
    g = _gen(sum(shape) + steps)
    if low_rank:  # a few directions, the others a thousand times smaller
        update = _randn(g, *shape[:-1], 6) @ _randn(g, *shape[:-2], 6, shape[-1]) + 1e-3 * _randn(g, *shape)
    else:
        update = 0.01 * _randn(g, *shape)
    update = update.to(dtype)
    got = enc.orthogonalize(update, steps=steps)
    assert got.shape == update.shape and got.dtype == dtype
    for one, of in zip(got.reshape(-1, *shape[-2:]), update.reshape(-1, *shape[-2:])):
        _near_plain(one, of, steps, dtype != torch.float32)
    for _ in range(3):  # the same bits, launch after launch
        assert torch.equal(got, enc.orthogonalize(update, steps=steps))


@pytest.mark.parametrize("steps", [2, 3, 4, 6, 7])
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_segments(enc, dtype, steps):  # noqa: F811
    """Segments of two and three steps and what follows them, few directions far above the others."""
    g = _gen(steps)
    update = (_randn(g, 450, 5) @ _randn(g, 5, 900) + 1e-3 * _randn(g, 450, 900)).to(dtype)
    _near_plain(enc.orthogonalize(update, steps=steps), update, steps, dtype != torch.float32)
    update = update.t()
    _near_plain(enc.orthogonalize(update, steps=steps), update, steps, dtype != torch.float32)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_orthogonalize_coefficients_at_the_limit(enc, dtype):  # noqa: F811
    """What is accepted is right where singular values are as large as they can be, 1 at
    first: a rank-one matrix' singular value runs through the polynomial.  Refused is
    what would pass binary16's range."""
    for shape in ((1, 1), (3, 200), (500, 800), (700, 1400)):
        update = torch.zeros(shape, device="cuda", dtype=dtype)
        update[0, 0] = 4.0
        for coefficients, steps in (((3.9, 0.0, 0.0), 2), ((1.9, 0.0, 0.0), 3), ((8.0, 0.0, 0.0), 1), ((8.0, 8.0, 8.0), 1),
                                    ((1.5, -0.5, 0.0), 20), (COEFFICIENTS, 100), ((3.4, -4.0, 1.5), 12)):
            got = enc.orthogonalize(update, steps=steps, coefficients=coefficients)
            s, slope = 1.0, 1.0
            for _ in range(steps):
                a, b, c = coefficients
                slope = max(1.0, slope * abs(a + 3 * b * s ** 2 + 5 * c * s ** 4))
                s = a * s + b * s ** 3 + c * s ** 5
            # A value's rounding, 2^-22, a few times a step, through the steps behind it.
            off = abs(got[0, 0].double().item() - s)
            assert off <= abs(s) * (U[dtype] + 64 * steps * slope * 2.0 ** -22), (shape, coefficients, steps, off)
            rest = got.double().clone()
            rest[0, 0] = 0.0
            assert not rest.any()
        for coefficients, steps in (((5.0, 0.0, 0.0), 2), ((8.0, 8.0, 8.0), 2)):
            with pytest.raises(ValueError, match="coefficients"):
                enc.orthogonalize(update, steps=steps, coefficients=coefficients)


def _muon64(p, m, grad, lr, momentum, nesterov, decay, steps=5):
    """The docstring's step in 64 bits: the weight and the momentum after it, and the update's norm."""
    m = momentum * m + grad.double()
    o = _orthogonal64(grad.double() + momentum * m if nesterov else m, steps)
    size = lr * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
    return p - size * o - lr * decay * p, m, size * o.norm()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (False, 0.1), (True, 0.01)])
@pytest.mark.parametrize("shape", [(40, 70), (90, 30), (70, 300)])
def test_muon_steps(enc, shape, nesterov, decay, dtype):  # noqa: F811
    """Eight steps by the formula.  An update is off by at most 2^-22 (a^5 + 5 a^4) of
    its norm, a binary32 weight by 4 roundings a step.  16-bit weights are kept in
    binary32 between the steps and show it rounded once, whatever the steps."""
    g = _gen(sum(shape))
    p = torch.nn.Parameter(_randn(g, *shape, dtype=dtype) * 0.2)
    lr, momentum = 0.02, 0.9
    opt = enc.Muon([p], lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=decay)
    want, m = p.detach().double(), torch.zeros(shape, dtype=torch.float64, device="cuda")
    a, slack = COEFFICIENTS[0], 0.0
    for _ in range(8):
        p.grad = _randn(g, *shape, dtype=dtype)
        opt.step()
        want, m, size = _muon64(want, m, p.grad, lr, momentum, nesterov, decay)
        slack += (a ** 5 + 5 * a ** 4) * 2.0 ** -22 * size.item() + 4 * 2.0 ** -24 * want.abs().max().item()
        bound = slack + U[dtype] * (want.abs() + slack)
        assert p.dtype == dtype and ((p.detach().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_muon_small_decay_and_momentum_last(enc, dtype):  # noqa: F811
    """Without gradients only the decay is left, 1 - 2e-4 a step: 500 steps take a tenth,
    although one is less than a 16-bit weight's rounding; each step rounds twice in binary32."""
    p = torch.nn.Parameter(torch.ones(16, 24, device="cuda", dtype=dtype))
    opt = enc.Muon([p], lr=0.02, weight_decay=0.01)
    p.grad = torch.zeros_like(p)
    for _ in range(500):
        opt.step()
    want = (1.0 - 0.02 * 0.01) ** 500
    assert abs(p[3, 5].item() - want) <= (U[dtype] + 1000 * 2.0 ** -24) * want
    # Momentum keeps what is below 2^-9 of it: 1 + 300 / 1024, not 1 (300 further roundings).
    p = torch.nn.Parameter(torch.zeros(16, 24, device="cuda", dtype=dtype))
    opt = enc.Muon([p], lr=0.0, momentum=1.0)
    p.grad = torch.ones_like(p)
    opt.step()
    p.grad = torch.full_like(p, 2.0 ** -10)
    for _ in range(300):
        opt.step()
    m = opt.state[p]["momentum"]
    assert m.dtype == torch.float32 and (m.double() - (1 + 300 / 1024)).abs().max() <= 300 * 2.0 ** -23


def test_muon_weights_set_from_outside_and_resumed(enc):  # noqa: F811
    """A 16-bit weight that was overwritten goes on from there, and a saved state goes on as if nothing was."""
    g = _gen(7)
    grads = [_randn(g, 20, 30, dtype=torch.bfloat16) for _ in range(6)]
    start = _randn(g, 20, 30, dtype=torch.bfloat16)

    def run(opt, p, some):
        for grad in some:
            p.grad = grad.clone()
            opt.step()

    def made(value):
        p = torch.nn.Parameter(value.clone())
        return p, enc.Muon([p], lr=1e-3, weight_decay=0.01)

    p, opt = made(start)
    run(opt, p, grads[:3])
    saved, weight = copy.deepcopy(opt.state_dict()), p.detach().clone()
    run(opt, p, grads[3:])
    q, other = made(weight)
    other.load_state_dict(saved)
    run(other, q, grads[3:])
    assert torch.equal(p, q)
    for key in opt.state[p]:
        assert torch.equal(opt.state[p][key], other.state[q][key])
    other_values = opt.state[p]["weight"].to(p.dtype) != 2.0
    with torch.no_grad():
        p.fill_(2.0)
    p.grad = torch.zeros_like(p)
    opt.state[p]["momentum"].zero_()
    opt.step()
    assert (p == 2.0).all()  # 2 - 2e-5, rounded
    assert (opt.state[p]["weight"][other_values] < 2.0).all() and other_values.sum() > 500


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES)
def test_muon_captured(enc, dtype):  # noqa: F811
    """A captured step, replayed with other gradients and eager work between, gives the eager steps' bits."""
    g = _gen(9)
    grads = [_randn(g, 30, 50, dtype=dtype) for _ in range(8)]
    start = _randn(g, 30, 50, dtype=dtype)

    def made():
        p = torch.nn.Parameter(start.clone())
        p.grad = grads[0].clone()
        return p, enc.Muon([p], lr=1e-4, weight_decay=0.01)

    p, eager = made()
    q, captured = made()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured.step()
    torch.cuda.current_stream().wait_stream(side)
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for grad in grads[1:]:
        q.grad.copy_(grad)
        graph.replay()
        torch.cuda.synchronize()
        p.grad.copy_(grad)
        eager.step()
        assert torch.equal(p, q)
        for key, value in eager.state[p].items():
            assert torch.equal(value, captured.state[q][key]), key


def test_muon_state_of_other_types(enc):  # noqa: F811
    """A state saved with a 16-bit momentum, or for weights of another type, is taken in the weight's state type."""
    g = _gen(10)
    for dtype, saved_type in ((torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.bfloat16)):
        p = torch.nn.Parameter(_randn(g, 12, 18, dtype=dtype))
        opt = enc.Muon([p])
        m = _randn(g, 12, 18, dtype=saved_type)
        opt.load_state_dict({"state": {0: {"momentum": m}}, "param_groups": opt.state_dict()["param_groups"]})
        kept = opt.state[p]["momentum"]
        assert kept.dtype == torch.float32 and torch.equal(kept, m.float())
        p.grad = torch.zeros_like(p)
        opt.step()
        assert torch.equal(opt.state[p]["momentum"], m.float() * 0.95) and m.dtype == saved_type
