"""Modules whose matrices are in 8 bits, cast and moved as torch's modules are: the matrices
keep their types and values."""
import copy

import pytest
import torch

CASTS = [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.float(), lambda m: m.double(),
         lambda m: m.to(m.gate_values.device, torch.float16), lambda m: m.type(torch.float16),
         lambda m: torch.nn.Sequential(m).to(torch.bfloat16)[0], lambda m: copy.deepcopy(m).to(torch.half)]


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


def _matrices(module):
    return [(name, t.dtype, t.view(torch.uint8).clone()) for name, t in module.named_buffers()]


def _check(module):
    want = _matrices(module)
    assert [t for _, t, _ in want] == [torch.float8_e4m3fn, torch.float8_e8m0fnu] * 3
    for cast in CASTS:
        got = _matrices(cast(module))
        assert [w[:2] for w in got] == [w[:2] for w in want]
        assert all(torch.equal(a[2], b[2]) for a, b in zip(got, want))


def test_casts_leave_blocks(enc, monkeypatch):
    def blocks(w):  # (the operator itself needs a GPU)
        values = torch.randint(0, 120, (w.shape[0], -(-w.shape[1] // 128) * 128), dtype=torch.uint8)
        scales = torch.randint(100, 140, (w.shape[0], 4), dtype=torch.uint8)[:, :values.shape[1] // 128]
        return enc.BlockScaled(values.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), w.shape[1])
    monkeypatch.setattr(enc, "quantize_blocks", blocks)
    _check(enc.FeedForward(250, 200, device="cpu").quantized())


@pytest.mark.gpu
def test_casts_are_served(enc):
    served = enc.FeedForward(250, 200).quantized()
    x = torch.randn(50, 250, device="cuda")
    want = {t: served(x.to(t)) for t in (torch.float32, torch.float16, torch.bfloat16)}
    _check(served)
    for t, y in want.items():
        assert torch.equal(served.to(t)(x.to(t)), y)
        assert torch.equal(copy.deepcopy(served).cpu().to(t).cuda()(x.to(t)), y)
