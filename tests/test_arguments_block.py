"""Refusals of the encoder's block, its 8-bit products and its distillation: the
package's argument checks, and the C entries' own, which hold before any device
work (no GPU needed).

torch has to be imported before xgboost, as in test_arguments_encoder.py.
"""
import ctypes

import pytest
import torch

I64, F32, P, INT = ctypes.c_int64, ctypes.c_float, ctypes.c_void_p, ctypes.c_int


def _struct(name, fields):
    return type(name, (ctypes.Structure,), {"_fields_": fields})


Forward = _struct("Forward", [(n, P) for n in ("y", "kept", "x", "gate", "up", "down")] +
                  [(n, I64) for n in ("rows", "dim", "hidden", "x_stride", "gate_stride", "up_stride", "down_stride")] +
                  [("activation", INT), ("dtype", INT)])
Gradient = _struct("Gradient", [(n, P) for n in ("dx", "dgate", "dup", "ddown", "grad", "x", "kept", "gate", "up", "down")] +
                   [(n, I64) for n in ("rows", "dim", "hidden", "grad_stride", "x_stride", "gate_stride", "up_stride",
                                       "down_stride")] + [("activation", INT), ("dtype", INT)])
Blocks = _struct("Blocks", [("values", P), ("scales", P)] + [(n, I64) for n in ("rows", "blocks", "stride", "scale_stride")])
Matmul = _struct("Matmul", [("out", P), ("x", Blocks), ("weight", Blocks), ("dtype", INT)])
Serve = _struct("Serve", [("y", P), ("x", P), ("gate", Blocks), ("up", Blocks), ("down", Blocks)] +
                [(n, I64) for n in ("rows", "dim", "hidden", "x_stride")] + [("activation", INT), ("dtype", INT)])
Distillation = _struct("Distillation", [(n, P) for n in ("loss", "lse", "dlogits", "grad", "logits", "values", "indices")] +
                       [(n, I64) for n in ("rows", "classes", "top", "stride", "value_stride", "index_stride", "grad_stride")] +
                       [("temperature", F32), ("dtype", INT), ("value_dtype", INT), ("index_bytes", INT)])
HERE = 256  # never read: every call below is refused
MUCH = ctypes.c_size_t(1 << 60)


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


@pytest.fixture(scope="module")
def lib():
    import xgboost.core as core
    lib = ctypes.CDLL(core._LIB.path)
    lib.mgb_last_error.restype = ctypes.c_char_p
    for name in ("feed_forward", "feed_forward_gradient", "block_matmul", "block_feed_forward", "distillation_loss"):
        getattr(lib, f"mgb_{name}_workspace_bytes").restype = ctypes.c_size_t
    return lib


def _refused(lib, ret, text):
    assert ret == -1 and text in lib.mgb_last_error().decode(), lib.mgb_last_error()


def _fill(struct, **changes):
    for name, kind in struct._fields_:
        if kind is P:
            setattr(struct, name, HERE)
    for name, value in changes.items():
        setattr(struct, name, value)
    return struct


@pytest.mark.parametrize("changes,text", [
    (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(dim=0), "sides"), (dict(hidden=0), "sides"),
    (dict(dim=(1 << 20) + 1), "sides"), (dict(hidden=(1 << 20) + 1), "sides"), (dict(activation=2), "activation"),
    (dict(dtype=3), "types"), (dict(x_stride=1 << 40), "stride"), (dict(down_stride=-(1 << 40)), "stride"),
    (dict(x=None), "null"), (dict(down=None), "null")])
def test_feed_forward_entries(lib, changes, text):
    sizes = dict(rows=4, dim=8, hidden=16, x_stride=8, gate_stride=8, up_stride=8, down_stride=16)
    p = _fill(Forward(), **{**sizes, **changes})
    _refused(lib, lib.mgb_feed_forward(ctypes.byref(p), P(HERE), MUCH, None), text)
    g = _fill(Gradient(), grad_stride=8, **{**sizes, **changes})
    _refused(lib, lib.mgb_feed_forward_gradient(ctypes.byref(g), P(HERE), MUCH, None), text)


def test_workspaces_are_checked(lib):
    sizes = dict(rows=4, dim=8, hidden=16, x_stride=8, gate_stride=8, up_stride=8, down_stride=16)
    p, g = _fill(Forward(), **sizes), _fill(Gradient(), grad_stride=8, **sizes)
    for name, a in (("feed_forward", p), ("feed_forward_gradient", g)):
        call = getattr(lib, "mgb_" + name)
        need = getattr(lib, f"mgb_{name}_workspace_bytes")(ctypes.byref(a))
        assert need > 0
        _refused(lib, call(ctypes.byref(a), P(HERE), ctypes.c_size_t(need - 1), None), "too small")
        _refused(lib, call(ctypes.byref(a), None, MUCH, None), "null")
        _refused(lib, call(ctypes.byref(a), P(HERE + 16), MUCH, None), "256")
        _refused(lib, call(None, P(HERE), MUCH, None), "null")
    m = Blocks(HERE, HERE, 16, 1, 128, 4)
    s = Serve(HERE, HERE, m, m, Blocks(HERE, HERE, 8, 1, 128, 4), 4, 8, 16, 8, 0, 2)
    need = lib.mgb_block_feed_forward_workspace_bytes(ctypes.byref(s))
    assert need > 0
    _refused(lib, lib.mgb_block_feed_forward(ctypes.byref(s), P(HERE), ctypes.c_size_t(need - 1), None), "too small")
    b = Matmul(HERE, m, m, 0)
    assert lib.mgb_block_matmul_workspace_bytes(ctypes.byref(b)) == 0  # (few rows are read as they are)
    many = Blocks(HERE, HERE, 64, 1, 128, 4)
    b = Matmul(HERE, many, m, 0)
    need = lib.mgb_block_matmul_workspace_bytes(ctypes.byref(b))
    assert need > 0
    _refused(lib, lib.mgb_block_matmul(ctypes.byref(b), P(HERE), ctypes.c_size_t(need - 1), None), "too small")


def _block(rows=4, blocks=2, stride=256, scale_stride=4, values=HERE, scales=HERE):
    return Blocks(values, scales, rows, blocks, stride, scale_stride)


@pytest.mark.parametrize("changes,text", [
    (dict(rows=-1), "rows"), (dict(blocks=0), "blocks"), (dict(blocks=8193, stride=1 << 20), "blocks"),
    (dict(stride=255), "16-byte"), (dict(stride=264), "16-byte"), (dict(stride=128), "16-byte"),
    (dict(scale_stride=2), "words"), (dict(scale_stride=6), "words"), (dict(values=264), "16 bytes"),
    (dict(scales=258), "at 4")])
def test_blocks_are_checked(lib, changes, text):
    good, bad = _block(), _block(**changes)
    _refused(lib, lib.mgb_quantize_blocks(ctypes.byref(bad), P(HERE), I64(256), I64(256), 0, None), text)
    for p in (Matmul(HERE, bad, good, 2), Matmul(HERE, good, bad, 2)):
        _refused(lib, lib.mgb_block_matmul(ctypes.byref(p), P(HERE), MUCH, None), text)
    for k in range(3):
        matrices = [bad if k == j else good for j in range(3)]
        p = Serve(HERE, HERE, *matrices, 4, 256, 4, 256, 0, 2)
        _refused(lib, lib.mgb_block_feed_forward(ctypes.byref(p), P(HERE), MUCH, None), text)


def test_block_entries(lib):
    good = _block()
    _refused(lib, lib.mgb_quantize_blocks(ctypes.byref(good), P(HERE), I64(257), I64(257), 0, None), "hold its values")
    _refused(lib, lib.mgb_quantize_blocks(ctypes.byref(good), P(HERE), I64(128), I64(128), 0, None), "hold its values")
    _refused(lib, lib.mgb_quantize_blocks(ctypes.byref(good), P(HERE), I64(200), I64(200), 3, None), "types")
    _refused(lib, lib.mgb_quantize_blocks(ctypes.byref(good), None, I64(200), I64(200), 0, None), "null")
    _refused(lib, lib.mgb_block_matmul(ctypes.byref(Matmul(HERE, good, _block(blocks=1), 2)), P(HERE), MUCH, None), "same blocks")
    _refused(lib, lib.mgb_block_matmul(ctypes.byref(Matmul(HERE, good, good, 5)), P(HERE), MUCH, None), "types")
    _refused(lib, lib.mgb_block_matmul(ctypes.byref(Matmul(None, good, good, 2)), P(HERE), MUCH, None), "null")
    gate, down = _block(rows=200), _block(rows=250, blocks=2)

    def serve(gate=gate, up=gate, down=down, rows=4, dim=250, hidden=200, activation=0, dtype=2):
        p = Serve(HERE, HERE, gate, up, down, rows, dim, hidden, dim, activation, dtype)
        return lib.mgb_block_feed_forward(ctypes.byref(p), P(HERE), MUCH, None)

    _refused(lib, serve(dim=251), "do not fit")
    _refused(lib, serve(hidden=199), "do not fit")
    _refused(lib, serve(up=_block(rows=199)), "do not fit")
    _refused(lib, serve(up=_block(rows=200, stride=512)), "lie alike")
    _refused(lib, serve(activation=7), "activation")
    _refused(lib, serve(dtype=4), "types")
    _refused(lib, serve(rows=-1), "rows")


@pytest.mark.parametrize("changes,text", [
    (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(classes=0), "logits"), (dict(classes=1 << 31), "logits"),
    (dict(top=-1), "entries"), (dict(top=1025), "entries"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(index_bytes=2), "int32 or int64"), (dict(dtype=3), "types"),
    (dict(value_dtype=-1), "types"), (dict(stride=1 << 40), "stride"), (dict(logits=None), "null"), (dict(values=None), "null"),
    (dict(lse=None), "null")])
def test_distillation_entries(lib, changes, text):
    p = _fill(Distillation(), **{**dict(rows=4, classes=10, top=2, stride=10, value_stride=2, index_stride=2, grad_stride=1,
                                        temperature=1.0, index_bytes=8), **changes})
    _refused(lib, lib.mgb_distillation_loss(ctypes.byref(p), P(HERE), MUCH, None), text)
    _refused(lib, lib.mgb_distillation_gradient(ctypes.byref(p), None), text)


def _calls(enc, device):
    x, w = torch.ones(4, 8, device=device), torch.ones(16, 8, device=device)
    down, kept = torch.ones(8, 16, device=device), torch.zeros(4, 2, 16, device=device)
    at, stat = torch.zeros(4, 1, dtype=torch.int64, device=device), torch.zeros(4, device=device)
    return x, (lambda t: enc.feed_forward(t, w, w, down),
               lambda t: enc.feed_forward_gradient(t, x, kept, w, w, down), lambda t: enc.quantize_blocks(t),
               lambda t: enc.distillation_loss(t, x[:, :1], at),
               lambda t: enc.distillation_gradient(stat, t, stat, x[:, :1], at))


def test_package_refuses_bad_arguments(enc):
    x, calls = _calls(enc, "cpu")
    for call in calls:
        with pytest.raises(ValueError, match="on a GPU"):
            call(x)
        with pytest.raises((TypeError, ValueError), match="must be"):
            call(x.double())
        with pytest.raises((TypeError, AttributeError)):
            call("x")
    for call in (lambda: enc.block_matmul(x, x), lambda: enc.block_feed_forward(x, x, x, x)):
        with pytest.raises(TypeError, match="BlockScaled"):
            call()
    with pytest.raises(ValueError, match="one length"):
        enc.block_matmul(enc.BlockScaled(x, x, 8), enc.BlockScaled(x, x, 9))


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_and_traces_are_refused(enc, device):
    from torch.fx.experimental.proxy_tensor import make_fx
    x, calls = _calls(enc, device)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls[:-1]:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)
    for call in calls:
        def result(t):
            out = call(t)  # pylint: disable=cell-var-from-loop
            return out if isinstance(out, torch.Tensor) else out[0]
        for trace in (lambda: torch.jit.trace(result, x), lambda: make_fx(result)(x)):
            with pytest.raises(NotImplementedError, match="trace"):
                trace()


@pytest.mark.gpu
def test_package_refuses_mismatches(enc):
    x, w = torch.ones(4, 8, device="cuda"), torch.ones(16, 8, device="cuda")
    d, kept = torch.ones(8, 16, device="cuda"), torch.zeros(4, 2, 16, device="cuda")
    at, stat = torch.zeros(4, 2, dtype=torch.int64, device="cuda"), torch.zeros(4, device="cuda")
    v = x[:, :2]
    q = enc.quantize_blocks(w)
    qd = enc.quantize_blocks(d)
    B = enc.BlockScaled
    bad = [
        (ValueError, "gate must have shape", lambda: enc.feed_forward(x, w[:, :7], w, d)),
        (ValueError, "gate must have shape", lambda: enc.feed_forward(x, w[0], w, d)),
        (ValueError, "up must have shape", lambda: enc.feed_forward(x, w, w[:15], d)),
        (ValueError, "down must have shape", lambda: enc.feed_forward(x, w, w, d.t())),
        (TypeError, "gate must be", lambda: enc.feed_forward(x, w.half(), w, d)),
        (TypeError, "x must be", lambda: enc.feed_forward(x.double(), w, w, d)),
        (ValueError, "must be on", lambda: enc.feed_forward(x, w.cpu(), w, d)),
        (ValueError, "activation", lambda: enc.feed_forward(x, w, w, d, activation="relu")),
        (ValueError, "activation", lambda: enc.feed_forward(x, w, w, d, activation=None)),
        (ValueError, "last axis", lambda: enc.feed_forward(x[:, :0], w[:, :0], w[:, :0], d[:0])),
        (ValueError, "gate must have shape", lambda: enc.feed_forward(x, w[:0], w[:0], d[:, :0])),
        (ValueError, "grad must be like", lambda: enc.feed_forward_gradient(x.half(), x, kept, w, w, d)),
        (ValueError, "grad must be like", lambda: enc.feed_forward_gradient(x[:3], x, kept, w, w, d)),
        (ValueError, "kept must be", lambda: enc.feed_forward_gradient(x, x, kept[:, 0], w, w, d)),
        (ValueError, "kept must be", lambda: enc.feed_forward_gradient(x, x, kept.half(), w, w, d)),
        (ValueError, "last axis", lambda: enc.quantize_blocks(x[:, :0])),
        (TypeError, "float8_e4m3fn", lambda: enc.block_matmul(B(w, q.scales, 8), q)),
        (TypeError, "float8_e8m0fnu", lambda: enc.block_matmul(q, B(q.values, q.scales.float(), 8))),
        (ValueError, "scales must have shape", lambda: enc.block_matmul(q, B(q.values, q.scales[:3], 8))),
        (ValueError, "whole blocks", lambda: enc.block_matmul(q, B(q.values[:, :64], q.scales, 8))),
        (ValueError, "must be a matrix", lambda: enc.block_matmul(q, B(q.values[0], q.scales[0], 8))),
        (ValueError, "be on", lambda: enc.block_matmul(q, B(q.values.cpu(), q.scales.cpu(), 8))),
        (TypeError, "dtype must be", lambda: enc.block_matmul(q, q, dtype=torch.float64)),
        (TypeError, "dtype must be", lambda: enc.block_matmul(q, q, dtype="f32")),
        (ValueError, "gate must have rows of 2 blocks", lambda: enc.block_feed_forward(torch.ones(4, 200, device="cuda"), q, q, qd)),
        (ValueError, "up must have shape", lambda: enc.block_feed_forward(x, q, enc.quantize_blocks(w[:15]), qd)),
        (ValueError, "down must have", lambda: enc.block_feed_forward(x, q, q, q)),
        (ValueError, "last axis", lambda: enc.distillation_loss(x[:, :0], v, at)),
        (ValueError, "values must have shape", lambda: enc.distillation_loss(x, v[:3], at[:3])),
        (ValueError, "values must have shape", lambda: enc.distillation_loss(x, v[0], at[0])),
        (ValueError, "indices must have shape", lambda: enc.distillation_loss(x, v, at[:, :1])),
        (TypeError, "int32 or int64", lambda: enc.distillation_loss(x, v, at.float())),
        (TypeError, "values must be", lambda: enc.distillation_loss(x, v.double(), at)),
        (ValueError, "must be on", lambda: enc.distillation_loss(x, v, at.cpu())),
        (ValueError, "temperature", lambda: enc.distillation_loss(x, v, at, temperature=0.0)),
        (ValueError, "temperature", lambda: enc.distillation_loss(x, v, at, temperature=float("nan"))),
        (ValueError, "temperature", lambda: enc.distillation_loss(x, v, at, temperature=1e-60)),
        (ValueError, "1,024", lambda: enc.distillation_loss(torch.ones(1, 2000, device="cuda"), torch.ones(1, 1025, device="cuda"),
                                                          torch.zeros(1, 1025, device="cuda", dtype=torch.int32))),
        (ValueError, "grad must be", lambda: enc.distillation_gradient(stat[:3], x, stat, v, at)),
        (ValueError, "lse must be", lambda: enc.distillation_gradient(stat, x, stat.half(), v, at)),
    ]
    for kind, text, call in bad:
        with pytest.raises(kind, match=text):
            call()
    for call in (lambda t: enc.block_feed_forward(t, q, q, qd), lambda t: enc.block_matmul(enc.quantize_blocks(t), q),
                 lambda t: enc.feed_forward_gradient(t, x, kept, w, w, d)[2],
                 lambda t: enc.distillation_gradient(stat, t, stat, v, at)):
        out = call(x.clone().requires_grad_())
        with pytest.raises(NotImplementedError, match="no derivative"):
            out.float().sum().backward()
