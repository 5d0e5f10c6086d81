"""The leaf encoder's refusals: the package's argument checks, and the C
entries' own, which hold before any device work (no GPU needed).

torch has to be imported before xgboost.  This file's name comes before those
of the tests that import the package at their head, so a whole run does that.
"""
import ctypes
import subprocess
import sys

import pytest
import torch


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


def _lib():
    import xgboost.core as core
    lib = ctypes.CDLL(core._LIB.path)
    lib.mgb_last_error.restype = ctypes.c_char_p
    for name in ("embedding_gradient", "layer_norm_gradient", "orthogonalize"):
        getattr(lib, f"mgb_{name}_workspace_bytes").restype = ctypes.c_size_t
    return lib


def _refused(lib, ret, text):
    assert ret == -1 and text in lib.mgb_last_error().decode()


I64, F32, P = ctypes.c_int64, ctypes.c_float, ctypes.c_void_p


def test_c_entries_refuse_bad_sizes_and_pointers():
    lib = _lib()
    one = P(256)  # never read: every call below is refused

    def lookup(rows=1, bag=1, table=4, dim=8, stride=8, dtype=0, token=4, out=one):
        return lib.mgb_embedding_lookup(out, one, one, I64(rows), I64(bag), I64(table), I64(dim), I64(stride),
                                        F32(1), dtype, token, None)

    _refused(lib, lookup(rows=-1), "out of range")
    _refused(lib, lookup(bag=-1), "out of range")
    _refused(lib, lookup(rows=1 << 39, bag=(1 << 31) - 1), "out of range")
    _refused(lib, lookup(table=0), "table")
    _refused(lib, lookup(table=1 << 31), "table")
    _refused(lib, lookup(dim=0), "row must have")
    _refused(lib, lookup(dtype=3), "types")
    _refused(lib, lookup(token=2), "int32 or int64")
    _refused(lib, lookup(out=None), "null")

    def gradient(rows=10, bag=1, workspace=one, size=1 << 40):
        return lib.mgb_embedding_gradient(one, one, one, I64(rows), I64(bag), I64(4), I64(8), I64(8), F32(1), 0, 4,
                                          workspace, ctypes.c_size_t(size), None)

    _refused(lib, gradient(rows=1 << 31), "below 2^31")
    _refused(lib, gradient(rows=1 << 20, bag=1 << 11), "below 2^31")
    _refused(lib, gradient(workspace=None), "null")
    need = lib.mgb_embedding_gradient_workspace_bytes(I64(10), I64(1), I64(4), I64(8), 0)
    _refused(lib, gradient(size=need - 1), "workspace too small")

    def norm(rows=1, dim=8, weight=one, bias=one, dtype=0, weight_dtype=0):
        return lib.mgb_layer_norm(one, one, one, one, weight, bias, I64(rows), I64(dim), I64(dim), F32(1e-5), dtype,
                                  weight_dtype, None)

    _refused(lib, norm(rows=-1), "rows")
    _refused(lib, norm(rows=1 << 31), "rows")
    _refused(lib, norm(dim=0), "1 to 2^31")
    _refused(lib, norm(weight=None), "bias needs a weight")
    _refused(lib, norm(dtype=1, weight_dtype=2), "types")
    _refused(lib, norm(dtype=7), "types")

    def norm_gradient(dweight=one, dbias=one, size=1 << 40, workspace=one):
        return lib.mgb_layer_norm_gradient(one, dweight, dbias, one, one, one, one, one, I64(5), I64(8), I64(8), I64(8),
                                           0, 0, workspace, ctypes.c_size_t(size), None)

    _refused(lib, norm_gradient(dweight=None), "needs the weight's")
    _refused(lib, norm_gradient(size=8), "workspace too small")
    _refused(lib, norm_gradient(workspace=None), "null workspace")

    def orthogonalize(batch=1, rows=4, columns=4, steps=5, c=(3.0, -4.0, 2.0), dtype=0, size=1 << 40):
        return lib.mgb_orthogonalize(one, one, I64(batch), I64(rows), I64(columns), I64(4), I64(16), steps,
                                     (ctypes.c_float * 3)(*c), F32(1e-7), dtype, one, ctypes.c_size_t(size), None)

    _refused(lib, orthogonalize(batch=65536), "65,535")
    _refused(lib, orthogonalize(rows=(1 << 20) + 1), "2^20")
    _refused(lib, orthogonalize(steps=0), "steps")
    _refused(lib, orthogonalize(steps=101), "steps")
    _refused(lib, orthogonalize(c=(9.0, 0.0, 0.0)), "coefficients")
    _refused(lib, orthogonalize(c=(3.0, float("nan"), 0.0)), "coefficients")
    _refused(lib, orthogonalize(dtype=5), "types")
    _refused(lib, orthogonalize(size=100), "workspace too small")


def test_package_refuses_bad_arguments(enc):
    x = torch.zeros(4, 8)
    ids = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: enc.embedding_lookup(x, ids), lambda: enc.embedding_gradient(x, ids, 5),
                 lambda: enc.layer_norm(x), lambda: enc.layer_norm_gradient(x, x, x[:, 0], x[:, 0]),
                 lambda: enc.orthogonalize(x)):
        with pytest.raises(ValueError, match="on a GPU"):
            call()
    for call in (lambda: enc.embedding_lookup([1.0], ids), lambda: enc.layer_norm("x"),
                 lambda: enc.orthogonalize(None), lambda: enc.embedding_lookup(x.double(), ids),
                 lambda: enc.layer_norm(x.int()), lambda: enc.orthogonalize(x.to(torch.complex64))):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError, match="matrices"):
        enc.Muon([torch.nn.Parameter(torch.zeros(5))])
    with pytest.raises(TypeError, match="Booster"):
        enc.LeafTokenizer("model")


def test_torch_comes_first():
    """Two HIP runtimes in one process are refused with the reason."""
    path = [p for p in sys.path if p.endswith("python")][0]
    code = f"import sys; sys.path.insert(0, {path!r}); import xgboost, torch; from xgboost import encoder"
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, check=False)
    assert done.returncode != 0 and "import torch first" in done.stderr
    code = f"import sys; sys.path.insert(0, {path!r}); import torch, xgboost; from xgboost import encoder"
    assert subprocess.run([sys.executable, "-c", code], check=False).returncode == 0


@pytest.mark.gpu
def test_package_refuses_mismatches(enc):
    x = torch.zeros(4, 8, device="cuda")
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    bad = [
        (ValueError, "table of rows", lambda: enc.embedding_lookup(x[0], ids)),
        (TypeError, "int32 or int64", lambda: enc.embedding_lookup(x, ids.float())),
        (ValueError, "must be on", lambda: enc.embedding_lookup(x, ids.cpu())),
        (ValueError, "axis", lambda: enc.embedding_lookup(x, ids[0], pool=True)),
        (ValueError, "row must have", lambda: enc.embedding_lookup(x[:, :0], ids)),
        (ValueError, "table must have", lambda: enc.embedding_lookup(x[:0], ids)),
        (ValueError, "must have shape", lambda: enc.embedding_gradient(x[:3], ids, 5)),
        (ValueError, "num_embeddings", lambda: enc.embedding_gradient(x, ids, 0)),
        (ValueError, "last axis", lambda: enc.layer_norm(x[:, :0])),
        (ValueError, "bias needs", lambda: enc.layer_norm(x, None, x[0])),
        (ValueError, "weight must have shape", lambda: enc.layer_norm(x, x[0, :7])),
        (TypeError, "weight must be", lambda: enc.layer_norm(x, x[0].half())),
        (TypeError, "bias must be", lambda: enc.layer_norm(x.half(), x[0], x[0].half())),
        (ValueError, "must be on", lambda: enc.layer_norm(x, x[0], x[0].cpu())),
        (ValueError, "grad must be like", lambda: enc.layer_norm_gradient(x.half(), x, x[:, 0], x[:, 0])),
        (ValueError, "mean must be", lambda: enc.layer_norm_gradient(x, x, x[0], x[:, 0])),
        (ValueError, "matrix", lambda: enc.orthogonalize(x[0])),
        (ValueError, "three", lambda: enc.orthogonalize(x, coefficients=(1.0, 2.0))),
        (ValueError, "steps", lambda: enc.orthogonalize(x, steps=0)),
        (ValueError, "coefficients", lambda: enc.orthogonalize(x, coefficients=(1.0, 20.0, 1.0))),
    ]
    for kind, text, call in bad:
        with pytest.raises(kind, match=text):
            call()


def test_coefficients_that_leave_the_products_range_are_refused():
    """Singular values begin within [0, 1]; where the steps can take one so far that
    a product's operand passes what binary16 holds, the C entry refuses, before any
    device work."""
    lib = _lib()
    one = P(256)  # never read: every call below is refused

    def call(c, steps, dtype=0, eps=1e-7):
        return lib.mgb_orthogonalize(one, one, I64(1), I64(1), I64(1), I64(1), I64(1), steps, (ctypes.c_float * 3)(*c),
                                     F32(eps), dtype, one, ctypes.c_size_t(1 << 40), None)

    for dtype in (0, 1, 2):
        _refused(lib, call((5.0, 0.0, 0.0), 2, dtype), "coefficients")      # A = 25
        _refused(lib, call((8.0, 0.0, 0.0), 2, dtype), "coefficients")      # A = 64
        _refused(lib, call((2.0, 0.0, 0.0), 3, dtype), "coefficients")      # A = 16
        _refused(lib, call((1.0, 4.0, -1.0), 2, dtype), "coefficients")     # the largest value at 1: 4
        _refused(lib, call((8.0, -8.0, -8.0), 2, dtype), "coefficients")    # - 8 at 1
        _refused(lib, call((3.4445, -4.775, 2.6), 6, dtype), "coefficients")  # grows with every step
        _refused(lib, call((3.0, -4.0, 2.0), 5, dtype, -1e-3), "eps")
        _refused(lib, call((3.0, -4.0, 2.0), 5, dtype, float("nan")), "eps")


# Without a GPU the first argument alone is looked at before the device is.
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _calls(enc, device):
    x, w, ids = torch.ones(4, 8, device=device), torch.ones(8, device=device), torch.zeros(4, dtype=torch.int64, device=device)
    stat = torch.zeros(4, device=device)
    first = (lambda t: enc.embedding_lookup(t, ids), lambda t: enc.embedding_gradient(t, ids, 5), lambda t: enc.layer_norm(t),
             lambda t: enc.layer_norm_gradient(t, x, stat, stat), lambda t: enc.orthogonalize(t))
    later = (lambda t: enc.layer_norm(x, t[0]), lambda t: enc.layer_norm(x, w, t[0]),
             lambda t: enc.layer_norm_gradient(x, t, stat, stat), lambda t: enc.layer_norm_gradient(x, x, t[:, 0], stat),
             lambda t: enc.layer_norm_gradient(x, x, stat, t[:, 0]), lambda t: enc.layer_norm_gradient(x, x, stat, stat, t[0]))
    return x, first if device == "cpu" else first + later


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_derivatives_are_refused(enc, device):
    """A dual tensor's tangent would be lost: no operator takes one."""
    x, calls = _calls(enc, device)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(dual)


@pytest.mark.parametrize("device", DEVICES)
def test_tracing_is_refused(enc, device):
    """A trace would hold the result as a constant."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, calls = _calls(enc, device)
    for call in calls:
        def result(t):
            out = call(t)  # pylint: disable=cell-var-from-loop
            return out if isinstance(out, torch.Tensor) else out[0]
        for trace in (lambda: torch.jit.trace(result, x), lambda: make_fx(result)(x),
                      lambda: make_fx(result, tracing_mode="fake")(x)):
            with pytest.raises(NotImplementedError, match="trace"):
                trace()


def test_muon_refuses_later_groups(enc):
    """A group that is added later is looked at as the first ones are, and left out if refused."""
    opt = enc.Muon([torch.nn.Parameter(torch.zeros(4, 5))])
    for shape in ((5,), (2, 3, 4), ()):
        with pytest.raises(ValueError, match="matrices"):
            opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3, 3)), torch.nn.Parameter(torch.zeros(shape))]})
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, 7))], "lr": 0.5})
    assert [len(group["params"]) for group in opt.param_groups] == [1, 1] and opt.param_groups[1]["lr"] == 0.5
