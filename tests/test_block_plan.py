"""How the encoder's products divide their work (csrc/feed_forward.hpp, csrc/product.hpp),
on the host: tests/block_plan.cpp goes through the sizes that the entries take."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch  # noqa: F401  (before the package: both then use one HIP runtime)

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    out = tmp_path_factory.mktemp("plan") / "block_plan"
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-O1", "-std=c++17", f"-I{ROOT / 'include'}",
                    f"-I{ROOT / 'xgboost-metal_amd' / 'csrc'}", "-o", str(out), str(ROOT / "tests" / "block_plan.cpp")],
                   check=True)

    def run(*args):
        done = subprocess.run([str(out), *args], capture_output=True, text=True, check=False)
        assert done.returncode == 0, done
        return done.stdout.split()
    return run


def test_every_depth_has_shares(plan):
    assert plan("shares") == ["plans", str(8 * 8192), "wrong", "0"]


def test_scales_are_read_within_their_rows(plan):
    """Shares that begin at any step: the words that hold their scales, no byte behind the
    last row, and every byte where its lanes look for it."""
    out = plan("scales")
    assert int(out[1]) > 1000 and out[2:] == ["wrong", "0"], out


def test_scales_are_read_within_the_panel(plan):
    assert plan("ahead") == ["reads", str(64 * 65 // 2), "wrong", "0"]


def test_every_number_of_rows_can_be_launched(plan):
    out = plan("launches")
    assert int(out[1]) > 2000 and out[2:] == ["wrong", "0"], out


@pytest.mark.parametrize("blocks", [4096, 4097, 8192])
def test_workspaces_of_long_rows(plan, blocks):
    """The entries' own answers for the longest rows that they take."""
    assert plan("shares")[-1] == "0"  # (a size without a plan would end this process)
    import xgboost.core as core
    from test_arguments_block import HERE, Blocks, Matmul, Serve
    lib = ctypes.CDLL(core._LIB.path)
    for name in ("block_matmul", "block_feed_forward"):
        getattr(lib, f"mgb_{name}_workspace_bytes").restype = ctypes.c_size_t

    def matrix(rows, blocks):
        return Blocks(HERE, HERE, rows, blocks, blocks * 128, (blocks + 3) // 4 * 4)

    for dtype in (1, 2):
        m = Matmul(HERE, matrix(64, blocks), matrix(64, blocks), dtype)
        shares = -(-blocks // 64)
        assert lib.mgb_block_matmul_workspace_bytes(ctypes.byref(m)) >= shares * 64 * 64 * 4
        hidden = (blocks - 1) * 128 + 1
        s = Serve(HERE, HERE, matrix(hidden, 1), matrix(hidden, 1), matrix(64, blocks), 40, 64, hidden, 64, 0, dtype)
        assert lib.mgb_block_feed_forward_workspace_bytes(ctypes.byref(s)) >= shares * 40 * 64 * 4 + 40 * hidden
