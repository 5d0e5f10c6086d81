"""Matrices in blocks whose rows' lengths do not fit are refused, whole blocks of padding
or not (no GPU needed: before any device work)."""
import pytest
import torch


@pytest.fixture(scope="module")
def enc():
    from xgboost import encoder
    return encoder


def _matrix(enc, rows, dim):
    blocks = -(-dim // 128)
    return enc.BlockScaled(torch.zeros(rows, blocks * 128, dtype=torch.uint8).view(torch.float8_e4m3fn),
                           torch.full((rows, blocks), 127, dtype=torch.uint8).view(torch.float8_e8m0fnu), dim)


@pytest.mark.parametrize("name,sizes", [
    ("gate", dict(gate=(200, 200))), ("gate", dict(gate=(200, 251))), ("up", dict(up=(200, 249))),
    ("down", dict(down=(250, 250))), ("down", dict(down=(250, 199))), ("gate", dict(x=200)), ("down", dict(gate=(201, 250), up=(201, 250)))])
def test_served_lengths(enc, name, sizes):
    sizes = {**dict(x=250, gate=(200, 250), up=(200, 250), down=(250, 200)), **sizes}
    x = torch.zeros(4, sizes["x"])
    with pytest.raises(ValueError, match=f"{name} must have rows of"):
        enc.block_feed_forward(x, *(_matrix(enc, *sizes[m]) for m in ("gate", "up", "down")))


def test_lengths_that_blocks_do_not_have(enc):
    """A length that is not that of the values' blocks."""
    m = _matrix(enc, 200, 250)
    for dim in (0, -5, 128, 257, 10_000):
        with pytest.raises(ValueError, match="rows of 2 blocks do not hold"):
            enc.block_matmul(m._replace(dim=dim), m._replace(dim=dim))
