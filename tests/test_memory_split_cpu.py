"""Which calls of linear attention split a long axis: those whose games and heads, a block
each, leave the card's 256 CUs idle. A split needs workspace, so the size of that tells.
No GPU."""

from __future__ import annotations

import ctypes as C

import pytest

pytest.importorskip("torch")


@pytest.fixture(scope="module")
def jl():
    from junqi_amd import _lib
    return _lib


def _segments(jl, dtype, batch, plies, heads, key_dim, value_dim):
    a = jl.Attention(dtype, batch, plies, heads, key_dim, value_dim, 1.0, 64)
    n = C.c_int64(-1)
    assert jl.lib.jq_attention_workspace(C.byref(a), 0, C.byref(n)) == jl.JQ_OK
    each = batch * heads * (key_dim * value_dim + 1) * 4
    assert n.value % each == 0
    return n.value // each


@pytest.mark.parametrize("dim", [20, 32, 64, 100, 128])
def test_few_blocks_are_split_at_any_width(jl, dim):
    for heads in (1, 8, 32, 63, 64, 65, 128):
        for dtype in (jl.F32, jl.BF16):
            assert _segments(jl, dtype, 1, 8192, heads, dim, dim) >= 4, (heads, dtype)
    assert _segments(jl, jl.BF16, 8, 16000, 8, dim, dim) >= 4


@pytest.mark.parametrize("dim,most", [(20, 511), (32, 511), (40, 255), (64, 255), (100, 128), (128, 128)])
def test_blocks_that_fill_the_card_are_not(jl, dim, most):
    for dtype in (jl.F32, jl.BF16):
        assert _segments(jl, dtype, most, 8192, 1, dim, dim) >= 4
        for batch, heads in ((most + 1, 1), (64, 8), (256, 4)):
            assert _segments(jl, dtype, batch, 8192, heads, dim, dim) == 0, (batch, heads, dtype)


def test_short_axes_are_not(jl):
    for dtype, chunk in ((jl.F32, 16), (jl.BF16, 32)):
        assert _segments(jl, dtype, 2, 15 * chunk, 2, 64, 64) == 0
        assert _segments(jl, dtype, 2, 16 * chunk, 2, 64, 64) == 4


def test_short_axes_of_many_wide_blocks_are_not(jl):
    """Two more launches and states between cost more than a few chunks a block save."""
    for dtype, plies in ((jl.BF16, 512), (jl.F32, 256)):
        for heads in (65, 96, 128):
            assert _segments(jl, dtype, 1, plies, heads, 128, 100) == 0, (heads, dtype)
            assert _segments(jl, dtype, 1, 2 * plies, heads, 128, 100) >= 4, (heads, dtype)
        for heads, dim in ((64, 128), (255, 64), (255, 32)):
            assert _segments(jl, dtype, 1, plies, heads, dim, dim) == 4, (heads, dim, dtype)
