"""Sizes past what the memory operators' kernels index are refused before any launch, by the C
entry points and, where these could not even be told of them, by the Python layer. No GPU."""

from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

INT_MAX = 2 ** 31 - 1
WIDEST = INT_MAX - 1024   # the columns of a row are walked 1,024 at a time


@pytest.fixture(scope="module")
def jl():
    from junqi_amd import _lib
    return _lib


@pytest.mark.parametrize("width", [INT_MAX, INT_MAX - 1, INT_MAX - 7, WIDEST + 1])
@pytest.mark.parametrize("dtype", ["F32", "BF16"])
def test_norm_widths(jl, width, dtype):
    n, dt = C.c_int64(), getattr(jl, dtype)
    assert jl.lib.jq_layer_norm_workspace(2, width, C.byref(n)) == jl.JQ_E_ARG
    assert jl.lib.jq_layer_norm_forward(dt, jl.F32, 2, width, 64, width, None, None, 1e-5, 64, width, None, None, None) == jl.JQ_E_ARG
    assert jl.lib.jq_layer_norm_backward(dt, jl.F32, 2, width, 64, width, None, 64, 64, 64, width, 64, width, None, None, None, 0,
                                         None) == jl.JQ_E_ARG
    assert jl.lib.jq_layer_norm_workspace(2, WIDEST, C.byref(n)) == jl.JQ_OK and n.value == 2 * 4 * WIDEST


def test_the_python_layer():
    """Tensors without memory behind them: a call that is not refused for its sizes ends at their data."""
    from torch._subclasses import FakeTensorMode

    from junqi_amd import memory
    with FakeTensorMode():
        def z(*shape, dt=torch.float32):
            return torch.empty(shape, dtype=dt, device="cuda")
        far = 2 ** 32 + 2     # 2, in 32 bits
        ld = z(1)

        def attention(b, t, h):
            return memory.linear_attention(z(b, t, h, 4), z(b, t, h, 4), z(b, t, h, 4), ld if h == 1 else z(h))

        def step(b, h):
            return memory.linear_attention_step(z(b, h, 4), z(b, h, 4), z(b, h, 4), ld if h == 1 else z(h), z(b, h, 4, 4))

        def rotary(heads, dim):
            return memory.rotary(z(3, heads, dim), z(3, 1, dt=torch.int32), z(2), (2,))
        for call in (lambda: attention(far, 3, 1), lambda: attention(2, far, 1), lambda: attention(2, 3, far),
                     lambda: attention(2, INT_MAX, 1), lambda: attention(1 << 12, 2, 1 << 11),
                     lambda: step(far, 1), lambda: step(2, far), lambda: step(1 << 13, 1 << 10),
                     lambda: rotary(far, 4), lambda: rotary(2, far), lambda: rotary(1 << 16, 1 << 15),
                     lambda: memory.layer_norm(z(3, far)), lambda: memory.layer_norm(z(3, INT_MAX))):
            with pytest.raises(ValueError, match="too (large|many|wide)|out of range"):
                call()
