"""What the selective operators and the masked logits refuse, beside test_selective_cpu.py:
without a GPU, every refusal comes before any launch."""

from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def jl():
    from junqi_amd import _lib
    return _lib


@pytest.mark.parametrize("name,number", [("frequency", 1e39), ("presence", -1e39), ("repetition", 1e39), ("repetition", 1e-50),
                                         ("repetition", 3.4028236e38), ("frequency", float("-inf")), ("repetition", 7e-46)])
def test_penalties_that_float32_does_not_hold(name, number):
    """They would reach the kernel as an infinity, or as a repetition of 0."""
    from torch._subclasses import FakeTensorMode

    from junqi_amd import masks
    with FakeTensorMode():      # a call that is not refused ends at the data, with another error
        x = torch.empty(4, 70, device="cuda")
        recent = torch.empty(4, 5, dtype=torch.int32, device="cuda")
        with pytest.raises(ValueError, match=name):
            masks.action_logits(x, recent=recent, **{name: number})


def _scan(jl, **over):
    s = jl.Scan(jl.F32, 2, 3, 8, 4, 2, 1, 64)
    for n in ("u", "delta", "out", "b", "c", "d_out", "du", "ddelta", "db", "dc"):
        setattr(s, n, jl.Rows(64, 24, 8, 4))
    s.saved, s.workspace, s.workspace_bytes = 64, 64, 1 << 30
    for n, x in over.items():
        setattr(s, n, x)
    return s


@pytest.mark.parametrize("name", ["a", "skip", "delta_bias", "lengths", "initial_state", "final_state", "saved"])
def test_scan_forward_alignment(jl, name):
    assert jl.lib.jq_scan_forward(C.byref(_scan(jl, **{name: 66})), None) == jl.JQ_E_ARG
    assert name.encode() in jl.lib.jq_last_error()


@pytest.mark.parametrize("name", ["a", "skip", "delta_bias", "lengths", "saved", "da", "dskip", "ddelta_bias", "d_final", "d_initial"])
def test_scan_backward_alignment(jl, name):
    assert jl.lib.jq_scan_backward(C.byref(_scan(jl, **{name: 66})), None) == jl.JQ_E_ARG
    assert name.encode() in jl.lib.jq_last_error()


def test_step_alignment(jl):
    for name in ("a", "skip", "delta_bias"):
        assert jl.lib.jq_scan_step(C.byref(_scan(jl, plies=1, **{name: 66})), 64, 2, None, None, None) == jl.JQ_E_ARG
        assert name.encode() in jl.lib.jq_last_error()
    assert jl.lib.jq_scan_step(C.byref(_scan(jl, plies=1)), 64, 2, 68, None, None) == jl.JQ_E_ARG
    assert b"rows" in jl.lib.jq_last_error()
    v = jl.Conv(jl.F32, jl.F32, 2, 1, 8, 4, 1, 64)
    v.x = v.out = jl.Rows(64, 8, 8, 0)
    assert jl.lib.jq_conv_step(C.byref(v), 64, 2, 68, None, None) == jl.JQ_E_ARG
    assert b"rows" in jl.lib.jq_last_error()


def test_conv_lengths_alignment(jl):
    v = jl.Conv(jl.F32, jl.F32, 2, 3, 8, 4, 1, 64)
    v.x = v.out = v.d_out = v.dx = jl.Rows(64, 24, 8, 0)
    v.lengths = 66
    assert jl.lib.jq_conv_forward(C.byref(v), None) == jl.JQ_E_ARG and b"lengths" in jl.lib.jq_last_error()
    assert jl.lib.jq_conv_backward(C.byref(v), None) == jl.JQ_E_ARG and b"lengths" in jl.lib.jq_last_error()


@pytest.mark.parametrize("name", ["recent_lengths", "repetitions", "frequencies", "presences"])
def test_logits_alignment(jl, name):
    g = jl.Logits(jl.F32, jl.MASK_BYTES, 2, 8, 3, 0, 64, 8)
    g.repetition, g.recent, g.recent_stride = 1.0, 64, 3
    setattr(g, name, 66)
    assert jl.lib.jq_logits_forward(C.byref(g), 64, 8, None) == jl.JQ_E_ARG and name.encode() in jl.lib.jq_last_error()
    assert jl.lib.jq_logits_backward(C.byref(g), 64, 8, 64, 8, None, None, 0, None) == jl.JQ_E_ARG and name.encode() in jl.lib.jq_last_error()


def test_logits_bias_gradient_alignment(jl):
    g = jl.Logits(jl.F32, jl.MASK_BYTES, 2, 8, 0, 0, 64, 8)
    g.repetition = 1.0
    assert jl.lib.jq_logits_backward(C.byref(g), 64, 8, 64, 8, 66, 64, 1 << 20, None) == jl.JQ_E_ARG
    assert b"d_bias" in jl.lib.jq_last_error()


@pytest.mark.parametrize("stride,good", [(0, False), (1, False), (7, False), (8, True), (9, True)])
def test_rows_of_out_that_share_memory(stride, good):
    """Games that write the same elements would race; rows apart, or one game, go on to the call."""
    from torch._subclasses import FakeTensorMode

    from junqi_amd import memory
    with FakeTensorMode():
        def z(*shape):
            return torch.empty(shape, device="cuda")
        out = z(64).as_strided((5, 8), (stride, 1))
        for call in (lambda o, b: memory.selective_scan_step(z(b, 8), z(b, 8), z(8, 4), z(b, 4), z(b, 4), z(b, 8, 4), out=o),
                     lambda o, b: memory.causal_conv_step(z(b, 8), z(8, 4), z(b, 3, 8), out=o)):
            for o, b, ok in ((out, 5, good), (out[:1], 1, True)):
                with pytest.raises(Exception) as e:     # without a GPU every call ends somewhere
                    call(o, b)
                assert ("share memory" in str(e.value)) != ok
