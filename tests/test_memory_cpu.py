"""Argument checks of the memory operators' C entry points and the Python layer,
without a GPU: every refusal here comes before any launch."""

from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def jl():
    from junqi_amd import _lib
    return _lib


def _args(jl, **over):
    a = jl.Attention(jl.F32, 2, 3, 1, 8, 8, 1.0, 64)
    for n in ("q", "k", "v", "out", "d_out", "dq", "dk", "dv"):
        setattr(a, n, jl.Rows(64, 24, 8, 8))
    for n, x in over.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("over", [{"dtype": 2}, {"batch": -1}, {"plies": -1}, {"heads": 0}, {"key_dim": 0}, {"key_dim": 129},
                                  {"value_dim": 129}, {"log_decay": None}, {"batch": 1 << 30, "heads": 1 << 10},
                                  {"plies": 2 ** 31 - 1}])
def test_attention_arguments(jl, over):
    a = _args(jl, **over)
    assert jl.lib.jq_attention_forward(C.byref(a), None) == jl.JQ_E_ARG
    assert jl.lib.jq_attention_backward(C.byref(a), None) == jl.JQ_E_ARG


@pytest.mark.parametrize("name", ["q", "k", "v", "out"])
def test_attention_pointers(jl, name):
    for rows in (jl.Rows(), jl.Rows(66, 24, 8, 8)):
        a = _args(jl, **{name: rows})
        assert jl.lib.jq_attention_forward(C.byref(a), None) == jl.JQ_E_ARG
        assert name.encode() in jl.lib.jq_last_error()


def test_attention_gradients_go_together(jl):
    for over in ({"dk": jl.Rows()}, {"dv": jl.Rows()}, {"dk": jl.Rows(), "dv": jl.Rows(), "d_initial": 64}, {"d_out": jl.Rows()}):
        assert jl.lib.jq_attention_backward(C.byref(_args(jl, **over)), None) == jl.JQ_E_ARG
    assert jl.lib.jq_attention_forward(None, None) == jl.JQ_E_ARG
    assert jl.lib.jq_attention_workspace(C.byref(_args(jl)), 0, None) == jl.JQ_E_ARG


def test_workspaces(jl):
    """Small and wide segments take none; sizes do not overflow."""
    n = C.c_int64(-1)
    assert jl.lib.jq_attention_workspace(C.byref(_args(jl)), 1, C.byref(n)) == jl.JQ_OK and n.value == 0
    assert jl.lib.jq_layer_norm_workspace(1 << 30, 1 << 20, C.byref(n)) == jl.JQ_OK and n.value > 0
    assert jl.lib.jq_layer_norm_workspace(-1, 4, C.byref(n)) == jl.JQ_E_ARG
    assert jl.lib.jq_layer_norm_workspace(4, 0, C.byref(n)) == jl.JQ_E_ARG


def test_step_arguments(jl):
    r = jl.Rows(64, 8, 0, 8)
    ok = dict(dtype=jl.F32, batch=2, heads=1, dk=8, dv=8, scale=1.0, ld=64, q=r, k=r, v=r, out=r, state=64, n=2, rows=None, st=None)
    for over in ({"dtype": 5}, {"batch": -1}, {"heads": 0}, {"dk": 129}, {"dv": 0}, {"ld": None}, {"q": jl.Rows()}, {"n": -1},
                 {"state": None}, {"state": 66}, {"out": jl.Rows(65)}):
        assert jl.lib.jq_attention_step(*{**ok, **over}.values(), None) == jl.JQ_E_ARG, over


def test_rotary_arguments(jl):
    r = jl.Rows(64, 8, 8, 8)
    ok = dict(dtype=jl.BF16, n0=1, n1=2, heads=1, dim=8, pairs=4, x=r, out=r, pos=64, p64=0, p0=4, p1=2, axes=2,
              ends=(C.c_int32 * 2)(2, 4), f=64, inter=0, inv=0)
    for over in ({"dtype": -1}, {"n0": -1}, {"dim": 7}, {"pairs": 5}, {"pairs": -1}, {"axes": 0}, {"axes": 5},
                 {"ends": (C.c_int32 * 2)(3, 2)}, {"ends": (C.c_int32 * 2)(2, 3)}, {"ends": (C.c_int32 * 2)(-1, 4)},
                 {"ends": None}, {"pos": None}, {"f": None}, {"x": jl.Rows()}, {"out": jl.Rows(65)}, {"pos": 66},
                 {"n0": 1 << 40, "n1": 1 << 10}):
        assert jl.lib.jq_rotary(*{**ok, **over}.values(), None) == jl.JQ_E_ARG, over


def test_norm_arguments(jl):
    ok = dict(dtype=jl.BF16, wdtype=jl.F32, rows=2, width=8, x=64, xs=8, w=None, b=None, eps=1e-5, out=64, os=8, mean=None, rstd=None)
    for over in ({"dtype": 3}, {"wdtype": 3}, {"dtype": jl.F32, "wdtype": jl.BF16}, {"rows": -1}, {"rows": 1 << 40}, {"width": 0},
                 {"x": None}, {"out": None}, {"x": 65}):
        assert jl.lib.jq_layer_norm_forward(*{**ok, **over}.values(), None) == jl.JQ_E_ARG, over
    ok = dict(dtype=jl.BF16, wdtype=jl.F32, rows=2, width=8, x=64, xs=8, w=None, mean=64, rstd=64, d=64, ds=8, dx=64, dxs=8, dw=64,
              db=64, work=64, bytes=1 << 20)
    for over in ({"mean": None}, {"rstd": None}, {"d": None}, {"bytes": 8}, {"work": None}, {"work": 66}, {"dx": 65}, {"width": -1}):
        assert jl.lib.jq_layer_norm_backward(*{**ok, **over}.values(), None) == jl.JQ_E_ARG, over


def test_python_layer_refuses_host_tensors():
    from junqi_amd import memory
    q = torch.zeros(2, 5, 3, 8)
    for call in (lambda: memory.linear_attention(q, q, q, torch.zeros(3)),
                 lambda: memory.linear_attention_step(q[0], q[0], q[0], torch.zeros(3), torch.zeros(5, 3, 8, 8)),
                 lambda: memory.rotary(q, torch.zeros(2, 5, 1, dtype=torch.int32), torch.zeros(4), (4,)),
                 lambda: memory.layer_norm(q)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_frequencies():
    from junqi_amd import memory
    f = memory.rotary_frequencies((4, 2), base=16.0)
    assert f.dtype == torch.float32
    assert f.tolist() == [1.0, 0.5, 0.25, 0.125, 1.0, 0.25]
