"""Argument checks of the selective operators' and the masked logits' C entry points and
Python layer, without a GPU: every refusal here comes before any launch."""

from __future__ import annotations

import ctypes as C

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def jl():
    from junqi_amd import _lib
    return _lib


def _scan(jl, **over):
    s = jl.Scan(jl.F32, 2, 3, 8, 4, 2, 1, 64)
    for n in ("u", "delta", "out", "b", "c", "d_out", "du", "ddelta", "db", "dc"):
        setattr(s, n, jl.Rows(64, 24, 8, 4))
    s.saved, s.workspace, s.workspace_bytes = 64, 64, 1 << 30
    for n, x in over.items():
        setattr(s, n, x)
    return s


def _conv(jl, **over):
    v = jl.Conv(jl.F32, jl.F32, 2, 3, 8, 4, 1, 64)
    for n in ("x", "out", "d_out", "dx"):
        setattr(v, n, jl.Rows(64, 24, 8, 0))
    v.dweight, v.workspace, v.workspace_bytes = 64, 64, 1 << 30
    for n, x in over.items():
        setattr(v, n, x)
    return v


def _logits(jl, **over):
    g = jl.Logits(jl.F32, jl.MASK_BYTES, 2, 8, 0, 0, 64, 8)
    g.repetition = 1.0
    for n, x in over.items():
        setattr(g, n, x)
    return g


@pytest.mark.parametrize("over", [
    {"dtype": 2}, {"batch": -1}, {"plies": -1}, {"plies": (1 << 30) + 1}, {"channels": 0}, {"channels": (1 << 20) + 2},
    {"states": 0}, {"states": 65}, {"groups": 0}, {"groups": 3}, {"a": None}, {"batch": 2 ** 31 - 1, "plies": 1 << 30},
    {"workspace": None}, {"workspace_bytes": 8}, {"workspace": 66}])
def test_scan_arguments(jl, over):
    s = _scan(jl, **over)
    if not {"workspace", "workspace_bytes"} & set(over):
        assert jl.lib.jq_scan_forward(C.byref(s), None) == jl.JQ_E_ARG
    assert jl.lib.jq_scan_backward(C.byref(s), None) == jl.JQ_E_ARG


@pytest.mark.parametrize("name", ["u", "delta", "b", "c", "out"])
def test_scan_pointers(jl, name):
    for rows in (jl.Rows(), jl.Rows(66, 24, 8, 4)):
        s = _scan(jl, **{name: rows})
        assert jl.lib.jq_scan_forward(C.byref(s), None) == jl.JQ_E_ARG
        assert name.encode() in jl.lib.jq_last_error()


def test_scan_backward_arguments(jl):
    for over in ({"saved": None}, {"d_out": jl.Rows()}, {"dgate": jl.Rows(64, 24, 8, 0)}, {"du": jl.Rows(66, 24, 8, 0)}):
        assert jl.lib.jq_scan_backward(C.byref(_scan(jl, **over)), None) == jl.JQ_E_ARG, over
    assert jl.lib.jq_scan_forward(None, None) == jl.JQ_E_ARG
    assert jl.lib.jq_scan_workspace(C.byref(_scan(jl)), 0, None) == jl.JQ_E_ARG
    assert jl.lib.jq_scan_saved(C.byref(_scan(jl)), None) == jl.JQ_E_ARG


def test_scan_step_arguments(jl):
    for args, over in (((64, -1, None, None), {}), ((None, 2, None, None), {}), ((66, 2, None, None), {}),
                       ((64, 2, None, None), {"plies": 2}), ((64, 2, None, None), {"plies": 1, "out": jl.Rows()})):
        s = _scan(jl, **{"plies": 1, **over})
        assert jl.lib.jq_scan_step(C.byref(s), *args, None) == jl.JQ_E_ARG, (args, over)


def test_sizes(jl):
    """Workspaces and saved states of the largest calls do not overflow; long axes of few rows take some."""
    n = C.c_int64(-1)
    assert jl.lib.jq_scan_workspace(C.byref(_scan(jl)), 0, C.byref(n)) == jl.JQ_OK and n.value == 0
    assert jl.lib.jq_scan_workspace(C.byref(_scan(jl, plies=4096)), 0, C.byref(n)) == jl.JQ_OK and n.value > 0
    big = _scan(jl, batch=1 << 12, plies=1 << 30, channels=1, groups=1, states=64)
    for backward in (0, 1):
        assert jl.lib.jq_scan_workspace(C.byref(big), backward, C.byref(n)) == jl.JQ_OK and n.value >= 0
    assert jl.lib.jq_scan_saved(C.byref(big), C.byref(n)) == jl.JQ_OK and n.value == (1 << 39) * 64 * 4
    assert jl.lib.jq_conv_workspace(C.byref(_conv(jl)), C.byref(n)) == jl.JQ_OK and n.value == 5 * 8 * 4
    assert jl.lib.jq_logits_workspace(C.byref(_logits(jl)), C.byref(n)) == jl.JQ_OK and n.value >= 8 * 4


@pytest.mark.parametrize("over", [
    {"dtype": 2}, {"weight_dtype": 1}, {"batch": -1}, {"plies": -1}, {"channels": 0}, {"taps": 0}, {"taps": 9}, {"weight": None},
    {"weight": 66}, {"bias": 66}, {"initial_state": 66}, {"workspace": None}, {"workspace_bytes": 8}, {"workspace": 66}])
def test_conv_arguments(jl, over):
    v = _conv(jl, **over)
    if not {"workspace", "workspace_bytes"} & set(over):
        assert jl.lib.jq_conv_forward(C.byref(v), None) == jl.JQ_E_ARG
    assert jl.lib.jq_conv_backward(C.byref(v), None) == jl.JQ_E_ARG


def test_conv_pointers(jl):
    for name in ("x", "out"):
        for rows in (jl.Rows(), jl.Rows(66, 24, 8, 0)):
            assert jl.lib.jq_conv_forward(C.byref(_conv(jl, **{name: rows})), None) == jl.JQ_E_ARG
            assert name.encode() in jl.lib.jq_last_error()
    for over in ({"d_out": jl.Rows()}, {"dx": jl.Rows(66, 24, 8, 0)}, {"d_final": 66}, {"d_initial": 66}, {"dweight": 66}, {"dbias": 66}):
        assert jl.lib.jq_conv_backward(C.byref(_conv(jl, **over)), None) == jl.JQ_E_ARG, over
    for args, over in (((64, -1, None, None), {}), ((None, 2, None, None), {}), ((66, 2, None, None), {}), ((64, 2, None, None), {"plies": 3})):
        assert jl.lib.jq_conv_step(C.byref(_conv(jl, **{"plies": 1, **over})), *args, None) == jl.JQ_E_ARG
    assert jl.lib.jq_conv_workspace(C.byref(_conv(jl)), None) == jl.JQ_E_ARG


@pytest.mark.parametrize("over", [
    {"dtype": 3}, {"rows": -1}, {"rows": 1 << 31}, {"actions": 0}, {"actions": 2 ** 31 - 1}, {"recent_count": -1}, {"recent_count": 2},
    {"recent": 66, "recent_count": 2}, {"recent": 68, "recent_count": 2, "recent64": 1}, {"mask": 64, "mask_kind": 2},
    {"mask": 66, "mask_kind": 0}, {"bias": 66}, {"logits": 66}])
def test_logits_arguments(jl, over):
    g = _logits(jl, **over)
    assert jl.lib.jq_logits_forward(C.byref(g), 64, 8, None) == jl.JQ_E_ARG
    assert jl.lib.jq_logits_backward(C.byref(g), 64, 8, 64, 8, None, None, 0, None) == jl.JQ_E_ARG


def test_logits_pointers(jl):
    g = C.byref(_logits(jl))
    assert jl.lib.jq_logits_forward(g, None, 8, None) == jl.JQ_E_ARG
    assert jl.lib.jq_logits_forward(g, 66, 8, None) == jl.JQ_E_ARG
    assert jl.lib.jq_logits_forward(C.byref(_logits(jl, logits=None)), 64, 8, None) == jl.JQ_E_ARG
    for args in ((None, 8, 64, 8, None, None, 0), (66, 8, 64, 8, None, None, 0), (64, 8, 66, 8, None, None, 0),
                 (64, 8, 64, 8, 64, None, 1 << 20), (64, 8, 64, 8, 64, 64, 8), (64, 8, 64, 8, 64, 66, 1 << 20)):
        assert jl.lib.jq_logits_backward(g, *args, None) == jl.JQ_E_ARG, args


def test_python_layer_refuses_host_tensors():
    from junqi_amd import masks, memory
    u, n = torch.zeros(2, 5, 8), torch.zeros(2, 5, 4)
    for call in (lambda: memory.selective_scan(u, u, torch.zeros(8, 4), n, n),
                 lambda: memory.selective_scan_step(u[0], u[0], torch.zeros(8, 4), n[0], n[0], torch.zeros(5, 8, 4)),
                 lambda: memory.causal_conv(u, torch.zeros(8, 4)),
                 lambda: memory.causal_conv_step(u[0], torch.zeros(8, 4), torch.zeros(5, 3, 8)),
                 lambda: masks.action_logits(torch.zeros(2, 8))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_python_layer():
    """Tensors without memory behind them: a call that is not refused ends at their data."""
    from torch._subclasses import FakeTensorMode

    from junqi_amd import masks, memory
    far, bf = 2 ** 32 + 2, torch.bfloat16
    with FakeTensorMode():
        def z(*shape, dt=torch.float32, grad=False):
            return torch.empty(shape, dtype=dt, device="cuda", requires_grad=grad)

        def scan(u=(2, 5, 8), delta=None, a=(8, 4), b=(2, 5, 4), c=None, dt=torch.float32, **more):
            return memory.selective_scan(z(*u, dt=dt), z(*(delta or u), dt=dt), z(*a), z(*b, dt=dt), z(*(c or b), dt=dt), **more)

        def scan_step(state=(5, 8, 4), **more):
            return memory.selective_scan_step(z(5, 8), z(5, 8), z(8, 4), z(5, 4), z(5, 4), z(*state), **more)

        def conv(x=(2, 5, 8), w=(8, 4), dt=torch.float32, wdt=torch.float32, **more):
            return memory.causal_conv(z(*x, dt=dt), z(*w, dt=wdt), **more)

        def conv_step(state=(5, 3, 8), **more):
            return memory.causal_conv_step(z(5, 8), z(8, 4), z(*state), **more)

        def logits(shape=(4, 70), dt=torch.float32, **more):
            return masks.action_logits(z(*shape, dt=dt), **more)
        calls = (
            # sizes that do not fit
            lambda: scan(u=(far, 5, 8), b=(far, 5, 4)), lambda: scan(u=(2, far, 8), b=(2, far, 4)),
            lambda: scan(u=(2, 5, far), a=(far, 4)), lambda: scan(u=(2, 5, 0), a=(0, 4)), lambda: conv(x=(far, 5, 8)),
            lambda: conv(x=(2, far, 8)), lambda: conv(x=(2, 5, far), w=(far, 4)), lambda: logits((far, 70)), lambda: logits((4, far)),
            lambda: logits((4, 0)),
            # shapes
            lambda: scan(u=(5, 8)), lambda: scan(delta=(2, 5, 7)), lambda: scan(a=(8, 5)), lambda: scan(b=(2, 4, 4)), lambda: scan(c=(2, 5, 5)),
            lambda: scan(b=(2, 5, 3, 4)), lambda: scan(b=(2, 5, 0, 4)), lambda: scan(a=(8, 65), b=(2, 5, 65)), lambda: scan(a=(8, 0), b=(2, 5, 0)),
            lambda: scan(gate=z(2, 5, 7)), lambda: scan(skip=z(7)), lambda: scan(delta_bias=z(7)), lambda: scan(initial_state=z(2, 8, 5)),
            lambda: scan(starts=z(2, 4, dt=torch.bool)), lambda: scan(lengths=z(3, dt=torch.int32)),
            lambda: conv(w=(7, 4)), lambda: conv(w=(8, 9)), lambda: conv(w=(8, 0)), lambda: conv(bias=z(7)), lambda: conv(initial_state=z(2, 4, 8)),
            lambda: conv(x=(2, 8)), lambda: logits(bias=z(69)), lambda: logits(legal=z(4, 69, dt=torch.bool)),
            lambda: logits(legal=z(4, 2, dt=torch.int32)), lambda: logits(recent=z(3, 5, dt=torch.int32)), lambda: logits(recent=z(4, dt=torch.int32)),
            lambda: logits(recent_lengths=z(4, dt=torch.int32)), lambda: logits(recent=z(4, 5, dt=torch.int32), recent_lengths=z(5, dt=torch.int32)),
            lambda: logits((4,)), lambda: logits(repetition=z(5)),
            # types
            lambda: scan(dt=torch.float16), lambda: scan(gate=z(2, 5, 8, dt=bf)), lambda: scan(skip=z(8, dt=bf)), lambda: scan(dt=bf, initial_state=z(2, 8, 4, dt=bf)),
            lambda: scan(starts=z(2, 5)), lambda: scan(lengths=z(2)), lambda: conv(wdt=bf), lambda: conv(dt=bf, wdt=bf, bias=z(8)),
            lambda: conv(dt=bf, initial_state=z(2, 3, 8)), lambda: logits(dt=torch.float16), lambda: logits(legal=z(4, 70, dt=torch.uint8)),
            lambda: logits(bias=z(70, dt=bf), dt=bf), lambda: logits(recent=z(4, 5)), lambda: logits(recent=z(4, 5, dt=torch.int32), recent_lengths=z(4, dt=torch.int64)),
            # numbers
            lambda: logits(repetition=0.0), lambda: logits(repetition=-1.0), lambda: logits(presence=float("inf")), lambda: logits(frequency=float("nan")),
            # steps
            lambda: scan_step(state=(4, 8, 4)), lambda: scan_step(state=(5, 8, 5)), lambda: scan_step(rows=z(5, dt=torch.int32)), lambda: scan_step(rows=z(4, dt=torch.int64)),
            lambda: scan_step(starts=z(5)), lambda: scan_step(out=z(5, 7)), lambda: scan_step(out=z(5, 8, dt=bf)), lambda: scan_step(out=z(1, 8).expand(5, 8)),
            lambda: scan_step(out=z(8, 5).t()), lambda: scan_step(out=z(5, 8, grad=True)), lambda: scan_step(gate=z(5, 8, grad=True)),
            lambda: memory.selective_scan_step(z(5, 8), z(5, 8), z(8, 4), z(5, 4), z(5, 4), z(8, 4, 5).permute(2, 0, 1)),
            lambda: conv_step(state=(4, 3, 8)), lambda: conv_step(state=(5, 4, 8)), lambda: conv_step(bias=z(8, grad=True)), lambda: conv_step(out=z(1, 8).expand(5, 8)),
            lambda: conv_step(rows=z(5, dt=torch.int32)),
        )
        for i, call in enumerate(calls):
            with pytest.raises(ValueError):
                call()
                print("not refused:", i)
