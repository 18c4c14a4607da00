"""The selective scan and the causal convolution (junqi_amd.memory) on an MI355X against
their definitions in 64 bits (tests/selective_oracle.py, which has the tolerances)."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import selective_oracle as O  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def memory():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import memory as M
    return M


def _cpu(x):
    """The inputs of a case for the definition."""
    return {k: v.detach().cpu().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else
            v.cpu() if isinstance(v, torch.Tensor) else v for k, v in x.items()}


def _masks(g, b, t, starts, lengths):
    s = {"none": None, "some": torch.rand(b, t, generator=g) < 0.1, "all": torch.ones(b, t, dtype=torch.bool)}[starts]
    n = None
    if lengths == "some":
        n = torch.randint(-1, t + 3, (b,), generator=g, dtype=torch.int32)
        n[:4] = torch.tensor([t, 0, 1, t + 9], dtype=torch.int32)[:b]
    return None if s is None else s.cuda(), None if n is None else n.cuda()


def _scan_inputs(seed, b, t, d, n, groups, dtype=F32, starts="some", lengths="some", state=True, gate=True, skip=True,
                 bias=True, softplus=True, time_major=False):
    g = torch.Generator().manual_seed(seed)

    def rows(*last, scale=1.0):
        x = (scale * torch.randn(*((t, b) if time_major else (b, t)), *last, generator=g)).to(dtype).cuda()
        return x.transpose(0, 1) if time_major else x

    def f32(*shape):
        return torch.randn(*shape, generator=g).cuda()
    x = {"u": rows(d), "delta": rows(d, scale=0.5), "gate": rows(d) if gate else None, "b": rows(groups, n), "c": rows(groups, n),
         "a": -(0.5 + torch.rand(d, n, generator=g) * n).cuda(), "skip": f32(d) if skip else None,
         "delta_bias": f32(d) - 3.0 if bias else None, "softplus": softplus, "state": f32(b, d, n) if state else None,
         "d_out": rows(d), "d_state": f32(b, d, n) if state else None}
    if not softplus:   # steps as they are
        x["delta"] = (0.1 * x["delta"].abs()).to(dtype)
        x["delta_bias"] = 0.01 * f32(d).abs() if bias else None
    x["starts"], x["lengths"] = _masks(g, b, t, starts, lengths)
    return x


SCAN_LEAVES = ("u", "delta", "a", "b", "c", "skip", "gate", "delta_bias", "state")


def _run_scan(memory, x, grads=True):
    leaves = {k: x[k].detach().requires_grad_(grads) for k in SCAN_LEAVES if x[k] is not None}
    p = {**x, **leaves}
    out, state = memory.selective_scan(p["u"], p["delta"], p["a"], p["b"], p["c"], skip=p["skip"], gate=p["gate"],
                                       delta_bias=p["delta_bias"], softplus=x["softplus"], starts=x["starts"],
                                       lengths=x["lengths"], initial_state=p["state"], return_state=True)
    got = {"out": out, "state": state}
    if grads:
        res = ([out, state], [x["d_out"], x["d_state"]]) if x["d_state"] is not None else ([out], [x["d_out"]])
        got.update(zip(("d_" + k for k in leaves), torch.autograd.grad(res[0], list(leaves.values()), res[1])))
    return got


def _check_scan(memory, x, grads=True, floor=1e-36):
    c = _cpu(x) if grads else {**_cpu(x), "d_out": None}
    want, size, steps = O.scan(c), O.scan(c, size=True), O.scan_roundings(c)
    got = _run_scan(memory, x, grads)
    for k, v in got.items():
        leaf = x[k[2:]] if k.startswith("d_") else None
        dtype = x["u"].dtype if k == "out" else F32 if k == "state" else leaf.dtype
        assert v.dtype == dtype, k
        O.close(k, v, want[k], size[k], steps, dtype, floor)
    return got


# games, plies, channels, states, groups
SHAPES = [(1, 1, 1, 1, 1), (4, 2, 5, 3, 1), (3, 9, 64, 16, 1), (4, 17, 130, 16, 2), (5, 8, 64, 4, 1), (2, 33, 70, 8, 2),
          (4, 21, 66, 12, 3), (2, 16, 128, 32, 1), (3, 7, 65, 64, 1), (2, 15, 24, 33, 2), (4, 25, 9, 17, 9), (2, 40, 192, 5, 1)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("masks", [("none", "none", False), ("some", "some", True), ("all", "none", True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_scan(memory, shape, masks, dtype):
    starts, lengths, state = masks
    x = _scan_inputs(hash((shape, starts)) % 1000, *shape, dtype=dtype, starts=starts, lengths=lengths, state=state)
    _check_scan(memory, x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 300, 64, 16, 1), (2, 519, 40, 12, 1), (1, 1030, 3, 1, 1), (3, 260, 66, 24, 2), (1, 777, 64, 64, 1)])
def test_scan_of_long_axes(memory, shape, dtype):
    """Few rows: the axis is split."""
    x = _scan_inputs(7, *shape, dtype=dtype, starts="none", lengths="some" if shape[0] > 2 else "none")
    if shape[0] == 2:    # one game that starts anew in a few places, one that ends inside a part
        x["starts"] = torch.zeros(2, shape[1], dtype=torch.bool, device="cuda")
        x["starts"][0, [0, 130, 131, 400]] = True
        x["lengths"] = torch.tensor([shape[1], 203], dtype=torch.int32, device="cuda")
    _check_scan(memory, x)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("skip", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("softplus", [False, True])
def test_scan_without_its_options(memory, gate, skip, bias, softplus):
    x = _scan_inputs(11, 3, 19, 70, 16, 1, gate=gate, skip=skip, bias=bias, softplus=softplus)
    _check_scan(memory, x)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_orders_and_strides(memory, dtype):
    """Time-major rows, parts of wider rows at odd elements, shared rows."""
    x = _scan_inputs(3, 4, 12, 64, 16, 1, dtype=dtype, time_major=True)
    x["starts"] = x["starts"].t().contiguous().t()
    got = _check_scan(memory, x)
    assert got["out"].stride() == x["u"].stride()
    y = _scan_inputs(4, 3, 13, 66, 16, 2, dtype=dtype)
    for k in ("u", "delta", "gate", "b", "c", "d_out"):
        last = y[k].shape[-1]
        wide = torch.full((*y[k].shape[:-1], last + 3), float("nan"), dtype=dtype, device="cuda")
        wide[..., 1:1 + last] = y[k]
        y[k] = wide[..., 1:1 + last]
    _check_scan(memory, y)
    z = _scan_inputs(5, 3, 13, 66, 16, 2, dtype=dtype)
    z["delta"] = z["delta"][:1].expand(3, -1, -1)
    z["b"] = z["b"][:, :1].expand(-1, 13, -1, -1)
    z["gate"] = z["gate"][..., :1].expand(-1, -1, 66)
    _check_scan(memory, z)
    w = _scan_inputs(6, 2, 9, 64, 16, 1, dtype=dtype)
    w["u"] = w["u"].transpose(1, 2).contiguous().transpose(1, 2)     # elements apart
    _check_scan(memory, w)


def test_scan_of_one_group_without_its_dimension(memory):
    x = _scan_inputs(8, 3, 10, 32, 8, 1)
    out = memory.selective_scan(x["u"], x["delta"], x["a"], x["b"], x["c"], softplus=True)
    flat = memory.selective_scan(x["u"], x["delta"], x["a"], x["b"][:, :, 0], x["c"][:, :, 0], softplus=True)
    assert torch.equal(out, flat)


@pytest.mark.parametrize("shape", [(3, 40, 64, 16, 1), (2, 21, 70, 24, 2), (1, 600, 64, 16, 1)])
def test_what_a_ply_does_not_see_does_not_reach_it(memory, shape):
    """Infinities and NaN before a game's start, behind its length, and in a state that a start discards."""
    b, t, d, n, groups = shape
    x = _scan_inputs(9, *shape, starts="none", lengths="none")
    x["starts"] = torch.zeros(b, t, dtype=torch.bool, device="cuda")
    x["starts"][:, 12] = True
    x["lengths"] = torch.full((b,), t - 5, dtype=torch.int32, device="cuda")
    c = _cpu(x)
    want, size, steps = O.scan(c), O.scan(c, size=True), O.scan_roundings(c)
    y = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    for k in ("u", "b", "gate"):
        y[k][:, 11, ..., :3] = float("inf")
        y[k][:, t - 5:] = float("nan")
    y["delta"][:, 3] = float("nan")
    y["c"][:, t - 5:] = float("nan")
    y["d_out"][:, t - 5:] = float("nan")
    y["state"][:] = float("nan")
    got = _run_scan(memory, y)
    for k in ("out", "state", "d_u", "d_delta", "d_b", "d_c", "d_gate"):
        rows = (slice(None), slice(12, t - 5)) if k not in ("state",) else slice(None)
        O.close(k, got[k][rows], want[k][rows], size[k][rows], steps, F32)
        if k not in ("state",):
            assert not got[k][:, t - 5:].any(), k
    # and what sees an infinity has it
    z = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    z["u"][0, 20, 0] = float("inf")
    want = O.scan({**_cpu(z), "d_out": None})
    got = _run_scan(memory, z, grads=False)
    for k in ("out", "state"):
        assert torch.equal(got[k].cpu().isfinite(), want[k].isfinite()), k
        assert torch.equal(got[k].cpu().isnan(), want[k].isnan()), k


def test_scan_of_far_steps(memory):
    """Steps of 1e-6 and of 80, decays that are 1 and 0 in float32."""
    x = _scan_inputs(13, 2, 12, 64, 16, 1)
    x["delta"][:, :, :20] = -14.0
    x["delta"][:, :, 20:40] = 80.0
    x["delta_bias"].zero_()
    # a decay below 2^-126 counts as 0: a term that has it is off by 2^-126 times its other
    # factors, at most a step (80), a rate (16 states of at most 16.5 each), a state and its
    # gradient, which the plies' terms are summed to; and there are as many terms as plies
    top = {k: v.abs().max().item() for k, v in _cpu(x).items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    plies, step = 2 * 12, 81.0
    h = plies * step * top["u"] * top["b"] + top["state"]
    dh = plies * top["c"] * top["d_out"] * top["gate"] + top["d_state"]
    _check_scan(memory, x, floor=2.0 ** -126 * plies * step * 16 * 16.5 * (top["u"] + 1) * h * dh)
    x["softplus"] = False
    x["delta"] = torch.randn_like(x["delta"])      # steps back: decays above 1
    x["a"] = 0.1 * x["a"]
    x["starts"] = None
    c = _cpu(x)
    want = O.scan(c)
    got = _run_scan(memory, x)
    size = O.scan(c, size=True)
    for k in got:
        O.close(k, got[k], want[k], size[k], O.scan_roundings(c), F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_gradients_that_are_not_wanted(memory, dtype):
    """Each input alone has the gradient that all together have."""
    x = _scan_inputs(15, 3, 20, 70, 16, 2, dtype=dtype)
    both = _run_scan(memory, x)
    for k in SCAN_LEAVES:
        p = {n: x[n].detach() if x[n] is not None else None for n in SCAN_LEAVES}
        p[k] = p[k].requires_grad_()
        out, state = memory.selective_scan(p["u"], p["delta"], p["a"], p["b"], p["c"], skip=p["skip"], gate=p["gate"],
                                           delta_bias=p["delta_bias"], softplus=True, starts=x["starts"], lengths=x["lengths"],
                                           initial_state=p["state"], return_state=True)
        g = torch.autograd.grad([out, state], [p[k]], [x["d_out"], x["d_state"]])[0]
        assert torch.equal(g, both["d_" + k]), k
    # the state's gradient alone
    p = {n: x[n].detach().requires_grad_() for n in SCAN_LEAVES}
    _, state = memory.selective_scan(p["u"], p["delta"], p["a"], p["b"], p["c"], skip=p["skip"], gate=p["gate"],
                                     delta_bias=p["delta_bias"], softplus=True, starts=x["starts"], lengths=x["lengths"],
                                     initial_state=p["state"], return_state=True)
    g = torch.autograd.grad([state], [p["u"], p["state"], p["c"]], [x["d_state"]])
    c = _cpu({**x, "d_out": torch.zeros_like(x["d_out"])})
    want, size = O.scan(c), O.scan(c, size=True)
    for k, v in zip(("d_u", "d_state", "d_c"), g):
        O.close(k, v, want[k], size[k], O.scan_roundings(c), v.dtype)


def test_scan_of_nothing(memory):
    for b, t in ((0, 3), (2, 0), (0, 0)):
        x = _scan_inputs(1, b, t, 8, 4, 2, starts="none", lengths="none")
        got = _run_scan(memory, x)
        assert got["out"].shape == (b, t, 8)
        assert torch.equal(got["state"], x["state"]) and torch.equal(got["d_state"], x["d_state"])
        assert not got["d_a"].any() and not got["d_skip"].any() and not got["d_delta_bias"].any()


def test_scan_is_the_same_every_time(memory):
    for shape in ((5, 100, 200, 16, 1), (1, 700, 70, 24, 2)):
        x = _scan_inputs(21, *shape, dtype=BF16)
        first = _run_scan(memory, x)
        for _ in range(3):
            for k, v in _run_scan(memory, x).items():
                assert torch.equal(v, first[k]), k


# ------------------------------------------------------------------ the scan's step
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (5, 64, 16, 1), (7, 66, 12, 2), (3, 40, 3, 1), (4, 65, 64, 1), (6, 10, 33, 2), (200, 33, 5, 3),
                                   (300, 512, 16, 1)])
@pytest.mark.parametrize("options", [True, False])
def test_scan_step(memory, shape, dtype, options):
    """One ply of each game, then rows of a state of several seats: those of no game stay."""
    b, d, n, groups = shape
    x = _scan_inputs(31, b, 1, d, n, groups, dtype=dtype, starts="some", lengths="none", gate=options, skip=options, bias=options,
                     softplus=options)
    c = {**_cpu(x), "d_out": None}
    want, size, steps = O.scan(c), O.scan(c, size=True), O.scan_roundings(c)
    kw = dict(skip=x["skip"], delta_bias=x["delta_bias"], softplus=options, gate=x["gate"][:, 0] if options else None)
    args = [x[k][:, 0] for k in ("u", "delta")] + [x["a"], x["b"][:, 0], x["c"][:, 0]]
    state = x["state"].clone()
    out = memory.selective_scan_step(*args, state, starts=x["starts"][:, 0], **kw)
    O.close("out", out, want["out"][:, 0], size["out"][:, 0], steps, dtype)
    O.close("state", state, want["state"], size["state"], steps, F32)
    # rows in an order of their own, some of no state
    g = torch.Generator().manual_seed(b)
    rows = torch.randperm(3 * b, generator=g)[:b]
    held = torch.randn(3 * b, d, n, generator=g).cuda()
    held[rows] = x["state"]
    given = rows.clone()
    given[::3] = torch.tensor([-1, 3 * b, 2 ** 40])[torch.arange(len(given[::3])) % 3]
    before, into = held.clone(), torch.full((b, d + 5), 7.0, dtype=dtype, device="cuda")
    out = memory.selective_scan_step(*args, held, starts=x["starts"][:, 0], rows=given.cuda(), out=into[:, 1:1 + d], **kw)
    on = torch.ones(b, dtype=torch.bool)
    on[::3] = False
    O.close("out", out[on.cuda()], want["out"][:, 0][on], size["out"][:, 0][on], steps, dtype)
    assert not out[~on.cuda()].any()
    assert (into[:, 0] == 7).all() and (into[:, 1 + d:] == 7).all()
    O.close("state", held[rows[on].cuda()], want["state"][on], size["state"][on], steps, F32)
    rest = torch.ones(3 * b, dtype=torch.bool)
    rest[rows[on]] = False
    assert torch.equal(held[rest.cuda()], before[rest.cuda()])


def test_steps_follow_the_segment(memory):
    """Plies one by one give the segment's results, and a state that is at an odd address too."""
    x = _scan_inputs(33, 4, 9, 48, 16, 1, lengths="none")
    c = {**_cpu(x), "d_out": None}
    want, size, steps = O.scan(c), O.scan(c, size=True), O.scan_roundings(c)
    raw = torch.empty(x["state"].numel() + 1, device="cuda")
    state = raw[1:].view_as(x["state"]).copy_(x["state"])
    for t in range(9):
        out = memory.selective_scan_step(x["u"][:, t], x["delta"][:, t], x["a"], x["b"][:, t], x["c"][:, t], state, skip=x["skip"],
                                         gate=x["gate"][:, t], delta_bias=x["delta_bias"], softplus=True, starts=x["starts"][:, t])
        O.close("out", out, want["out"][:, t], size["out"][:, t], steps, F32)
    O.close("state", state, want["state"], size["state"], steps, F32)


# ------------------------------------------------------------------ convolution
def _conv_inputs(seed, b, t, d, taps, dtype=F32, wdtype=F32, starts="some", lengths="some", state=True, bias=True, silu=True,
                 time_major=False):
    g = torch.Generator().manual_seed(seed)

    def rows(*last):
        x = torch.randn(*((t, b) if time_major else (b, t)), *last, generator=g).to(dtype).cuda()
        return x.transpose(0, 1) if time_major else x
    x = {"x": rows(d), "weight": torch.randn(d, taps, generator=g).to(wdtype).cuda(), "bias": torch.randn(d, generator=g).to(wdtype).cuda() if bias else None,
         "silu": silu, "state": torch.randn(b, taps - 1, d, generator=g).to(dtype).cuda() if state else None, "d_out": rows(d),
         "d_state": torch.randn(b, taps - 1, d, generator=g).to(dtype).cuda() if state else None}
    x["starts"], x["lengths"] = _masks(g, b, t, starts, lengths)
    return x


CONV_LEAVES = ("x", "weight", "bias", "state")


def _check_conv(memory, x, only=None):
    c = _cpu(x)
    want, size = O.conv(c), O.conv(c, size=True)
    b, t, d = x["x"].shape
    steps = x["weight"].shape[1] + 16      # of a sum and its slope
    sums = steps + b * t                   # of the gradients over all plies
    leaves = {k: x[k].detach().requires_grad_() for k in CONV_LEAVES if x[k] is not None and (only is None or k in only)}
    p = {**x, **leaves}
    out, state = memory.causal_conv(p["x"], p["weight"], p["bias"], silu=x["silu"], starts=x["starts"], lengths=x["lengths"],
                                    initial_state=p["state"], return_state=True)
    O.close("out", out, want["out"], size["out"], steps, x["x"].dtype)
    assert torch.equal(state.double().cpu(), want["state"]), "state"
    res = ([out, state], [x["d_out"], x["d_state"]]) if x["d_state"] is not None else ([out], [x["d_out"]])
    for k, g in zip(leaves, torch.autograd.grad(*[res[0], list(leaves.values()), res[1]])):
        assert g.dtype == x[k].dtype, k
        O.close("d_" + k, g, want["d_" + k], size["d_" + k], sums if k in ("weight", "bias") else steps, x[k].dtype)
    return out


# games, plies, channels, taps
CONV_SHAPES = [(1, 1, 1, 1), (4, 2, 5, 2), (3, 20, 64, 4), (4, 37, 130, 3), (5, 9, 63, 8), (2, 70, 24, 5), (6, 33, 9, 4), (1, 100, 520, 4),
               (2, 50, 7, 7), (4, 17, 513, 6)]


@pytest.mark.parametrize("types", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("masks", [("none", "none", False), ("some", "some", True), ("all", "none", True)])
@pytest.mark.parametrize("shape", CONV_SHAPES)
def test_conv(memory, shape, masks, types):
    starts, lengths, state = masks
    x = _conv_inputs(sum(shape), *shape, dtype=types[0], wdtype=types[1], starts=starts, lengths=lengths, state=state and shape[3] > 1,
                     silu=shape[2] % 2 == 0 or starts == "some")
    _check_conv(memory, x)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_conv_orders_and_strides(memory, dtype):
    x = _conv_inputs(41, 4, 22, 64, 4, dtype=dtype, time_major=True)
    out = _check_conv(memory, x)
    assert out.stride() == x["x"].stride()
    y = _conv_inputs(42, 3, 21, 37, 4, dtype=dtype, bias=False)
    for k in ("x", "d_out"):
        wide = torch.full((3, 21, 40), float("nan"), dtype=dtype, device="cuda")
        wide[..., 1:38] = y[k]
        y[k] = wide[..., 1:38]
    _check_conv(memory, y)
    z = _conv_inputs(43, 3, 21, 36, 3, dtype=dtype)
    z["x"] = z["x"][:1].expand(3, -1, -1)
    z["d_out"] = z["d_out"][:, :1].expand(-1, 21, -1)
    _check_conv(memory, z)
    for k in CONV_LEAVES:
        _check_conv(memory, _conv_inputs(44, 3, 30, 20, 4, dtype=dtype), only=(k,))


def test_what_a_tap_does_not_reach(memory):
    """Infinities and NaN before a start, behind a length and in a discarded state."""
    x = _conv_inputs(45, 3, 40, 36, 4, starts="none", lengths="none")
    x["starts"] = torch.zeros(3, 40, dtype=torch.bool, device="cuda")
    x["starts"][:, [0, 20]] = True
    x["lengths"] = torch.full((3,), 33, dtype=torch.int32, device="cuda")
    clean = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    x["x"][:, 17:20] = float("inf")
    x["x"][:, 33:] = float("nan")
    x["d_out"][:, 33:] = float("nan")
    x["state"][:] = float("nan")
    c = _cpu(clean)
    want, size = O.conv(c), O.conv(c, size=True)
    leaf = x["x"].detach().requires_grad_()
    out, state = memory.causal_conv(leaf, x["weight"], x["bias"], silu=True, starts=x["starts"], lengths=x["lengths"],
                                    initial_state=x["state"], return_state=True)
    dx = torch.autograd.grad([out, state], [leaf], [x["d_out"], x["d_state"]])[0]
    for rows in (slice(0, 17), slice(20, 33)):
        O.close("out", out[:, rows], want["out"][:, rows], size["out"][:, rows], 20, F32)
    O.close("dx", dx[:, 20:33], want["d_x"][:, 20:33], size["d_x"][:, 20:33], 20, F32)
    assert not out[:, 33:].any() and not dx[:, 33:].any()
    assert torch.equal(state.double().cpu(), want["state"])


def test_conv_of_nothing(memory):
    for b, t in ((0, 3), (2, 0)):
        x = _conv_inputs(1, b, t, 8, 4, starts="none", lengths="none")
        leaves = [x[k].requires_grad_() for k in CONV_LEAVES]
        out, state = memory.causal_conv(*leaves[:3], silu=True, initial_state=leaves[3], return_state=True)
        assert out.shape == (b, t, 8) and torch.equal(state, x["state"])
        g = torch.autograd.grad([out, state], leaves, [x["d_out"], x["d_state"]])
        assert not g[1].any() and not g[2].any() and torch.equal(g[3], x["d_state"])


@pytest.mark.parametrize("types", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("shape", [(1, 1, 1), (5, 64, 4), (7, 70, 3), (300, 520, 4), (9, 33, 8), (4, 17, 6), (6, 12, 2)])
def test_conv_step(memory, shape, types):
    b, d, taps = shape
    x = _conv_inputs(51, b, 1, d, taps, dtype=types[0], wdtype=types[1], lengths="none", state=True)
    c = {**_cpu(x), "d_out": None}
    want, size = O.conv(c), O.conv(c, size=True)
    state = x["state"].clone()
    out = memory.causal_conv_step(x["x"][:, 0], x["weight"], state, x["bias"], silu=True, starts=x["starts"][:, 0])
    O.close("out", out, want["out"][:, 0], size["out"][:, 0], taps + 16, types[0])
    # the state after a ply that starts a game holds that ply alone
    assert torch.equal(state.double().cpu(), want["state"])
    g = torch.Generator().manual_seed(b)
    rows = torch.randperm(2 * b + 1, generator=g)[:b]
    held = torch.randn(2 * b + 1, taps - 1, d, generator=g).to(types[0]).cuda()
    held[rows] = x["state"]
    before, given = held.clone(), rows.clone()
    given[::2] = -5
    given[::4] = 2 * b + 1
    out = memory.causal_conv_step(x["x"][:, 0], x["weight"], held, x["bias"], silu=True, starts=x["starts"][:, 0], rows=given.cuda())
    on = torch.ones(b, dtype=torch.bool)
    on[::2] = False
    O.close("out", out[on.cuda()], want["out"][:, 0][on], size["out"][:, 0][on], taps + 16, types[0])
    assert not out[~on.cuda()].any()
    assert torch.equal(held[rows[on].cuda()].double().cpu(), want["state"][on])
    rest = torch.ones(2 * b + 1, dtype=torch.bool)
    rest[rows[on]] = False
    assert torch.equal(held[rest.cuda()], before[rest.cuda()])


# ------------------------------------------------------------------ calls
def test_on_another_stream_and_in_a_graph(memory):
    x = _scan_inputs(61, 3, 300, 64, 16, 1, dtype=BF16)
    y = _conv_inputs(62, 3, 50, 64, 4, dtype=BF16)

    def both():
        out = _run_scan(memory, x)
        leaves = [y[k].detach().requires_grad_() for k in CONV_LEAVES]
        o, s = memory.causal_conv(*leaves[:3], silu=True, starts=y["starts"], lengths=y["lengths"], initial_state=leaves[3], return_state=True)
        return {**out, "conv": o, "conv_state": s, **dict(enumerate(torch.autograd.grad([o, s], leaves, [y["d_out"], y["d_state"]])))}
    want = {k: v.clone() for k, v in both().items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    for k in want:
        assert torch.equal(got[k], want[k]), k
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        got = both()
    for _ in range(4):
        for v in got.values():
            v.detach().fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]), k
        _run_scan(memory, _scan_inputs(63, 2, 300, 64, 16, 1))      # eager work between the replays
        torch.cuda.synchronize()


def test_two_graphs_and_steps(memory):
    """Two captured steps over one state, replayed in turn, are the plies in turn."""
    x = _scan_inputs(64, 5, 2, 64, 16, 1, lengths="none", starts="none")
    state = x["state"].clone()
    want = memory.selective_scan(x["u"], x["delta"], x["a"], x["b"], x["c"], softplus=True, initial_state=state, return_state=True)
    graphs, outs = [], []
    held = state.clone()
    for t in range(2):
        g = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
            outs.append(memory.selective_scan_step(x["u"][:, t], x["delta"][:, t], x["a"], x["b"][:, t], x["c"][:, t], held, softplus=True))
        graphs.append(g)
    for _ in range(3):
        held.copy_(state)
        for t in range(2):
            graphs[t].replay()
        torch.cuda.synchronize()
        assert torch.allclose(held, want[1], rtol=1e-5, atol=1e-6)
        for t in range(2):
            assert torch.allclose(outs[t], want[0][:, t], rtol=1e-5, atol=1e-5)


def test_what_autograd_is_told(memory):
    x = _scan_inputs(65, 3, 4, 16, 4, 1, starts="none", lengths="none")
    with pytest.raises(ValueError, match="no gradient"):
        memory.selective_scan_step(x["u"][:, 0].requires_grad_(), x["delta"][:, 0], x["a"], x["b"][:, 0], x["c"][:, 0], x["state"])
    state = x["state"].clone().requires_grad_()
    saved = (state * state).sum()
    with torch.no_grad():
        memory.selective_scan_step(x["u"][:, 0], x["delta"][:, 0], x["a"], x["b"][:, 0], x["c"][:, 0], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    # a second derivative is refused
    u = x["u"].detach().requires_grad_()
    out = memory.selective_scan(u, x["delta"], x["a"], x["b"], x["c"], softplus=True)
    g = torch.autograd.grad(out.sum(), u, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), u)
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x["u"].detach(), torch.ones_like(x["u"]))
        with pytest.raises(Exception):
            memory.selective_scan(dual, x["delta"], x["a"], x["b"], x["c"])
        with pytest.raises(ValueError, match="forward-mode"):
            memory.selective_scan_step(dual[:, 0], x["delta"][:, 0], x["a"], x["b"][:, 0], x["c"][:, 0], x["state"])
