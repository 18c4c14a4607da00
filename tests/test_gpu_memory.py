"""Operators of a policy's memory (junqi_amd.memory) on an MI355X against their
definitions in 64 bits on the CPU.

Tolerances are bounds on rounding: a result that is a sum of terms is off by at
most (number of roundings) * 2^-24 * (sum of the terms' magnitudes), which the
same definition gives on absolute values; bfloat16 results may round at 2^-8 of
their magnitude (2^-9 each for the result and for one operand of each product)."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def memory():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import memory as M
    return M


def _cpu(t):
    return None if t is None else t.detach().double().cpu()


# ------------------------------------------------------------------ linear attention
def _define(q, k, v, log_decay, starts, lengths, state, scale, d_out=None, d_state=None):
    """Ply by ply in 64 bits; gradients by going back. q, k, v (B, T, H, D) CPU doubles."""
    b, t, h, dk = q.shape
    dv = v.shape[-1]
    lam = torch.exp(log_decay)[None, :, None, None]
    starts = torch.zeros(b, t, dtype=torch.bool) if starts is None else starts.bool().cpu()
    count = torch.full((b,), t) if lengths is None else lengths.cpu().long().clamp(0, t)
    s = torch.zeros(b, h, dk, dv, dtype=torch.float64) if state is None else state.clone()
    out = torch.zeros(b, t, h, dv, dtype=torch.float64)
    dq, d_k, d_v = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(t):
        on = (i < count)[:, None, None]
        old = torch.where(starts[:, i][:, None, None, None], 0.0, lam * s)
        new = old + k[:, i][..., None] * v[:, i][..., None, :]
        s = torch.where(on[..., None], new, s)
        out[:, i] = torch.where(on, scale * (q[:, i][..., None] * s).sum(-2), 0.0)
        if d_out is not None:
            dq[:, i] = torch.where(on, scale * (s * d_out[:, i][..., None, :]).sum(-1), 0.0)
    if d_out is None:
        return out, s
    ds = torch.zeros_like(s) if d_state is None else d_state.clone()
    for i in reversed(range(t)):
        on = (i < count)[:, None, None]
        full = ds + scale * q[:, i][..., None] * d_out[:, i][..., None, :]
        d_k[:, i] = torch.where(on, (full * v[:, i][..., None, :]).sum(-1), 0.0)
        d_v[:, i] = torch.where(on, (full * k[:, i][..., None]).sum(-2), 0.0)
        ds = torch.where(on[..., None], torch.where(starts[:, i][:, None, None, None], 0.0, lam * full), ds)
    return out, s, dq, d_k, d_v, ds


def _inputs(seed, b, t, h, dk, dv, dtype, starts="some", lengths="some", state=True, time_major=False):
    g = torch.Generator().manual_seed(seed)
    lead = (t, b) if time_major else (b, t)

    def rows(d):
        x = torch.randn(*lead, h, d, generator=g).to(dtype).cuda()
        return x.transpose(0, 1) if time_major else x
    q, k, v, d_out = rows(dk), rows(dk), rows(dv), rows(dv)
    ld = -torch.exp2(-torch.rand(h, generator=g) * 8)          # memories of 1 to 256 plies
    st = {"none": None, "all": torch.ones(b, t, dtype=torch.bool),
          "some": torch.rand(b, t, generator=g) < 0.05, "few": torch.rand(b, t, generator=g) < 0.005}[starts]
    n = None
    if lengths == "some":
        n = torch.randint(-1, t + 3, (b,), generator=g, dtype=torch.int32)
        n[:4] = torch.tensor([0, 1, t, t + 9], dtype=torch.int32)[:b]
    s0 = torch.randn(b, h, dk, dv, generator=g).cuda() if state else None
    ds = torch.randn(b, h, dk, dv, generator=g).cuda() if state else None
    return {"q": q, "k": k, "v": v, "log_decay": ld.cuda(), "starts": None if st is None else st.cuda(),
            "lengths": None if n is None else n.cuda(), "state": s0, "d_out": d_out, "d_state": ds}


def _bounds(x, scale, log_decay):
    """Largest errors of out, state, dq, dk, dv, d_state (see the module's head)."""
    absolute = {n: None if x[n] is None else _cpu(x[n]).abs() for n in ("q", "k", "v", "state", "d_out", "d_state")}
    mags = _define(absolute["q"], absolute["k"], absolute["v"], _cpu(log_decay), x["starts"], x["lengths"],
                   absolute["state"], abs(scale), absolute["d_out"], absolute["d_state"])
    b, t, h, dk = x["q"].shape
    dv = x["v"].shape[-1]
    # roundings of a term: both dims' and the plies' sums, the decays' exponents and products
    steps = dk + dv + t * (3 + _cpu(log_decay).abs().clamp(max=8).max().item()) + 64
    f32 = [m * steps * EPS + 1e-37 for m in mags]
    if x["q"].dtype == F32:
        return f32
    # the states are float32 sums of products of which one factor may be held as two bfloat16 parts (2^-17)
    return [f + m * (2.0 ** -16 if i in (1, 5) else 2.0 ** -8 + 2.0 ** -9) for i, (f, m) in enumerate(zip(f32, mags))]


def _close(name, got, want, bound):
    got, want = got.detach().double().cpu(), want
    assert got.shape == want.shape, name
    off = (got - want).abs()
    assert bool((off <= bound).all()), (
        f"{name}: off by {off.max().item():.3g}, bound there {bound.flatten()[(off - bound).argmax()].item():.3g}")


def _check_attention(memory, x, scale=None, grads=True):
    dk = x["q"].shape[-1]
    s = dk ** -0.5 if scale is None else scale
    want = _define(*(_cpu(x[n]) for n in ("q", "k", "v", "log_decay")), x["starts"], x["lengths"], _cpu(x["state"]), s,
                   _cpu(x["d_out"]), _cpu(x["d_state"]))
    bounds = _bounds(x, s, x["log_decay"])
    leaves = [x[n].detach().requires_grad_(grads) for n in ("q", "k", "v")]
    s0 = None if x["state"] is None else x["state"].detach().requires_grad_(grads)
    out, state = memory.linear_attention(*leaves, x["log_decay"], starts=x["starts"], lengths=x["lengths"],
                                         initial_state=s0, scale=scale, return_state=True)
    assert out.dtype == x["q"].dtype and state.dtype == F32
    _close("out", out, want[0], bounds[0])
    _close("state", state, want[1], bounds[1])
    if not grads:
        return
    if s0 is None:
        got = torch.autograd.grad([out], leaves, [x["d_out"]])
    else:
        got = torch.autograd.grad([out, state], [*leaves, s0], [x["d_out"], x["d_state"]])
    for i, name in enumerate(("dq", "dk", "dv", "d_state")[:len(got)]):
        _close(name, got[i], want[2 + i], bounds[2 + i])


SHAPES = [(1, 1, 1, 1, 1), (5, 2, 1, 5, 7), (3, 63, 2, 64, 64), (4, 64, 1, 16, 16), (5, 65, 1, 64, 32), (2, 127, 3, 40, 56),
          (4, 129, 1, 128, 128), (2, 200, 2, 50, 36), (3, 100, 1, 24, 128), (6, 31, 2, 96, 33), (1, 500, 1, 32, 32)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("masks", [("none", "none", False), ("some", "some", True), ("few", "none", True)])
def test_attention_shapes(memory, shape, dtype, masks):
    starts, lengths, state = masks
    print(f"[attention] {shape} {dtype} {masks}", flush=True)
    _check_attention(memory, _inputs(sum(shape), *shape, dtype, starts, lengths, state))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_of_time_major_views_and_slices(memory, dtype):
    """Transposed rollout buffers, heads out of one packed projection, an odd
    element offset, a key shared by all heads: any strides give the same."""
    x = _inputs(3, 3, 90, 2, 32, 32, dtype, time_major=True)
    _check_attention(memory, x)
    y = _inputs(4, 3, 90, 2, 32, 32, dtype)
    pack = torch.randn(3, 90, 3, 2, 32, device="cuda").to(dtype)
    y["q"], y["k"], y["v"] = pack.unbind(2)
    _check_attention(memory, y)
    y["k"] = y["k"][:, :, :1].expand(3, 90, 2, 32)
    _check_attention(memory, y)
    odd = torch.randn(3 * 90 * 2 * 33 + 1, device="cuda").to(dtype)[1:].view(3, 90, 2, 33)
    y["q"], y["v"] = odd[..., :32], odd[..., 1:]
    y["starts"] = torch.rand(90, 6, device="cuda")[:, ::2].T < 0.05
    _check_attention(memory, y)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("starts", ["all", "edges"])
def test_attention_where_games_start(memory, dtype, starts):
    x = _inputs(5, 3, 140, 2, 32, 48, dtype, "all")
    if starts == "edges":
        x["starts"][:] = False
        x["starts"][0, [0, 1, 31, 32, 63, 64, 65, 127, 128, 139]] = True
        x["starts"][1, 0] = True
        x["starts"][2, 139] = True
        x["lengths"] = None
    _check_attention(memory, x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("decay", [0.0, -1e-6, -5.0, -100.0, -math.inf])
def test_attention_decays(memory, dtype, decay):
    x = _inputs(6, 2, 150, 2, 32, 32, dtype, "few")
    x["log_decay"][0] = decay
    _check_attention(memory, x)


@pytest.mark.parametrize("b,t", [(1, 5000), (2, 4097), (1, 20011)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_of_long_records(memory, b, t, dtype):
    """Few rows and a long axis, games starting here and there."""
    x = _inputs(7, b, t, 1, 32, 24, dtype, "few", "none", True)
    x["starts"][:, 2500:] = False      # a long part without a start
    _check_attention(memory, x)
    if b == 2:
        x["lengths"] = torch.tensor([t - 700, 3], dtype=torch.int64, device="cuda")
        _check_attention(memory, x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_sees_nothing_of_bad_plies_elsewhere(memory, dtype, bad):
    """NaN and infinities in padding, in plies after, in games before a start and
    in the state that a start discards do not reach what does not see them."""
    x = _inputs(8, 4, 150, 2, 32, 32, dtype, "none", "none", True)
    x["starts"] = torch.zeros(4, 150, dtype=torch.bool, device="cuda")
    x["starts"][:, 70] = True
    x["starts"][3, 0] = True
    x["lengths"] = torch.tensor([150, 150, 100, 150], dtype=torch.int32, device="cuda")
    clean = {n: None if t is None else t.clone() for n, t in x.items()}
    for n in ("q", "k", "v", "d_out"):
        x[n][0, 66] = bad                       # before the start at 70
        x[n][1, 120] = bad                      # after it: plies 70..119 do not see it forward
        x[n][2, 100:] = bad                     # padding
    x["state"][3] = bad                         # a game starts at once
    args = dict(starts=x["starts"], lengths=x["lengths"], return_state=True)
    leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "state")]
    out, state = memory.linear_attention(*leaves[:3], x["log_decay"], initial_state=leaves[3], **args)
    dq, dk, dv, ds = torch.autograd.grad([out, state], leaves, [x["d_out"], x["d_state"]])
    want = _define(*(_cpu(clean[n]) for n in ("q", "k", "v", "log_decay")), clean["starts"], clean["lengths"],
                   _cpu(clean["state"]), 32 ** -0.5, _cpu(clean["d_out"]), _cpu(clean["d_state"]))
    bounds = _bounds(clean, 32 ** -0.5, clean["log_decay"])
    fine = {"out": [(0, slice(0, 66)), (0, slice(70, 150)), (1, slice(0, 120)), (2, slice(0, 150)), (3, slice(0, 150))],
            "dq": [(0, slice(0, 66)), (0, slice(70, 150)), (1, slice(0, 120)), (2, slice(0, 150)), (3, slice(0, 150))],
            "dk": [(0, slice(67, 150)), (1, slice(0, 70)), (1, slice(121, 150)), (2, slice(0, 150)), (3, slice(0, 150))],
            "dv": [(0, slice(67, 150)), (1, slice(0, 70)), (1, slice(121, 150)), (2, slice(0, 150)), (3, slice(0, 150))]}
    for i, (name, got) in enumerate((("out", out), (None, None), ("dq", dq), ("dk", dk), ("dv", dv))):
        if name:
            for b, at in fine[name]:
                _close(f"{name} of row {b}", got[b, at], want[i][b, at], bounds[i][b, at])
    for b in (0, 2, 3):
        _close("state", state[b], want[1][b], bounds[1][b])
    for b in (1, 2, 3):
        _close("d_state", ds[b], want[5][b], bounds[5][b])
    assert not torch.isfinite(out[1, 120:]).any() and not torch.isfinite(state[1]).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_of_nothing(memory, dtype):
    for b, t in ((0, 5), (3, 0), (0, 0)):
        x = _inputs(9, b, t, 2, 16, 8, dtype, "none", "none")
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "state")]
        out, state = memory.linear_attention(*leaves[:3], x["log_decay"], initial_state=leaves[3], return_state=True)
        assert out.shape == (b, t, 2, 8) and torch.equal(state, x["state"])
        grads = torch.autograd.grad([out, state], leaves, [x["d_out"], x["d_state"]])
        assert grads[0].shape == x["q"].shape and torch.equal(grads[3], x["d_state"])
        out, state = memory.linear_attention(x["q"], x["k"], x["v"], x["log_decay"], return_state=True)
        assert not state.any()


def test_attention_gradient_against_differences(memory):
    """The loss is linear in each of q, k, v and the state alone: a difference of
    two losses is the gradient's product with the step, whatever its length."""
    x = _inputs(10, 3, 150, 2, 40, 24, F32, "few")
    names = ("q", "k", "v", "state")
    weight, d_state = x["d_out"].double(), x["d_state"].double()

    def loss(**over):
        y = {**x, **over}
        out, state = memory.linear_attention(y["q"], y["k"], y["v"], x["log_decay"], starts=x["starts"],
                                             lengths=x["lengths"], initial_state=y["state"], return_state=True)
        return ((out.double() * weight).sum() + (state.double() * d_state).sum()).item()
    leaves = [x[n].detach().requires_grad_() for n in names]
    out, state = memory.linear_attention(*leaves[:3], x["log_decay"], starts=x["starts"], lengths=x["lengths"],
                                         initial_state=leaves[3], return_state=True)
    grads = torch.autograd.grad([out, state], leaves, [x["d_out"], x["d_state"]])
    size = [m.sum().item() for m in _bounds(x, 40 ** -0.5, x["log_decay"])]
    # rounding of two losses: every output's bound times a weight of order 1 (at most 6 for normal numbers)
    bound = 12 * (size[0] + size[1])
    for n, g in zip(names, grads):
        step = torch.randn(x[n].shape, generator=torch.Generator().manual_seed(1)).cuda()
        diff = loss(**{n: x[n] + step}) - loss()
        assert abs(diff - (g.double() * step.double()).sum().item()) <= bound, n


def test_attention_partial_gradients(memory):
    """Only the output or only the state used; only some inputs with gradients."""
    x = _inputs(11, 2, 70, 2, 16, 32, F32)
    full = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "state")]
    kw = dict(starts=x["starts"], lengths=x["lengths"], return_state=True)
    out, state = memory.linear_attention(*full[:3], x["log_decay"], initial_state=full[3], **kw)
    a = torch.autograd.grad([out], full, [x["d_out"]], retain_graph=True)
    b = torch.autograd.grad([state], full, [x["d_state"]], allow_unused=True)
    want = _define(*(_cpu(x[n]) for n in ("q", "k", "v", "log_decay")), x["starts"], x["lengths"], _cpu(x["state"]),
                   16 ** -0.5, _cpu(x["d_out"]), torch.zeros_like(_cpu(x["state"])))
    bounds = _bounds(x, 16 ** -0.5, x["log_decay"])
    for i in range(4):
        _close(f"gradient {i} of out", a[i], want[2 + i], bounds[2 + i])
    want = _define(*(_cpu(x[n]) for n in ("q", "k", "v", "log_decay")), x["starts"], x["lengths"], _cpu(x["state"]),
                   16 ** -0.5, torch.zeros_like(_cpu(x["d_out"])), _cpu(x["d_state"]))
    for i in range(1, 4):
        _close(f"gradient {i} of state", b[i], want[2 + i], bounds[2 + i])
    assert b[0] is None or not b[0].any()
    q = x["q"].detach().requires_grad_()
    out = memory.linear_attention(q, x["k"], x["v"], x["log_decay"], starts=x["starts"], lengths=x["lengths"],
                                  initial_state=x["state"])
    _close("dq alone", torch.autograd.grad(out, q, x["d_out"])[0], a[0].double().cpu(), torch.zeros(()))


def test_attention_is_the_same_every_time(memory):
    x = _inputs(12, 2, 3000, 2, 64, 64, BF16, "few", "none")
    runs = []
    for _ in range(3):
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "state")]
        out, state = memory.linear_attention(*leaves[:3], x["log_decay"], starts=x["starts"], initial_state=leaves[3],
                                             return_state=True)
        runs.append([out, state, *torch.autograd.grad([out, state], leaves, [x["d_out"], x["d_state"]])])
    for r in runs[1:]:
        assert all(torch.equal(u, w) for u, w in zip(r, runs[0]))


def test_attention_on_another_stream(memory):
    x = _inputs(13, 4, 200, 2, 64, 64, BF16, "few", "some")
    kw = dict(starts=x["starts"], lengths=x["lengths"], initial_state=x["state"])
    want = memory.linear_attention(x["q"], x["k"], x["v"], x["log_decay"], **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = memory.linear_attention(x["q"], x["k"], x["v"], x["log_decay"], **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


# ------------------------------------------------------------------ one ply
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (3, 2, 64, 64), (7, 1, 40, 56), (5, 3, 50, 33), (2, 2, 128, 128), (4, 1, 16, 128),
                                   (600, 4, 32, 20)])
def test_step(memory, shape, dtype):
    b, h, dk, dv = shape
    x = _inputs(sum(shape), b, 2, h, dk, dv, dtype, "none", "none")
    q, k, v = x["q"][:, 1], x["k"][:, 1], x["v"][:, 1]        # strided rows
    starts = torch.arange(b, device="cuda") % 3 == 1
    for rows in (None, torch.randperm(2 * b, generator=torch.Generator().manual_seed(b))[:b].cuda()):
        state = torch.randn(b if rows is None else 2 * b, h, dk, dv, device="cuda")
        use = state if rows is None else state[rows]
        if rows is not None and b > 2:
            rows[0], rows[2] = -1, 2 * b
        want, s = _define(*(_cpu(t[:, None]) for t in (q, k, v)), _cpu(x["log_decay"]), starts[:, None], None, _cpu(use),
                          dk ** -0.5)
        mag, smag = _define(*(_cpu(t[:, None]).abs() for t in (q, k, v)), _cpu(x["log_decay"]), starts[:, None], None,
                            _cpu(use).abs(), dk ** -0.5)
        got_state = state.clone()
        got = memory.linear_attention_step(q, k, v, x["log_decay"], got_state, rows=rows, starts=starts)
        live = torch.ones(b, dtype=torch.bool)
        if rows is not None and b > 2:
            live[[0, 2]] = False
        bound = mag[:, 0] * (dk + 8) * EPS + (0 if dtype == F32 else want[:, 0].abs() * 2.0 ** -8)
        _close("out", got[live.cuda()], want[live, 0], bound[live])
        assert not got[~live.cuda()].any()
        expect = state.double().cpu()
        r = torch.arange(b) if rows is None else rows.cpu()
        expect[r[live]] = s[live]
        off = torch.zeros_like(expect)
        off[r[live]] = smag[live] * 8 * EPS
        _close("state", got_state, expect, off)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("games,key_dim,value_dim", [(9, 5, 2), (9, 17, 3), (9, 64, 5), (9, 7, 17), (9, 33, 35), (9, 50, 50), (9, 128, 67),
                                                     (9, 127, 127), (22000, 50, 50)])   # the last: more than the caches hold
def test_step_of_odd_dims(memory, dtype, games, key_dim, value_dim):
    """Rows of a state that end inside a vector, and the elements beside the states untouched."""
    g = torch.Generator("cuda").manual_seed(value_dim)
    size = games * 2 * key_dim * value_dim
    store = torch.randn(size + 2, device="cuda", generator=g)
    state = store[1:-1].view(games, 2, key_dim, value_dim)
    before = store.clone()
    q, k = (torch.randn(games, 2, key_dim, device="cuda", generator=g).to(dtype) for _ in range(2))
    v = torch.randn(games, 2, value_dim, device="cuda", generator=g).to(dtype)
    decay = torch.tensor([-0.2, -0.01], device="cuda")
    out = memory.linear_attention_step(q, k, v, decay, state)
    assert store[0] == before[0] and store[-1] == before[-1]
    old, lam = before[1:-1].view_as(state).double(), decay.double().exp()[:, None, None]
    kv = k.double()[..., :, None] * v.double()[..., None, :]
    want = lam * old + kv
    assert ((state.double() - want).abs() <= (lam * old.abs() + kv.abs()) * 8 * EPS).all()
    scale = key_dim ** -0.5
    answer = (q.double()[..., None] * want).sum(-2) * scale
    mag = (q.double().abs()[..., None] * (lam * old.abs() + kv.abs())).sum(-2) * scale
    bound = mag * (key_dim + 8) * EPS + (0 if dtype == F32 else answer.abs() * 2.0 ** -8)
    assert ((out.double() - answer).abs() <= bound).all()


def test_step_follows_the_segments(memory):
    """Plies one by one, from a zero state, answer what the whole segment does."""
    x = _inputs(20, 5, 40, 2, 48, 64, F32, "some", "none", False)
    whole, last = memory.linear_attention(x["q"], x["k"], x["v"], x["log_decay"], starts=x["starts"], return_state=True)
    state = torch.zeros(5, 2, 48, 64, device="cuda")
    out = torch.empty(5, 40, 2, 64, device="cuda")
    for t in range(40):
        got = memory.linear_attention_step(x["q"][:, t], x["k"][:, t], x["v"][:, t], x["log_decay"], state,
                                           starts=x["starts"][:, t], out=out[:, t])
        assert got.data_ptr() == out[:, t].data_ptr()
    bounds = _bounds(x, 48 ** -0.5, x["log_decay"])
    _close("out", out, whole.double().cpu(), 2 * bounds[0])
    _close("state", state, last.double().cpu(), 2 * bounds[1])


def test_step_discards_a_bad_state(memory):
    x = _inputs(21, 3, 1, 1, 16, 16, F32, "none", "none")
    state = torch.full((3, 1, 16, 16), math.nan, device="cuda")
    out = memory.linear_attention_step(x["q"][:, 0], x["k"][:, 0], x["v"][:, 0], x["log_decay"], state,
                                       starts=torch.tensor([True, False, True], device="cuda"))
    assert torch.isfinite(out[[0, 2]]).all() and torch.isfinite(state[[0, 2]]).all()
    assert out[1].isnan().all() and state[1].isnan().all()


def test_step_of_an_unaligned_state(memory):
    """A state whose first element is not at a 16-byte boundary, and one that is."""
    x = _inputs(23, 4, 1, 1, 8, 8, F32, "none", "none")
    store = torch.randn(4 * 64 + 1, generator=torch.Generator().manual_seed(1)).cuda()
    odd, even = store[1:].view(4, 1, 8, 8), store[1:].clone().view(4, 1, 8, 8)
    args = [x[n][:, 0] for n in ("q", "k", "v")] + [x["log_decay"]]
    want = _define(*(_cpu(t[:, None]) for t in args[:3]), _cpu(x["log_decay"]), None, None, _cpu(even), 8 ** -0.5)
    mag = _define(*(_cpu(t[:, None]).abs() for t in args[:3]), _cpu(x["log_decay"]), None, None, _cpu(even).abs(), 8 ** -0.5)
    for s in (odd, even):
        out = memory.linear_attention_step(*args, s)
        _close("out", out, want[0][:, 0], mag[0][:, 0] * 16 * EPS)
        _close("state", s, want[1], mag[1] * 8 * EPS)


def test_step_of_nothing(memory):
    z = torch.empty(0, 2, 8, device="cuda")
    out = memory.linear_attention_step(z, z, z, torch.zeros(2, device="cuda"), torch.empty(0, 2, 8, 8, device="cuda"))
    assert out.shape == (0, 2, 8)


def test_step_in_a_graph(memory):
    """A captured step, replayed with the program's own work between."""
    x = _inputs(22, 64, 3, 2, 64, 64, BF16, "some", "none")
    q, k, v, st = (x[n][:, 0].clone() for n in ("q", "k", "v", "starts"))
    state, mirror = x["state"].clone(), x["state"].clone()
    out = torch.empty(64, 2, 64, dtype=BF16, device="cuda")
    memory.linear_attention_step(q, k, v, x["log_decay"], state.clone(), starts=st, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        memory.linear_attention_step(q, k, v, x["log_decay"], state, starts=st, out=out)
    for t in range(3):
        for dst, n in ((q, "q"), (k, "k"), (v, "v"), (st, "starts")):
            dst.copy_(x[n][:, t])
        graph.replay()
        want = memory.linear_attention_step(x["q"][:, t], x["k"][:, t], x["v"][:, t], x["log_decay"], mirror,
                                            starts=x["starts"][:, t])
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, mirror)


# ------------------------------------------------------------------ rotary positions
def _turned(x, positions, frequencies, sections, interleaved, sign=1.0):
    x, f = _cpu(x), _cpu(frequencies)
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    angle = positions.cpu().double()[..., axis] * f
    c, s = torch.cos(angle)[..., None, :], sign * torch.sin(angle)[..., None, :]
    n = f.numel()
    i = torch.arange(n) * 2 if interleaved else torch.arange(n)
    j = i + 1 if interleaved else i + n
    y = x.clone()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


def _rotary_bound(x, want):
    """Two products of order |x| with a cosine that is off by 4 * 2^-24 at most (the
    angle's last bit in half turns, and the function's), and the result's rounding."""
    size = _cpu(x).abs().amax(-1, keepdim=True)
    return 16 * EPS * size + (2.0 ** -8 * want.abs() if x.dtype == BF16 else 0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead,heads,dim,sections", [((5,), 1, 2, (1,)), ((3, 7), 2, 64, (12, 10, 10)), ((300,), 4, 56, (10, 10)),
                                                     ((2, 3, 5), 3, 33, (7, 0, 4, 5)), ((1,), 8, 128, (64,)), ((4, 129), 1, 24, (3, 2)),
                                                     ((1000,), 3, 200, (50, 50))])
def test_rotary(memory, dtype, interleaved, lead, heads, dim, sections):
    g = torch.Generator().manual_seed(dim)
    x = torch.randn(*lead, heads, dim, generator=g).to(dtype).cuda().requires_grad_()
    pos = torch.randint(-50, 1200, (*lead, len(sections)), generator=g, dtype=torch.int32 if dim % 3 else torch.int64).cuda()
    f = memory.rotary_frequencies(sections, device="cuda")
    out = memory.rotary(x, pos, f, sections, interleaved=interleaved)
    want = _turned(x, pos, f, sections, interleaved)
    assert out.dtype == dtype
    _close("out", out, want, _rotary_bound(x, want))
    d = torch.randn(*lead, heads, dim, generator=g).to(dtype).cuda()
    want = _turned(d, pos, f, sections, interleaved, -1.0)
    _close("gradient", torch.autograd.grad(out, x, d)[0], want, _rotary_bound(d, want))


def test_rotary_far_positions_and_views(memory):
    """Plies past 2^31 and heads out of a packed, time-major projection."""
    g = torch.Generator().manual_seed(1)
    pack = torch.randn(40, 3, 6, 32, generator=g).cuda()          # (T, B, q and k and v heads, D)
    x = pack.transpose(0, 1)[:, :, 1:5]
    pos = torch.stack([torch.arange(40).expand(3, 40) * 3 + 2 ** 31, torch.arange(40).expand(3, 40) % 17], -1).cuda()
    f = memory.rotary_frequencies((10, 6), device="cuda")
    out = memory.rotary(x, pos, f, (10, 6))
    want = _turned(x, pos, f, (10, 6), False)
    _close("out", out, want, _rotary_bound(x, want))
    loose = pos.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(memory.rotary(x, loose, f, (10, 6)), out)
    assert memory.rotary(torch.empty(0, 2, 8, device="cuda"), torch.empty(0, 1, dtype=torch.int32, device="cuda"),
                         f[:4], (4,)).shape == (0, 2, 8)


def test_rotary_gradient_against_differences(memory):
    g = torch.Generator().manual_seed(2)
    x, step, d = (torch.randn(50, 2, 24, generator=g).cuda() for _ in range(3))
    pos = torch.randint(0, 300, (50, 3), generator=g).cuda()
    f = memory.rotary_frequencies((5, 4, 3), device="cuda")

    def call(y):
        return memory.rotary(y, pos, f, (5, 4, 3))
    leaf = x.clone().requires_grad_()
    grad = torch.autograd.grad(call(leaf), leaf, d)[0]
    diff = ((call(x + step).double() - call(x).double()) * d.double()).sum()
    bound = 3 * 16 * EPS * 6 * d.abs().sum().double()          # three roundings of rows of normal numbers, at most 6
    assert abs(diff - (grad.double() * step.double()).sum()) <= bound


# ------------------------------------------------------------------ layer norm
def _normed(x, w, b, eps, d=None):
    x = _cpu(x)
    m = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    hat = (x - m) * r
    w1 = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else _cpu(w)
    out = hat * w1 + (0 if b is None else _cpu(b))
    if d is None:
        return out
    d = _cpu(d)
    g = d * w1
    dx = r * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
    lead = tuple(range(x.ndim - 1))
    return out, dx, (d * hat).sum(lead), d.sum(lead), hat, r, g


def _norm_bounds(x, w, b, eps, d):
    """Roundings: a row's mean is off by width roundings of its mean magnitude at
    most (far fewer in a tree), which hat and the sums over it carry on."""
    out, dx, dw, db, hat, r, g = _normed(x, w, b, eps, d)
    n = x.shape[-1]
    lead = tuple(range(x.ndim - 1))
    rows = max(1, x.numel() // n)
    e = (math.log2(n + 1) + n / 256 + 16) * EPS                # a tree over lanes of up to n / 256 elements in a row
    size = _cpu(x).abs().amax(-1, keepdim=True) * r            # mean's error in units of hat
    off = e * (size + hat.abs() + 1)
    wmax = 1.0 if w is None else _cpu(w).abs().max()
    low = 2.0 ** -8 if x.dtype == BF16 else 0.0
    b_out = off * wmax + low * out.abs() + 4 * EPS * out.abs() + (0 if b is None else 4 * EPS * _cpu(b).abs())
    gm = g.abs().amax(-1, keepdim=True)
    b_dx = r * 4 * (off + e) * gm * (1 + hat.abs()) * (1 + size) + low * dx.abs()
    er = (math.log2(rows + 1) + rows / 64 + 16) * EPS
    terms = (_cpu(d).abs() * (off + hat.abs() * er)).sum(lead)
    wlow = 2.0 ** -8 if w is not None and w.dtype == BF16 else 0.0
    return b_out, b_dx, terms + wlow * dw.abs(), _cpu(d).abs().sum(lead) * er + wlow * db.abs()


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("lead,width", [((1,), 1), ((3,), 2), ((7,), 28), ((2, 3), 64), ((65,), 65), ((5, 3, 2), 256), ((129,), 317),
                                        ((1100,), 130), ((9,), 1024), ((4,), 4097), ((3,), 8192), ((2,), 20001), ((5000,), 17)])
def test_norm(memory, dtype, wdtype, lead, width):
    g = torch.Generator().manual_seed(width)
    x = (torch.randn(*lead, width, generator=g) * 2 + 0.7).to(dtype).cuda().requires_grad_()
    w = (1 + torch.randn(width, generator=g) * 0.2).to(wdtype).cuda().requires_grad_()
    b = (torch.randn(width, generator=g) * 0.2).to(wdtype).cuda().requires_grad_()
    d = torch.randn(*lead, width, generator=g).to(dtype).cuda()
    out = memory.layer_norm(x, w, b)
    assert out.shape == x.shape and out.dtype == dtype
    want = _normed(x, w, b, 1e-5, d)
    bounds = _norm_bounds(x, w, b, 1e-5, d)
    grads = torch.autograd.grad(out, (x, w, b), d)
    assert grads[1].dtype == wdtype
    for i, (name, got) in enumerate(zip(("out", "dx", "dweight", "dbias"), (out, *grads))):
        _close(name, got, want[i], bounds[i])
    with torch.no_grad():
        assert torch.equal(memory.layer_norm(x, w, b), out)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width", [(2500, 2001), (5, 3001), (6, 12001), (4100, 129), (700, 500)])
def test_norm_widths(memory, dtype, rows, width):
    """Rows held by every shape of a block, ends inside a vector; more rows than groups."""
    g = torch.Generator().manual_seed(width)
    x = (torch.randn(rows, width, generator=g) * 2 + 0.7).to(dtype).cuda().requires_grad_()
    w = (1 + torch.randn(width, generator=g) * 0.2).cuda().requires_grad_()
    b = (torch.randn(width, generator=g) * 0.2).cuda().requires_grad_()
    d = torch.randn(rows, width, generator=g).to(dtype).cuda()
    out = memory.layer_norm(x, w, b)
    want = _normed(x, w, b, 1e-5, d)
    bounds = _norm_bounds(x, w, b, 1e-5, d)
    for i, (name, got) in enumerate(zip(("out", "dx", "dweight", "dbias"), (out, *torch.autograd.grad(out, (x, w, b), d)))):
        _close(name, got, want[i], bounds[i])


def test_norm_forms(memory):
    """Without weight or bias; row views; rows that are all the same; large offsets."""
    g = torch.Generator().manual_seed(3)
    base = torch.randn(50, 200, generator=g).cuda()
    x = base[::2, 1:101].detach().requires_grad_()
    d = torch.randn(25, 100, generator=g).cuda()
    for w, b in ((None, None), (torch.rand(100, generator=g).cuda(), None), (None, torch.rand(100, generator=g).cuda())):
        out = memory.layer_norm(x, w, b)
        want, bounds = _normed(x, w, b, 1e-5, d), _norm_bounds(x, w, b, 1e-5, d)
        _close("out", out, want[0], bounds[0])
        _close("dx", torch.autograd.grad(out, x, d)[0], want[1], bounds[1])
    same = torch.full((3, 64), 7.25, device="cuda")
    assert not memory.layer_norm(same).any()
    far = base[:10, :128] + 1000.0
    _close("far", memory.layer_norm(far), _normed(far, None, None, 1e-5), _norm_bounds(far, None, None, 1e-5, far)[0])
    assert memory.layer_norm(torch.empty(0, 5, device="cuda")).shape == (0, 5)
    x = torch.empty(0, 5, device="cuda")
    w = torch.ones(5, device="cuda", requires_grad=True)
    assert not torch.autograd.grad(memory.layer_norm(x, w), w, x)[0].any()
    t = base.detach().view(5, 10, 200).transpose(0, 1).requires_grad_()
    out = memory.layer_norm(t)
    dx = torch.autograd.grad(out, t, out.detach())[0]
    ref = base.detach().clone().requires_grad_()
    o2 = memory.layer_norm(ref)
    dx2 = torch.autograd.grad(o2, ref, o2.detach())[0]
    assert torch.equal(out, o2.view(5, 10, 200).transpose(0, 1)) and torch.equal(dx, dx2.view(5, 10, 200).transpose(0, 1))


def test_norm_of_a_broadcast_gradient(memory):
    """A loss that sums its outputs hands in a gradient of stride 0."""
    x = torch.randn(33, 96, generator=torch.Generator().manual_seed(4)).cuda().requires_grad_()
    w = torch.rand(96, device="cuda", requires_grad=True)
    got = torch.autograd.grad(memory.layer_norm(x, w).sum(), (x, w))
    ones = torch.ones(33, 96, device="cuda")
    want, bounds = _normed(x, w, None, 1e-5, ones), _norm_bounds(x, w, None, 1e-5, ones)
    _close("dx", got[0], want[1], bounds[1])
    _close("dweight", got[1], want[2], bounds[2])


def test_norm_gradient_against_differences(memory):
    """Central differences of step h: off by h^2 of the third derivatives (a few
    units for normal rows of 40) and rounding / h."""
    g = torch.Generator().manual_seed(5)
    x, sx, d = (torch.randn(30, 40, generator=g).cuda() for _ in range(3))
    w, sw, b, sb = (torch.randn(40, generator=g).cuda() for _ in range(4))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(memory.layer_norm(*leaves), leaves, d)
    h = 2.0 ** -7

    def loss(*a):
        return (memory.layer_norm(*a).double() * d.double()).sum().item()
    scale = (d.abs().sum() * w.abs().max() * 4).item()
    bound = scale * (8 * h * h + 32 * EPS / h)
    for got, step, at in ((grads[0], sx, 0), (grads[1], sw, 1), (grads[2], sb, 2)):
        a, c = [x, w, b], [x, w, b]
        a[at], c[at] = a[at] + h * step, c[at] - h * step
        assert abs((loss(*a) - loss(*c)) / (2 * h) - (got.double() * step.double()).sum().item()) <= bound


def test_norm_is_the_same_every_time(memory):
    x = torch.randn(30000, 64, device="cuda").bfloat16().requires_grad_()
    w, b = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    runs = [torch.autograd.grad(memory.layer_norm(x, w, b), (x, w, b), x.detach()) for _ in range(3)]
    assert all(torch.equal(u, v) for r in runs[1:] for u, v in zip(r, runs[0]))


# ------------------------------------------------------------------ refusals
def test_refusals(memory):
    z = lambda *s, dt=F32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    q, ld = z(2, 5, 3, 8), z(3)
    bad = [
        (z(2, 5, 3, 8, dt=torch.float16), q, q, ld, {}), (q.cpu(), q, q, ld, {}), (q, z(2, 5, 3, 9), q, ld, {}),
        (q, q, z(2, 4, 3, 8), ld, {}), (q[0], q[0], q[0], ld, {}), (q, q.bfloat16(), q, ld, {}), (q, q, q, z(2), {}),
        (q, q, q, ld.double(), {}), (q, q, q, ld.clone().requires_grad_(), {}), (z(2, 5, 3, 129), z(2, 5, 3, 129), q, ld, {}),
        (q, q, q, ld, {"starts": z(2, 5)}), (q, q, q, ld, {"starts": z(5, 2, dt=torch.bool)}),
        (q, q, q, ld, {"lengths": z(2)}), (q, q, q, ld, {"lengths": z(3, dt=torch.int32)}),
        (q, q, q, ld, {"initial_state": z(2, 3, 8, 9)}), (q, q, q, ld, {"initial_state": z(2, 3, 8, 8, dt=BF16)}),
        (z(2, 5, 0, 8), z(2, 5, 0, 8), z(2, 5, 0, 8), z(0), {}),
    ]
    for i, (a, b, c, d, kw) in enumerate(bad):
        with pytest.raises(ValueError):
            memory.linear_attention(a, b, c, d, **kw)
            pytest.fail(f"case {i} was taken")
    s, state = z(2, 3, 8), z(2, 3, 8, 8)
    for kw in ({"state": z(3, 3, 8, 8)}, {"state": state.transpose(2, 3)}, {"state": state.bfloat16()}, {"state": z(2, 3, 8)},
               {"rows": z(2, dt=torch.int32)}, {"rows": z(3, dt=torch.int64)}, {"starts": z(2)}, {"out": z(2, 3, 9)},
               {"out": z(2, 3, 8, dt=BF16)}, {"out": z(2, 8, 3).transpose(1, 2)}, {"k": z(2, 3, 7)}):
        args = {"q": s, "k": s, "v": s, "log_decay": ld, "state": state, **kw}
        with pytest.raises(ValueError):
            memory.linear_attention_step(**args)
            pytest.fail(f"{list(kw)} was taken")
    with pytest.raises(ValueError):
        memory.linear_attention_step(s.clone().requires_grad_(), s, s, ld, state)
    x, p, f = z(5, 2, 8), z(5, 2, dt=torch.int32), z(4)
    for a in ((x, p, f, (2, 3)), (x, p, f, (2, 1)), (x, p, f, (4,)), (x, p, f, (5, -1)), (x, z(5, 2), f, (2, 2)),
              (x, p, f.double(), (2, 2)), (x, p[:4], f, (2, 2)), (x, p, z(5), (3, 2)), (x.half(), p, f, (2, 2)),
              (x[0], p[0], f, (2, 2)), (x, p, f, ()), (x, z(5, 5, dt=torch.int32), f, (1, 1, 1, 1, 0)),
              (x, p, f.clone().requires_grad_(), (2, 2))):
        with pytest.raises(ValueError):
            memory.rotary(*a)
            pytest.fail(f"{a[3]} was taken")
    w = z(8)
    for a in ((x.half(),), (x.cpu(),), (x, z(7)), (x, w.bfloat16()), (x.bfloat16(), w, w.bfloat16()), (z(5, 0),), (x, None, w.cpu())):
        with pytest.raises(ValueError):
            memory.layer_norm(*a)
            pytest.fail("was taken")
