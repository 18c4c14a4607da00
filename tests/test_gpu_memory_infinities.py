"""Infinities and NaN in linear attention's rows and states on an MI355X: each result is
what the definition, ply by ply in 64 bits, makes of them, an infinity of its sign, NaN,
or (of the plies and columns that see none of them) a finite number."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from tests import memory_oracle as O  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def memory():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import memory as M
    return M


def _case(seed, b, t, h, dk, dv, dtype):
    g = torch.Generator("cuda").manual_seed(seed)

    def rows(*shape, to=dtype):
        # of one sign, so that infinities meet none of the other sign and stay what they are
        return (torch.randn(shape, generator=g, device="cuda").abs() + 0.01).to(to)
    x = {"q": rows(b, t, h, dk), "k": rows(b, t, h, dk), "v": rows(b, t, h, dv), "d_out": rows(b, t, h, dv),
         "state": rows(b, h, dk, dv, to=F32), "d_state": rows(b, h, dk, dv, to=F32),
         "log_decay": -torch.exp2(-6 * torch.rand(h, generator=g, device="cuda")),
         "starts": torch.zeros(b, t, dtype=torch.bool, device="cuda"), "lengths": None}
    return x


def _check(memory, x):
    dk = x["q"].shape[-1]
    dtype, scale = x["q"].dtype, dk ** -0.5

    def args(y):
        return (*(y[n].double() for n in ("q", "k", "v", "log_decay")), y["starts"], y["lengths"], y["state"].double(),
                scale, y["d_out"].double(), y["d_state"].double())
    want = O.define(*args(x))
    # a finite result has no term with an infinity or NaN: its errors are those of the other terms
    fine = {n: torch.nan_to_num(x[n], 0.0, 0.0, 0.0).abs() if n in ("q", "k", "v", "state", "d_out", "d_state") else x[n] for n in x}
    mags = O.define(*args(fine))
    leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "state")]
    out, last = memory.linear_attention(*leaves[:3], x["log_decay"], starts=x["starts"], lengths=x["lengths"],
                                        initial_state=leaves[3], return_state=True)
    got = (out, last, *torch.autograd.grad([out, last], leaves, [x["d_out"], x["d_state"]]))
    t = x["q"].shape[1]
    steps = dk + x["v"].shape[-1] + 4 * t + 64               # roundings of a term: both dims, and a ply's decay and sum
    for name, r, w, m in zip(O.NAMES, got, want, mags):
        r = r.detach().double()
        bound = m * steps * EPS
        if dtype == BF16:
            bound = bound + m * 2.0 ** -16 + (w.abs() * 2.0 ** -8 if name not in ("state", "d_state") else 0)
        finite = torch.isfinite(w)
        assert torch.equal(r.isnan(), w.isnan()), f"{name}: NaN in {int((r.isnan() & ~w.isnan()).sum())} places too many"
        assert torch.equal(torch.where(r.isinf(), r, 0.0), torch.where(w.isinf(), w, 0.0)), f"{name}: other infinities"
        assert ((r - w).abs() <= bound)[finite].all(), name
    return want


SHAPES = [(2, 100, 2, 24, 20), (2, 100, 2, 32, 32), (2, 100, 2, 64, 64), (2, 100, 2, 40, 56), (2, 70, 1, 128, 128), (2, 100, 1, 96, 16),
          (1, 2500, 1, 40, 24), (1, 1800, 1, 128, 72)]        # the last two: long axes in segments


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("where", ["q", "k", "v", "d_out", "state", "d_state"])
def test_infinities_stay_infinities(memory, shape, dtype, where):
    print(f"[infinities] {shape} {dtype} {where}", flush=True)
    x = _case(len(where), *shape, dtype)
    b, t, h, dk, dv = shape
    y = x[where]
    if where in ("state", "d_state"):
        y[0, 0, dk // 3, dv // 2] = math.inf
        y[-1, -1, dk - 1, 0] = -math.inf
    else:
        y[0, t // 2, 0, 3] = math.inf
        y[-1, t - 20, -1, y.shape[-1] - 1] = -math.inf
    want = _check(memory, x)
    assert any(w.isinf().any() for w in want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_does_not_see_them_stays_finite(memory, shape, dtype, bad):
    """Plies before a start, after, in padding, and a state that a start discards."""
    print(f"[bad plies] {shape} {dtype} {bad}", flush=True)
    x = _case(int(shape[-1]), *shape, dtype)
    b, t, h, dk, dv = shape
    x["starts"][:, t // 2 + 3] = True
    for n in ("q", "k", "v", "d_out"):
        x[n][0, t // 2] = bad                                   # three plies before a start
        x[n][0, t - 3, :, 1] = bad
        x[n][-1, t - 10:] = bad                                 # padding, where there are two games
    if b > 1:
        x["lengths"] = torch.tensor([t, t - 10], dtype=torch.int32, device="cuda")
        x["starts"][1, 0] = True
        x["state"][1] = bad
    want = _check(memory, x)
    assert torch.isfinite(want[0]).any() and not torch.isfinite(want[0]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("decay", [-2.0, -math.inf])
@pytest.mark.parametrize("shape", [(2, 90, 1, 64, 64), (1, 2500, 1, 32, 32), (1, 2500, 1, 128, 96)])
def test_an_infinity_under_a_strong_decay(memory, shape, dtype, decay):
    """A power of the decay that float32 holds as 0 is not 0: an infinity stays one. A decay of 0
    makes NaN of it."""
    print(f"[strong decay] {shape} {dtype} {decay}", flush=True)
    x = _case(3, *shape, dtype)
    x["log_decay"][:] = decay
    x["state"][0, 0, 5, 7] = math.inf
    x["d_state"][0, 0, 6, 8] = -math.inf
    _check(memory, x)
