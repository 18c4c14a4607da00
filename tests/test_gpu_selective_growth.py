"""The selective scan over split axes whose decays, taken over many plies at once, leave
float32: rates above 1 ply after ply, and rates whose product is below its smallest number.
Against the definition in 64 bits (tests/selective_oracle.py)."""

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


def _inputs(b, t, d, n, dtype, step, rate, starts=()):
    """Steps of `step` without a softplus, rates of about `rate`: decays of exp(step * rate)."""
    g = torch.Generator().manual_seed(b + t + d + n)

    def rows(*last):
        return torch.randn(b, t, *last, generator=g).to(dtype)
    x = {"u": rows(d), "delta": torch.full((b, t, d), step).to(dtype), "gate": None, "b": rows(1, n), "c": rows(1, n),
         "a": rate * (1.0 + 0.01 * torch.rand(d, n, generator=g)), "skip": None, "delta_bias": None, "softplus": False,
         "state": None, "lengths": None, "d_out": rows(d), "d_state": None, "starts": torch.zeros(b, t, dtype=torch.bool)}
    x["starts"][:, list(starts)] = True
    return x


def _run(memory, x):
    x = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    leaves = {k: x[k].requires_grad_() for k in ("u", "delta", "a", "b", "c", "state") if x[k] is not None}
    out, state = memory.selective_scan(x["u"], x["delta"], x["a"], x["b"], x["c"], starts=x["starts"], initial_state=x["state"],
                                       return_state=True)
    res = ([out, state], [x["d_out"], x["d_state"]]) if x["d_state"] is not None else ([out], [x["d_out"]])
    return {"out": out, "state": state, **dict(zip(("d_" + k for k in leaves), torch.autograd.grad(res[0], list(leaves.values()), res[1])))}


def _check(memory, x, most, plies):
    """`most`: largest magnitude of the sum of a chain's exponents, `plies` of a chain. An exponent
    dt * a is off by 2 roundings of it (a in powers of 2, the product), a power by one step more;
    over a part the steps are added first, which rounds each of its sums, at most the whole, once
    a ply; that times the rate is rounded twice more."""
    c = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in x.items()}
    want, size = O.scan(c), O.scan(c, size=True)
    steps = (2 + plies + 2) * most + 4 * plies + x["a"].shape[1] + x["u"].shape[2] + x["u"].shape[0] * x["u"].shape[1] + 40
    got = _run(memory, x)
    for k, v in got.items():
        assert (want[k].abs() < torch.finfo(F32).max).all(), k
        dtype = x["u"].dtype if k == "out" else F32 if k == "state" else x[k[2:]].dtype
        O.close(k, v, want[k], size[k], steps, dtype)
    return got, want


# channels, states: a lane's, many of a block's, fewer than a wave
SIZES = [(64, 16), (70, 24), (3, 1)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", SIZES)
def test_nothing_grows_to_nothing(memory, size, sign, dtype):
    """States, and gradients, that are 0 stay 0 over plies that would make 1 pass float32's end
    (2^3 a ply, parts of 80), steps back or rates above 0."""
    x = _inputs(1, 320, *size, dtype, 2.0 * sign, 1.04 * sign, starts=(20, 45, 290))   # no chain of more than 30 plies, e^63
    quiet = torch.ones(320, dtype=torch.bool)
    quiet[20:45] = quiet[300:] = False
    x["u"][:, quiet] = 0
    quiet[20:45] = True           # what reaches back from the last plies ends at ply 290
    quiet[25:44] = False
    x["d_out"][:, quiet] = 0
    got, want = _check(memory, x, 2.0 * 1.06 * 30, 30)
    assert got["d_u"].any() and got["state"].any() and got["d_a"].any()
    y = {**x, "starts": x["starts"].cuda()}
    plain = memory.selective_scan(*(y[k].cuda() for k in ("u", "delta", "a", "b", "c")), starts=y["starts"])
    assert torch.equal(plain, got["out"])


@pytest.mark.parametrize("size", SIZES)
def test_small_states_grow(memory, size):
    """A state of 1e-30 and a gradient of 1e-30 grow by 2^173 over a part: they stay numbers."""
    x = _inputs(1, 320, *size, F32, 1.0, 1.5, starts=(82, 238))
    x["u"].zero_()
    x["d_out"].zero_()
    g = torch.Generator().manual_seed(1)
    x["state"] = 1e-30 * torch.randn(1, *size, generator=g)
    x["d_state"] = 1e-30 * torch.randn(1, *size, generator=g)
    x["d_out"][:, 75:82] = 1e-30 * torch.randn(1, 7, size[0], generator=g)
    # of the state's end, which ply 238 hides from the beginning, and of the plies before 82
    _check(memory, x, 1.5 * 1.01 * 82, 82)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", SIZES)
def test_what_dies_is_dead(memory, size, dtype):
    """A state of 1e38 over parts whose decay is e^-1600 leaves nothing, not its product with
    float32's smallest number; nor does a gradient."""
    x = _inputs(1, 320, *size, dtype, 1.0, -20.0)
    x["u"].zero_()
    x["d_out"].zero_()
    x["state"] = torch.full((1, *size), 1e38)
    x["c"] = torch.ones_like(x["c"])
    got = _run(memory, x)
    # after 11 decays of at most e^-20 the sum of at most 24 states is below 2.4e39 e^-220 < 1e-56,
    # where float32's smallest number is 1.4e-45
    assert not got["out"][:, 10:].any() and not got["state"].any()
    x["state"], x["d_state"] = None, torch.full((1, *size), 1e38)
    got = _run(memory, x)
    assert got["d_b"].shape == x["b"].shape and not got["d_u"][:, :-11].any()   # b below 100


def test_infinities_stay(memory):
    """An infinity is one over any number of plies, behind decays and behind powers above 1."""
    for rate in (-0.5, 0.3):
        x = _inputs(1, 320, 64, 16, F32, 1.0, rate, starts=(300,) if rate > 0 else ())
        x["u"][:, 1:] = 0
        x["u"][:, :1] = 1e-30
        x["u"][0, 0, 5] = float("inf")
        x["b"] = x["b"].abs() + 0.5
        got = memory.selective_scan(*(x[k].cuda() for k in ("u", "delta", "a", "b", "c")), starts=x["starts"].cuda(), return_state=True)
        end = 300 if rate > 0 else 320
        for t in (0, 100, 200, end - 1):
            assert not got[0][0, t, 5].isfinite(), t
            assert got[0][0, t, 6].isfinite() or rate > 0
        assert bool(got[1][0, 5].isinf().all()) == (rate < 0)
        assert got[1][0, 6].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("plies", [20, 320])
@pytest.mark.parametrize("size", SIZES)
def test_a_start_has_no_decay(memory, size, plies, dtype):
    """The ply that starts a game, also with a decay past float32's end, sees its input alone:
    in segments, whole and split, as one ply by itself."""
    at = (0, 7, plies - 5)
    x = _inputs(2, plies, *size, dtype, 1.0, 0.01, starts=at)
    x["delta"][:, list(at)] = 9984.0     # e^99.8 to e^100.8; a number of bfloat16 too
    g = torch.Generator().manual_seed(5)
    x["state"] = torch.randn(2, *size, generator=g)
    got, _ = _check(memory, x, 0.0101 * plies, plies)
    y = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    state = y["state"].clone()
    for t in range(8):
        out = memory.selective_scan_step(y["u"][:, t], y["delta"][:, t], y["a"], y["b"][:, t], y["c"][:, t], state, starts=y["starts"][:, t])
        assert out.isfinite().all() and got["out"][:, t].isfinite().all()
        if t in at:
            assert (state - (y["delta"][:, t, :, None].float() * y["u"][:, t, :, None].float()) * y["b"][:, t].float()).abs().max() <= \
                2.0 ** -23 * state.abs().max()
