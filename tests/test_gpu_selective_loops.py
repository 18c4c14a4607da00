"""Calls of so many games that a wave or thread takes several, one after another: the loops that
large calls live in, with rows left out on the way, sums over several games, and states past the
caches. Against calls on parts of them, bit for bit, and the definitions in 64 bits."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import test_gpu_selective as S  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def memory():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import memory as M
    torch.cuda.empty_cache()
    yield M
    torch.cuda.empty_cache()


def _numbers(g, *shape, dtype=F32, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def _picked(g, games, rows):
    """Rows of a state in an order of their own, some of no state; and what starts."""
    pick = torch.randperm(rows, generator=g, device="cuda")[:games]
    pick[::5] = torch.tensor([-1, rows, 2 ** 40], device="cuda").repeat(-(-games // 15))[:len(pick[::5])]
    return pick, torch.rand(games, generator=g, device="cuda") < 0.1


# games, channels, states, groups, type: waves of at most 32,768 games' channels at once, so two to four
# games a wave; the last two with states past 400 MiB, which go past the caches
STEPS = [(5000, 1024, 4, 1, F32), (1500, 1024, 16, 2, BF16), (700, 1000, 33, 1, F32), (3000, 1030, 3, 1, BF16),
         (13001, 512, 16, 1, BF16), (3300, 1024, 33, 1, F32)]


@pytest.mark.parametrize("shape", STEPS)
def test_scan_steps(memory, shape):
    games, d, n, groups, dtype = shape
    g = torch.Generator("cuda").manual_seed(games)
    u, delta, gate = (_numbers(g, games, d, dtype=dtype) for _ in range(3))
    b, c = (_numbers(g, games, groups, n, dtype=dtype) for _ in range(2))
    a, skip, bias = -torch.rand(d, n, generator=g, device="cuda") * n, _numbers(g, d), _numbers(g, d) - 3.0
    rows = games + games // 3
    start = _numbers(g, rows, d, n)
    pick, starts = _picked(g, games, rows)

    def call(state, at):
        return memory.selective_scan_step(u[at], delta[at], a, b[at], c[at], state, skip=skip, gate=gate[at], delta_bias=bias,
                                          softplus=True, rows=pick[at], starts=starts[at])
    whole, parts = start.clone(), start.clone()
    out = call(whole, slice(None))
    for i in range(0, games, 97):       # one game a wave
        assert torch.equal(out[i:i + 97], call(parts, slice(i, i + 97))), i
    assert torch.equal(whole, parts) and not torch.equal(whole, start)
    gone = (pick < 0) | (pick >= rows)
    assert not out[gone].any() and out[~gone].any(1).all()


@pytest.mark.parametrize("shape", [(12000, 520, 4, BF16), (8000, 520, 8, F32), (9000, 1026, 3, BF16)])
def test_conv_steps(memory, shape):
    games, d, taps, dtype = shape
    g = torch.Generator("cuda").manual_seed(games)
    x, weight, bias = _numbers(g, games, d, dtype=dtype), _numbers(g, d, taps), _numbers(g, d)
    rows = games + games // 3
    start = _numbers(g, rows, taps - 1, d, dtype=dtype)
    pick, starts = _picked(g, games, rows)

    def call(state, at):
        return memory.causal_conv_step(x[at], weight, state, bias, silu=True, rows=pick[at], starts=starts[at])
    whole, parts = start.clone(), start.clone()
    out = call(whole, slice(None))
    for i in range(0, games, 500):      # one game a thread
        assert torch.equal(out[i:i + 500], call(parts, slice(i, i + 500))), i
    assert torch.equal(whole, parts) and not torch.equal(whole, start)
    gone = (pick < 0) | (pick >= rows)
    assert not out[gone].any() and out[~gone].any(1).all()


# games, plies, channels, states, groups: more games (and parts of an axis) than waves of a channel's
# gradients; all the channels and states of a wave, not all of them, several waves of states, split axes
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(300, 9, 1024, 16, 1), (300, 5, 1000, 12, 2), (150, 6, 512, 64, 1), (100, 5, 520, 33, 1), (4, 1280, 2048, 4, 1)])
def test_sums_of_several_games(memory, shape, dtype):
    x = S._scan_inputs(sum(shape), *shape, dtype=dtype)
    S._check_scan(memory, x)


@pytest.mark.parametrize("shape,types", [((1500, 4, 520, 4), (F32, F32)), ((1500, 4, 520, 4), (BF16, F32)), ((1500, 4, 520, 4), (BF16, BF16)),
                                         ((1400, 3, 516, 7), (BF16, F32))])
def test_sums_of_several_games_of_the_convolution(memory, shape, types):
    S._check_conv(memory, S._conv_inputs(sum(shape), *shape, dtype=types[0], wdtype=types[1]))


def test_segments_of_the_most_channels(memory):
    """2^20 channels leave the grid 64 games' waves (4 of a block) and 2,048 rows of threads."""
    d, games = 1 << 20, 150
    g = torch.Generator("cuda").manual_seed(1)
    for n in (1, 17):
        u, delta = (_numbers(g, games, 2, d, dtype=BF16) for _ in range(2))
        b, c = (_numbers(g, games, 2, n, dtype=BF16) for _ in range(2))
        a = -torch.rand(d, n, generator=g, device="cuda")
        lengths = torch.randint(0, 3, (games,), generator=g, device="cuda", dtype=torch.int32)
        lengths[-3:] = 2

        def call(at):
            return memory.selective_scan(u[at], delta[at], a, b[at], c[at], softplus=True, lengths=lengths[at])
        out = call(slice(None))
        for at in (slice(0, 5), slice(64, 70), slice(games - 5, games)):
            assert torch.equal(out[at], call(at))
        assert out[-1].any() and not out[lengths == 0].any()
        del u, delta, out
    games = 2100
    x = _numbers(g, 50, 1, d, dtype=BF16).repeat(42, 1, 1)
    x *= (1 + torch.arange(games, device="cuda") % 7)[:, None, None].to(BF16)
    weight = _numbers(g, d, 4)
    out = memory.causal_conv(x, weight, silu=True)
    for at in (slice(0, 3), slice(games - 60, games)):
        assert torch.equal(out[at], memory.causal_conv(x[at], weight, silu=True))


def test_gradients_of_many_groups_of_states(memory):
    """db and dc of more values than the threads that join them."""
    games, plies, d, n = 40000, 32, 64, 64
    g = torch.Generator("cuda").manual_seed(2)
    u, delta = (_numbers(g, games, plies, d, dtype=BF16) for _ in range(2))
    b, c = (_numbers(g, games, plies, n, dtype=BF16) for _ in range(2))
    a = -torch.rand(d, n, generator=g, device="cuda")

    def call(at):
        leaves = [t[at].clone().requires_grad_() for t in (b, c)]
        out = memory.selective_scan(u[at], delta[at], a, *leaves, softplus=True)
        return torch.autograd.grad(out, leaves, u[at])
    whole = call(slice(None))
    for at in (slice(0, 40), slice(games // 2, games // 2 + 40), slice(games - 40, games)):
        for p, q in zip(whole, call(at)):
            assert torch.equal(p[at], q) and q.any()


def test_logits_of_more_rows_than_waves():
    from junqi_amd import masks
    n, acts = 2 ** 25 + 1001, 3
    g = torch.Generator("cuda").manual_seed(3)
    x = _numbers(g, n, acts, dtype=BF16)
    legal = torch.rand(n, acts, generator=g, device="cuda") < 0.7
    recent = torch.randint(-1, acts + 1, (n, 2), generator=g, device="cuda", dtype=torch.int32)
    bias = _numbers(g, acts)

    def call(at):
        leaf = x[at].clone().requires_grad_()
        out = masks.action_logits(leaf, bias=bias, legal=legal[at], recent=recent[at], repetition=1.5, frequency=0.1, presence=0.2)
        return out.detach(), torch.autograd.grad(out, leaf, x[at])[0]
    whole = call(slice(None))
    for at in (slice(0, 1001), slice(2 ** 25 - 500, 2 ** 25 + 500), slice(n - 1001, n)):
        for p, q in zip(whole, call(at)):
            assert torch.equal(p[at], q)
    torch.cuda.empty_cache()


MASKS = [("none", "none", False), ("some", "some", True), ("all", "none", True)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("masks", range(3))
@pytest.mark.parametrize("shape", range(len(S.SHAPES)))
def test_scan_of_the_same_numbers_every_time(memory, shape, masks, dtype):
    """The shapes and masks of test_gpu_selective.test_scan, whose seeds differ from process to process."""
    starts, lengths, state = MASKS[masks]
    S._check_scan(memory, S._scan_inputs(1000 + 10 * shape + masks, *S.SHAPES[shape], dtype=dtype, starts=starts, lengths=lengths, state=state))
