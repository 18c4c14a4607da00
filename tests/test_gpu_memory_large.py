"""Linear attention over more than the caches hold (420 MB of rows or states): the kernels that
go past them, on an MI355X, against the definition in 64 bits."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import memory_oracle as O  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
EPS = 2.0 ** -24
STREAM_BYTES = 400 << 20


@pytest.fixture(scope="module")
def memory():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    from junqi_amd import memory as M
    return M


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("games,heads,key_dim,value_dim,offset", [(28000, 1, 64, 64, 0), (28000, 1, 64, 64, 1), (15000, 2, 40, 96, 0),
                                                                  (8000, 1, 128, 112, 3)])
def test_one_ply_of_many_games(memory, dtype, games, heads, key_dim, value_dim, offset):
    g = torch.Generator("cuda").manual_seed(value_dim + offset)
    rest = 100                                                  # states that no game has
    size = (games + rest) * heads * key_dim * value_dim
    assert games * heads * key_dim * value_dim * 4 > STREAM_BYTES and value_dim % 4 == 0
    store = torch.randn(size + 8, device="cuda", generator=g)
    state = store[offset:offset + size].view(games + rest, heads, key_dim, value_dim)
    before = store.clone()
    q, k = (torch.randn(games, heads, key_dim, device="cuda", generator=g).to(dtype) for _ in range(2))
    v = torch.randn(games, heads, value_dim, device="cuda", generator=g).to(dtype)
    starts = torch.rand(games, device="cuda", generator=g) < 0.1
    rows = torch.randperm(games + rest, device="cuda", generator=g)[:games]
    rows[::1000] = -1                                           # left out
    decay = -torch.rand(heads, device="cuda", generator=g)
    out = memory.linear_attention_step(q, k, v, decay, state, rows=rows, starts=starts)
    on = rows >= 0
    assert torch.equal(store[:offset], before[:offset]) and torch.equal(store[offset + size:], before[offset + size:])
    held = before[offset:offset + size].view_as(state)
    still = torch.ones(games + rest, dtype=torch.bool, device="cuda")
    still[rows[on]] = False
    assert torch.equal(state[still], held[still]) and not out[~on].any()
    for part in torch.arange(games, device="cuda")[on].split(4000):     # in 64 bits, some at a time
        old = held[rows[part]].double()
        lam = torch.where(starts[part, None], 0.0, decay.double().exp())[..., None, None]
        kv = k[part].double()[..., :, None] * v[part].double()[..., None, :]
        want = lam * old + kv
        mag = lam * old.abs() + kv.abs()
        assert ((state[rows[part]].double() - want).abs() <= mag * 8 * EPS).all()
        scale = key_dim ** -0.5
        answer = (q[part].double()[..., None] * want).sum(-2) * scale
        bound = (q[part].double().abs()[..., None] * mag).sum(-2) * scale * (key_dim + 8) * EPS
        if dtype == BF16:
            bound = bound + answer.abs() * 2.0 ** -8
        assert ((out[part].double() - answer).abs() <= bound).all()


@pytest.mark.parametrize("dtype,games", [(BF16, 280), (F32, 140)])
@pytest.mark.parametrize("plies,heads,key_dim,value_dim", [(400, 8, 64, 64), (200, 8, 128, 128), (800, 8, 32, 32)])
def test_segments_of_many_games(memory, dtype, games, plies, heads, key_dim, value_dim):
    g = torch.Generator("cuda").manual_seed(key_dim)
    b, t, h, dk, dv = games, plies, heads, key_dim, value_dim
    assert b * t * h * (dk + dv) * 2 * (2 if dtype == BF16 else 4) > STREAM_BYTES

    def rows(d):    # out of time-major buffers
        return torch.randn(t, b, h, d, device="cuda", generator=g).to(dtype).transpose(0, 1)
    q, k, v, d_out = rows(dk), rows(dk), rows(dv), rows(dv)
    state, d_state = (torch.randn(b, h, dk, dv, device="cuda", generator=g) for _ in range(2))
    decay = -torch.exp2(-8 * torch.rand(h, device="cuda", generator=g))
    starts = torch.rand(b, t, device="cuda", generator=g) < 0.01
    lengths = torch.randint(t // 2, t + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
    leaves = [x.detach().requires_grad_() for x in (q, k, v, state)]
    out, last = memory.linear_attention(*leaves[:3], decay, starts=starts, lengths=lengths, initial_state=leaves[3],
                                        return_state=True)
    got = (out, last, *torch.autograd.grad([out, last], leaves, [d_out, d_state]))
    some = torch.tensor([0, 1, b // 2, b - 1], device="cuda")
    args = (*(x[some].double() for x in (q, k, v)), decay.double(), starts[some], lengths[some], state[some].double(), dk ** -0.5,
            d_out[some].double(), d_state[some].double())
    want, terms = O.define(*args), O.spread(*args)
    for name, x, w, s in zip(O.NAMES, got, want, terms):
        O.check_rms(name, x.detach()[some], w, s, dtype)
    # the others: finite, and 0 past each game's end
    past = torch.arange(t, device="cuda") >= lengths[:, None]
    for x in (got[0], *got[2:5]):
        assert torch.isfinite(x).all() and not x.detach()[past].any()
