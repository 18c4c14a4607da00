"""That the check of mean errors sees what it is there for: the same definition in
chunks, in 64 bits, with one operand at a time held in fewer bits or one ply left out."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import memory_oracle as O  # noqa: E402

CHUNK = 32


def _parts(x, n):
    """x as a sum of n bfloat16 terms (None: as it is)."""
    if n is None:
        return x
    y = torch.zeros_like(x)
    for _ in range(n):
        y = y + (x - y).to(torch.bfloat16).double()
    return y


def _chunked(q, k, v, log_decay, state, scale, state_parts=None, p_parts=None, forget=None):
    """Outputs and the last state of (T, D) rows of one head, without starts."""
    out, lam = [], torch.exp(log_decay)
    for a in range(0, q.shape[0], CHUNK):
        x, y, z = (r[a:a + CHUNK] for r in (q, k, v))
        i = torch.arange(x.shape[0], dtype=torch.float64)
        p = (x @ y.T) * torch.where(i[:, None] >= i, lam ** (i[:, None] - i), 0.0) * scale
        out.append(_parts(p, p_parts) @ z + scale * lam ** (i[:, None] + 1) * (x @ _parts(state, state_parts)))
        left = lam ** (len(i) - 1 - i)
        if forget is not None and len(i) > forget:
            left[forget] = 0.0
        state = lam ** len(i) * state + (y * left[:, None]).T @ z
    return torch.cat(out), state


def _case(seed, t, dk, dv, memory):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(t, d, generator=g).to(torch.bfloat16).double() for d in (dk, dk, dv))
    return q, k, v, torch.tensor(-1.0 / memory, dtype=torch.float64), torch.randn(dk, dv, generator=g).double(), dk ** -0.5


def _check(case, **how):
    q, k, v, decay, state, scale = case
    args = (q[None, :, None], k[None, :, None], v[None, :, None], decay[None], None, None, state[None, None], scale)
    want, terms = O.define(*args), O.spread(*args)
    out, last = _chunked(*case, **how)
    O.check_rms("out", out.to(torch.bfloat16)[None, :, None], want[0], terms[0], torch.bfloat16)
    O.check_rms("state", last.float()[None, None], want[1], terms[1], torch.bfloat16)


CASES = [(500, 32, 32, 40), (300, 64, 36, 100), (200, 24, 128, 20), (129, 128, 96, 256), (70, 40, 56, 8)]


@pytest.mark.parametrize("t,dk,dv,memory", CASES)
def test_what_is_held_in_enough_bits_passes(t, dk, dv, memory):
    _check(_case(t, t, dk, dv, memory))
    _check(_case(t, t, dk, dv, memory), state_parts=2, p_parts=2)


@pytest.mark.parametrize("how", [{"state_parts": 1}, {"p_parts": 1}, {"state_parts": 2, "p_parts": 1}, {"forget": 31}, {"forget": 0}])
@pytest.mark.parametrize("t,dk,dv,memory", CASES)
def test_fewer_bits_and_a_lost_ply_are_seen(t, dk, dv, memory, how):
    with pytest.raises(AssertionError, match="off by"):
        _check(_case(t, t, dk, dv, memory), **how)
