"""The example policy holds a seat's last moves against their repetition, as its own penalties say."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_the_last_moves_change_the_logits():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import junqi_amd
    import selective_policy as E
    torch.manual_seed(1)
    games = 20
    r = junqi_amd.GpuRollout(games, show_mode=2, max_num_moves=1200)
    r.reset(3)
    policy = E.SelectivePolicy(dtype=torch.float32).to(r.device)
    buf = E.rollout(policy, r, policy.new_state(games, r.device), torch.zeros(games, dtype=torch.int32, device=r.device), 60, seed=1)
    legal = buf["logits"].isfinite()
    count = torch.zeros(*legal.shape, device=legal.device)
    recent = buf["recent"].long()
    count.scatter_add_(-1, recent.clamp(min=0), (recent >= 0).float())
    named = legal & (count > 0)
    assert named.any()            # a move back and forth within a seat's last ones is legal again
    raw = torch.randn(*legal.shape, generator=torch.Generator("cuda").manual_seed(2), device=legal.device)
    with torch.no_grad():
        got = policy.answer(raw, buf["legal"], buf["recent"])
        bias = policy.actions_bias.expand_as(raw)
    p = {k: torch.tensor(v, dtype=torch.float32).double().item() for k, v in E.PENALTIES.items()}
    x = raw.double()
    want = torch.where(x > 0, x / p["repetition"], x * p["repetition"]) - p["frequency"] * count - p["presence"] + bias
    # a quotient, a product's and three sums' roundings of at most the terms' magnitudes
    size = x.abs() * p["repetition"] + p["frequency"] * count + p["presence"] + bias.abs()
    assert ((got - want).abs() <= 6 * 2.0 ** -24 * size)[named].all()
    assert (got != raw + bias)[named].all()
    plain = legal & (count == 0)
    assert torch.equal(got[plain], (raw + bias)[plain])
