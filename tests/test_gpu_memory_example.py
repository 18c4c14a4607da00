"""The example policy: plies played one by one and the segment that is learned from
give the same logits, and an update reaches every parameter."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_play_and_learn():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import memory_policy as E
    import junqi_amd
    torch.manual_seed(1)
    games, plies = 24, 40
    r = junqi_amd.GpuRollout(games, show_mode=2, max_num_moves=25)   # games end and start inside a segment
    r.reset(3)
    policy = E.MemoryPolicy(dtype=torch.float32).to(r.device)
    state = policy.new_state(games, r.device)
    began = torch.zeros(games, dtype=torch.int32, device=r.device)
    buf = E.rollout(policy, r, state, began, 10, seed=1)
    buf = E.rollout(policy, r, state, buf["began"], plies, seed=2)   # from the state that the first left
    assert buf["starts"].any() and not buf["starts"][0].all()
    buf["rewards"] = torch.randn(plies, games, device=r.device)   # games of 25 plies are draws without one
    loss, logits = E.loss_of(policy, buf)
    # float32 throughout: two orders of summing products of normed rows (a few hundred roundings of 2^-24)
    # through layers of weights of order 1
    scale = buf["logits"].abs().max()
    assert (logits - buf["logits"]).abs().max() <= 2048 * 2.0 ** -24 * max(1.0, scale.item())
    loss.backward()
    for name, p in policy.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        assert p.grad.any(), name
