"""The example policy's seats: the pieces are hidden, so what one seat observed reaches no
other seat's logits, neither while playing nor in the segment that is learned from."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_a_seat_sees_only_its_own_plies():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import memory_policy as E
    import junqi_amd
    torch.manual_seed(2)
    games, plies = 16, 30
    r = junqi_amd.GpuRollout(games, show_mode=2, max_num_moves=21)
    r.reset(5)
    policy = E.MemoryPolicy(dtype=torch.float32).to(r.device)
    state, began = policy.new_state(games, r.device), torch.zeros(games, dtype=torch.int32, device=r.device)
    buf = E.rollout(policy, r, state, began, 7, seed=3)
    buf = E.rollout(policy, r, state, buf["began"], plies, seed=4)
    _, logits = E.loss_of(policy, buf)
    seat = buf["positions"][..., 1]                              # (plies, games)
    bound = 2048 * 2.0 ** -24 * max(1.0, logits.abs().max().item())   # float32 sums through layers of weights of order 1
    for s in range(4):
        other = dict(buf, glob=torch.where((seat == s)[..., None], buf["glob"] + torch.randn_like(buf["glob"]), buf["glob"]))
        moved = (E.loss_of(policy, other)[1] - logits).abs().amax(-1)
        assert (moved[seat != s] <= bound).all(), f"seat {s} reaches others"
        assert (moved[seat == s] > bound).any(), f"seat {s} reaches itself"


def test_a_ply_moves_only_the_acting_seats_memory():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import memory_policy as E
    games, dev = 5, torch.device("cuda")
    torch.manual_seed(3)
    policy = E.MemoryPolicy().to(dev)
    state = torch.randn_like(policy.new_state(games, dev))
    before = state.clone().view(games, 4, -1)
    seat = torch.tensor([0, 1, 2, 3, 1], device=dev)
    positions = torch.stack([torch.full_like(seat, 9), seat], -1).int()
    policy.play(torch.randn(games, E.GLOBALS, device=dev), positions, state, torch.tensor([0, 0, 1, 0, 0], device=dev).bool())
    after = state.view(games, 4, -1)
    for g in range(games):
        for s in range(4):
            if g == 2 and s != 2:
                assert not after[g, s].any()                     # its game starts with this ply
            else:
                assert torch.equal(after[g, s], before[g, s]) == (s != seat[g])
