"""The example policy with a selective memory: convolution, scan and masked logits together,
as they are used. Plies played one by one and the segment that is learned from give the
same logits, an update reaches every parameter, and seats learn nothing of each other."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def played():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected on a machine without a visible GPU")
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import junqi_amd
    import selective_policy as E
    torch.manual_seed(1)
    games, plies = 20, 40
    r = junqi_amd.GpuRollout(games, show_mode=2, max_num_moves=25)   # games end and start inside a segment
    r.reset(3)
    policy = E.SelectivePolicy(dtype=torch.float32).to(r.device)
    state = policy.new_state(games, r.device)
    began = torch.zeros(games, dtype=torch.int32, device=r.device)
    buf = E.rollout(policy, r, state, began, 10, seed=1)
    buf = E.rollout(policy, r, state, buf["began"], plies, seed=2)   # from the memories that the first left
    return E, policy, buf


def test_play_and_learn(played):
    E, policy, buf = played
    assert buf["starts"].any() and not buf["starts"][0].all()
    buf = dict(buf, rewards=torch.randn(buf["rewards"].shape, device=buf["rewards"].device))
    loss, logits = E.loss_of(policy, buf)
    legal = logits.isfinite()
    assert torch.equal(legal, buf["logits"].isfinite()) and legal.any(-1).all()
    assert legal.gather(-1, buf["actions"][..., None]).all()
    # float32 throughout: two orders of summing products of normed rows (a few hundred roundings of 2^-24)
    # through layers of weights of order 1
    scale = buf["logits"][legal].abs().max()
    assert (logits - buf["logits"])[legal].abs().max() <= 2048 * 2.0 ** -24 * max(1.0, scale.item())
    loss.backward()
    for name, p in policy.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
        assert p.grad.any(), name
    policy.zero_grad()


def test_the_masks_are_the_environments(played):
    """The words that were stored leave the actions that the logits have, and the last moves change them."""
    E, policy, buf = played
    words = buf["legal"]
    bits = (words[..., None] >> torch.arange(32, device=words.device)) & 1
    assert torch.equal(bits.flatten(-2)[..., :E.ACTIONS].bool(), buf["logits"].isfinite())
    raw = torch.randn(*words.shape[:2], E.ACTIONS, device=words.device)
    with torch.no_grad():
        with_moves = policy.answer(raw, words, buf["recent"])
        without = policy.answer(raw, words, torch.full_like(buf["recent"], -1))
    named = torch.zeros_like(with_moves, dtype=torch.bool)
    recent = buf["recent"].long()
    named.scatter_(-1, recent.clamp(min=0), recent >= 0)
    named |= torch.zeros_like(named).scatter_(-1, recent.clamp(min=0), True) & (recent == 0).any(-1, keepdim=True)
    legal = with_moves.isfinite()
    assert torch.equal(with_moves[legal & ~named], without[legal & ~named])


def test_a_seat_sees_only_its_own_plies(played):
    E, policy, buf = played
    with torch.no_grad():
        _, logits = E.loss_of(policy, buf)
        legal = logits.isfinite()
        bound = 2048 * 2.0 ** -24 * max(1.0, logits[legal].abs().max().item())
        for s in range(4):
            mine = buf["seats"] == s
            other = dict(buf, glob=torch.where(mine[..., None], buf["glob"] + torch.randn_like(buf["glob"]), buf["glob"]))
            moved = torch.where(legal, E.loss_of(policy, other)[1] - logits, 0.0).abs().amax(-1)
            assert (moved[~mine] <= bound).all(), f"seat {s} reaches others"
            assert (moved[mine] > bound).any(), f"seat {s} reaches itself"


def test_a_run_in_bfloat16(played):
    import junqi_amd
    E = played[0]
    torch.manual_seed(2)
    r = junqi_amd.GpuRollout(12, show_mode=2, max_num_moves=1200)
    r.reset(1)
    policy = E.SelectivePolicy().to(r.device)
    opt = torch.optim.Adam(policy.parameters(), lr=1e-3)
    state, began = policy.new_state(12, r.device), torch.zeros(12, dtype=torch.int32, device=r.device)
    for u in range(2):
        buf = E.rollout(policy, r, state, began, 9, seed=u)
        began = buf["began"]
        loss, _ = E.loss_of(policy, buf)
        opt.zero_grad()
        loss.backward()
        opt.step()
        assert torch.isfinite(loss)
        assert all(torch.isfinite(p).all() for p in policy.parameters())
