"""A policy whose memory forgets as the plies tell it to, playing and learning on the GPU.

As in memory_policy.py each seat of a game keeps a memory of its own, here the last
inputs of a short convolution and the states of a selective scan, in row game * 4 +
seat. While playing, a ply's token goes through `layer_norm`, `causal_conv_step` and
`selective_scan_step`, and its answer through `action_logits`, which takes the
environment's packed legal masks as they are and holds the seat's last moves against
their repetition. An update runs the same network over the stored segment with
`causal_conv` and `selective_scan`, each seat's plies one after another, and learns from
the rewards (REINFORCE) through the masked logits.

  python examples/selective_policy.py [games] [plies] [updates]
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
sys.path.insert(0, str(Path(__file__).resolve().parent))
import junqi_amd  # noqa: E402
from junqi_amd import masks, memory  # noqa: E402
from memory_policy import ACTIONS, EATS, GLOBALS, KILLED, SEATS, WIDTH, Norm, seat_rows  # noqa: E402

CHANNELS, STATES, TAPS = 2 * WIDTH, 16, 4
RECENT = 16            # moves of a seat that its next ones are held against
PENALTIES = {"repetition": 1.2, "frequency": 0.1, "presence": 0.2}


class SelectivePolicy(nn.Module):
    def __init__(self, rank: int = 32, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.dtype = dtype
        self.embed = nn.Linear(GLOBALS, WIDTH)
        self.norm_in, self.norm_out = Norm(), Norm()
        self.inputs = nn.Linear(WIDTH, 2 * CHANNELS, bias=False)
        self.taps = nn.Parameter(TAPS ** -0.5 * torch.randn(CHANNELS, TAPS))
        self.taps_bias = nn.Parameter(torch.zeros(CHANNELS))
        self.select = nn.Linear(CHANNELS, rank + 2 * STATES, bias=False)
        self.step = nn.Linear(rank, CHANNELS, bias=False)
        # rates of 1 to STATES times a channel's step, steps of 1/1,000 to 1/10
        self.log_rate = nn.Parameter(torch.log(torch.arange(1.0, STATES + 1)).repeat(CHANNELS, 1))
        self.step_bias = nn.Parameter(torch.log(torch.expm1(torch.exp(torch.linspace(math.log(1e-3), math.log(0.1), CHANNELS)))))
        self.skip = nn.Parameter(torch.ones(CHANNELS))
        self.mix = nn.Linear(CHANNELS, WIDTH, bias=False)
        self.out = nn.Linear(WIDTH, rank)
        self.actions = nn.Parameter(0.02 * torch.randn(rank, ACTIONS))
        self.actions_bias = nn.Parameter(torch.zeros(ACTIONS))

    def _token(self, glob):
        x = self.embed(glob)
        u, gate = self.inputs(self.norm_in(x)).to(self.dtype).chunk(2, -1)
        return x, u, gate

    def _selected(self, u):
        """What the scan takes of its inputs: delta, b and c."""
        by = self.select(u.float())
        rank = by.shape[-1] - 2 * STATES
        return self.step(by[..., :rank]).to(self.dtype), *by[..., rank:].to(self.dtype).split(STATES, -1)

    def _logits(self, x, y):
        return self.out(self.norm_out(x + self.mix(y.float()))) @ self.actions

    def answer(self, logits, legal, recent):
        """The logits of (..., actions) ready for a softmax; legal and recent: their rows'."""
        flat = masks.action_logits(logits.flatten(0, -2), bias=self.actions_bias, legal=legal.flatten(0, -2),
                                   recent=recent.flatten(0, -2), **PENALTIES)
        return flat.view_as(logits)

    def new_state(self, games: int, device) -> dict:
        rows = games * SEATS
        return {"inputs": torch.zeros(rows, TAPS - 1, CHANNELS, dtype=self.dtype, device=device),
                "states": torch.zeros(rows, CHANNELS, STATES, device=device)}

    @torch.no_grad()
    def play(self, glob, seats, state, starts):
        """Logits of one ply of every game; the acting seats' memories move on in place."""
        x, u, gate = self._token(glob)
        rows = torch.arange(len(starts), device=starts.device) * SEATS + seats
        for s in state.values():     # a game that starts anew: all of its seats' memories
            s.view(len(starts), SEATS, -1).masked_fill_(starts[:, None, None], 0)
        u = memory.causal_conv_step(u, self.taps, state["inputs"], self.taps_bias, silu=True, rows=rows)
        delta, b, c = self._selected(u)
        y = memory.selective_scan_step(u, delta, -self.log_rate.exp(), b, c, state["states"], skip=self.skip, gate=gate,
                                       delta_bias=self.step_bias, softplus=True, rows=rows)
        return self._logits(x, y)

    def forward(self, glob, seats, state, starts):
        """Logits of a segment's plies, (games, plies, ...), from the memories before it."""
        x, u, gate = self._token(glob)
        at, lengths, begins = seat_rows(seats, starts)
        rows, most = len(lengths), begins.shape[1]

        def by_seat(t):
            t = t.flatten(0, 1)
            return t.new_zeros(rows * most, t.shape[-1]).index_copy(0, at.flatten(), t).view(rows, most, -1)
        where = {"starts": begins, "lengths": lengths}
        u = memory.causal_conv(by_seat(u), self.taps, self.taps_bias, silu=True, initial_state=state["inputs"], **where)
        delta, b, c = self._selected(u)
        y = memory.selective_scan(u, delta, -self.log_rate.exp(), b, c, skip=self.skip, gate=by_seat(gate),
                                  delta_bias=self.step_bias, softplus=True, initial_state=state["states"], **where)
        return self._logits(x, y.flatten(0, 1).index_select(0, at.flatten()).view(*x.shape[:2], -1))


def rollout(policy: SelectivePolicy, r, state: dict, began: torch.Tensor, plies: int, seed: int) -> dict:
    """Play `plies` plies of every game. `began`: plies of each game so far (0: the next
    ply is its first). The buffers are time-major, (plies, games, ...)."""
    n, dev = r.num_envs, r.device
    g = torch.Generator(dev).manual_seed(seed)
    words = (ACTIONS + 31) // 32
    games = torch.arange(n, device=dev)
    last = torch.full((n, SEATS, RECENT), -1, dtype=torch.int32, device=dev)     # each seat's last moves
    buf = {"state": {k: s.clone() for k, s in state.items()}, "glob": torch.empty(plies, n, GLOBALS, device=dev),
           "seats": torch.empty(plies, n, dtype=torch.int64, device=dev), "starts": torch.empty(plies, n, dtype=torch.bool, device=dev),
           "legal": torch.empty(plies, n, words, dtype=torch.int32, device=dev),
           "recent": torch.empty(plies, n, RECENT, dtype=torch.int32, device=dev),
           "actions": torch.empty(plies, n, dtype=torch.int64, device=dev), "rewards": torch.empty(plies, n, device=dev), "logits": []}
    for t in range(plies):
        turn = r.turn_torch()
        seats = turn.long()
        _, glob = r.build_acting_seat_observation_torch(turn)
        buf["glob"][t].copy_(glob)
        buf["seats"][t], buf["starts"][t] = seats, began == 0
        last[buf["starts"][t]] = -1
        buf["legal"][t].copy_(r.batch.legal()["mask_words"].view(n, words))   # the environment writes them anew each ply
        buf["recent"][t].copy_(last[games, seats])
        logits = policy.answer(policy.play(buf["glob"][t], seats, state, buf["starts"][t]), buf["legal"][t], buf["recent"][t])
        buf["logits"].append(logits.detach())
        action = torch.multinomial(torch.softmax(logits.detach().float(), -1), 1, generator=g).squeeze(1)
        buf["actions"][t] = action
        last[games, seats] = torch.cat([last[games, seats][:, 1:], action.to(torch.int32)[:, None]], 1)
        step = r.step_device_torch(action.to(torch.int32), turn)
        event = step["event"]
        buf["rewards"][t] = step["rewards"] + 0.1 * (event == EATS).float() - 0.1 * (event == KILLED).float()
        began = torch.where(step["terminated"].bool(), 0, began + 1)
        r.update_beliefs_device(step, turn)
        r.reset_terminated_device(seed=seed + t)
    buf["logits"] = torch.stack(buf["logits"])
    buf["began"] = began
    return buf


def loss_of(policy: SelectivePolicy, buf: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """REINFORCE over the segment; also the masked logits, (plies, games, actions)."""
    by_game = {k: buf[k].transpose(0, 1) for k in ("glob", "seats", "starts")}
    logits = policy(by_game["glob"], by_game["seats"], buf["state"], by_game["starts"]).transpose(0, 1)
    logits = policy.answer(logits.contiguous(), buf["legal"], buf["recent"])
    taken = torch.log_softmax(logits.float(), -1).gather(-1, buf["actions"][..., None]).squeeze(-1)
    gain = buf["rewards"] - buf["rewards"].mean()
    return -(gain * taken).mean(), logits


def main(games: int = 256, plies: int = 64, updates: int = 3) -> None:
    torch.manual_seed(0)
    r = junqi_amd.GpuRollout(games, show_mode=2, max_num_moves=1200)
    r.reset(0)
    policy = SelectivePolicy().to(r.device)
    opt = torch.optim.Adam(policy.parameters(), lr=1e-3)
    state, began = policy.new_state(games, r.device), torch.zeros(games, dtype=torch.int32, device=r.device)
    for u in range(updates):
        buf = rollout(policy, r, state, began, plies, seed=1000 * u)
        began = buf["began"]
        loss, _ = loss_of(policy, buf)
        opt.zero_grad()
        loss.backward()
        opt.step()
        print(f"update {u}: loss {loss.item():+.5f}, mean reward {buf['rewards'].mean().item():+.5f}, "
              f"{int(buf['starts'].sum())} games begun", flush=True)


if __name__ == "__main__":
    main(*(int(a) for a in sys.argv[1:]))
