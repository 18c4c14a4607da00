"""A policy with a memory over plies, playing and learning on the GPU.

The pieces are hidden, so each seat of a game keeps a memory of its own: one state
per head, in row game * 4 + seat. While playing, a ply's token goes through
`layer_norm`, `rotary` at (ply, seat) and `linear_attention_step`, which carries the
acting seats' states along (`rows`); a game that ends starts anew in place, and so do
its memories. An update runs the same network over the stored segment, each seat's
plies one after another, with `linear_attention`, whose `starts` part the games and
whose `lengths` end the seats' plies, and learns from the rewards (REINFORCE).

  python examples/memory_policy.py [games] [plies] [updates]
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import junqi_amd  # noqa: E402
from junqi_amd import memory  # noqa: E402

GLOBALS = 28           # of an observation
ACTIONS = 16641        # canonical action ids
EATS, KILLED = 2, 4    # events of a ply
SEATS = 4
HEADS, DIM = 4, 64
WIDTH = HEADS * DIM


class Norm(nn.Module):
    def __init__(self) -> None:
        super().__init__()
        self.weight, self.bias = nn.Parameter(torch.ones(WIDTH)), nn.Parameter(torch.zeros(WIDTH))

    def forward(self, x):
        return memory.layer_norm(x, self.weight, self.bias)


class MemoryPolicy(nn.Module):
    """Logits of the canonical actions from an observation's globals and what the
    memory holds of the plies before."""

    def __init__(self, rank: int = 32, dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__()
        self.dtype = dtype
        self.embed = nn.Linear(GLOBALS, WIDTH)
        self.norm_in, self.norm_out = Norm(), Norm()
        self.qkv = nn.Linear(WIDTH, 3 * WIDTH, bias=False)
        self.out = nn.Linear(WIDTH, rank)
        self.actions = nn.Parameter(0.02 * torch.randn(rank, ACTIONS))
        self.sections = (24, 8)   # pairs of a head that turn with the ply and with the seat
        self.register_buffer("frequencies", memory.rotary_frequencies(self.sections))
        # memories of 8 to 512 plies
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(torch.linspace(-3.0, -9.0, HEADS))))

    def _token(self, glob, positions):
        x = self.embed(glob)
        qkv = self.qkv(self.norm_in(x)).to(self.dtype).unflatten(-1, (3 * HEADS, DIM))
        qk = memory.rotary(qkv[..., :2 * HEADS, :], positions, self.frequencies, self.sections)
        return x, qk[..., :HEADS, :], qk[..., HEADS:, :], qkv[..., 2 * HEADS:, :]

    def _logits(self, x, mixed):
        return self.out(self.norm_out(x + mixed.flatten(-2).to(x.dtype))) @ self.actions

    def new_state(self, games: int, device) -> torch.Tensor:
        return torch.zeros(games * SEATS, HEADS, DIM, DIM, device=device)

    @torch.no_grad()
    def play(self, glob, positions, state, starts):
        """Logits of one ply of every game; the acting seats' states move on in place. (games, ...)"""
        x, q, k, v = self._token(glob, positions)
        games = torch.arange(len(starts), device=starts.device)
        state.view(len(starts), SEATS, -1).masked_fill_(starts[:, None, None], 0.0)
        mixed = memory.linear_attention_step(q, k, v, self.log_decay, state, rows=games * SEATS + positions[:, 1])
        return self._logits(x, mixed)

    def forward(self, glob, positions, state, starts):
        """Logits of a segment's plies, (games, plies, ...), from the states before it."""
        x, q, k, v = self._token(glob, positions)
        at, lengths, begins = seat_rows(positions[..., 1], starts)
        rows, most = len(lengths), begins.shape[1]

        def by_seat(t):
            t = t.flatten(0, 1)
            return t.new_zeros(rows * most, HEADS, DIM).index_copy(0, at.flatten(), t).view(rows, most, HEADS, DIM)
        mixed = memory.linear_attention(by_seat(q), by_seat(k), by_seat(v), self.log_decay, starts=begins, lengths=lengths,
                                        initial_state=state)
        return self._logits(x, mixed.flatten(0, 1).index_select(0, at.flatten()).view_as(q))


def seat_rows(seats, starts):
    """Where a segment's plies, (games, plies), lie with each seat's one after another: their
    index in (games * 4, most), how many each row has, and where it begins a new game."""
    games, plies = seats.shape
    acts = torch.nn.functional.one_hot(seats.long(), SEATS)                                  # (games, plies, 4)
    nth = (acts.cumsum(1) - 1).gather(2, seats.long()[..., None]).squeeze(-1)
    lengths = acts.sum(1).flatten()
    most = int(lengths.max())
    row = torch.arange(games, device=seats.device)[:, None] * SEATS + seats.long()
    at = row * most + nth
    # games begun before or with each ply: a seat's ply is its first of a game where that is more
    # than at its ply before (0 before the segment: a game goes on where none has begun since)
    begun = starts.cumsum(1).flatten()
    held = torch.zeros(games * SEATS * most, dtype=begun.dtype, device=seats.device).index_copy(0, at.flatten(), begun)
    held = held.view(-1, most)
    return at, lengths, held != torch.nn.functional.pad(held[:, :-1], (1, 0))


def rollout(policy: MemoryPolicy, r, state: torch.Tensor, began: torch.Tensor, plies: int, seed: int) -> dict:
    """Play `plies` plies of every game. `began`: plies of each game so far (0: the
    next ply is its first). The buffers are time-major, (plies, games, ...)."""
    n, dev = r.num_envs, r.device
    g = torch.Generator(dev).manual_seed(seed)
    buf = {"state": state.clone(), "glob": torch.empty(plies, n, GLOBALS, device=dev),
           "positions": torch.empty(plies, n, 2, dtype=torch.int32, device=dev),
           "starts": torch.empty(plies, n, dtype=torch.bool, device=dev),
           "mask": torch.empty(plies, n, ACTIONS, dtype=torch.bool, device=dev),
           "actions": torch.empty(plies, n, dtype=torch.int64, device=dev),
           "rewards": torch.empty(plies, n, device=dev), "logits": []}
    for t in range(plies):
        turn = r.turn_torch()
        _, glob = r.build_acting_seat_observation_torch(turn)
        buf["glob"][t].copy_(glob)
        buf["positions"][t] = torch.stack([began, turn.int()], -1)
        buf["starts"][t] = began == 0
        buf["mask"][t].copy_(r.batch.legal(mask_words=False, mask_bool=True)["mask_bool"].bool())
        logits = policy.play(buf["glob"][t], buf["positions"][t], state, buf["starts"][t])
        buf["logits"].append(logits)
        p = torch.softmax(logits.float().masked_fill(~buf["mask"][t], -torch.inf), -1)
        buf["actions"][t] = torch.multinomial(p, 1, generator=g).squeeze(1)
        step = r.step_device_torch(buf["actions"][t].to(torch.int32), turn)
        # games are won late: a captured and a lost piece count a little
        event = step["event"]
        buf["rewards"][t] = step["rewards"] + 0.1 * (event == EATS).float() - 0.1 * (event == KILLED).float()
        began = torch.where(step["terminated"].bool(), 0, began + 1)
        r.update_beliefs_device(step, turn)
        r.reset_terminated_device(seed=seed + t)
    buf["logits"] = torch.stack(buf["logits"])
    buf["began"] = began
    return buf


def loss_of(policy: MemoryPolicy, buf: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """REINFORCE over the segment; also the logits, (plies, games, actions)."""
    by_game = {k: buf[k].transpose(0, 1) for k in ("glob", "positions", "starts")}
    logits = policy(by_game["glob"], by_game["positions"], buf["state"], by_game["starts"]).transpose(0, 1)
    logp = torch.log_softmax(logits.float().masked_fill(~buf["mask"], -torch.inf), -1)
    taken = logp.gather(-1, buf["actions"][..., None]).squeeze(-1)
    gain = buf["rewards"] - buf["rewards"].mean()
    return -(gain * taken).mean(), logits


def main(games: int = 256, plies: int = 64, updates: int = 3) -> None:
    torch.manual_seed(0)
    r = junqi_amd.GpuRollout(games, show_mode=2, max_num_moves=1200)
    r.reset(0)
    policy = MemoryPolicy().to(r.device)
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
