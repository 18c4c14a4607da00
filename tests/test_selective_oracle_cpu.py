"""The 64-bit definitions that the selective operators are held to, against autograd of the
formulas written out another way and against differences. No GPU."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from tests import selective_oracle as O  # noqa: E402

F64 = torch.float64


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, dtype=F64)


def _scan_inputs(seed, b=3, t=7, d=6, n=4, groups=2):
    g = torch.Generator().manual_seed(seed)
    return {"u": _rand(g, b, t, d), "delta": _rand(g, b, t, d), "gate": _rand(g, b, t, d), "b": _rand(g, b, t, groups, n),
            "c": _rand(g, b, t, groups, n), "a": -torch.rand(d, n, generator=g, dtype=F64), "skip": _rand(g, d),
            "delta_bias": _rand(g, d), "starts": torch.rand(b, t, generator=g) < 0.2, "lengths": torch.tensor([t, 0, 4][:b]),
            "state": _rand(g, b, d, n), "softplus": True, "d_out": _rand(g, b, t, d), "d_state": _rand(g, b, d, n)}


def _scan_plain(x):
    """The scan with a decay between every two plies, for autograd."""
    b, t, d = x["u"].shape
    groups = x["b"].shape[-2]
    live = torch.arange(t) < x["lengths"][:, None]
    dt = torch.log1p(torch.exp(x["delta"] + x["delta_bias"])) * live[..., None]
    gain = (dt * x["u"])[..., None] * x["b"].repeat_interleave(d // groups, 2)          # (b, t, d, n)
    upto = torch.cat([torch.zeros_like(dt[:, :1]), dt.cumsum(1)], 1)                    # of the plies before each
    game = (x["starts"] & live).cumsum(1)
    i, j = torch.arange(t)[:, None], torch.arange(t)
    span = torch.exp((upto[:, 1:, None] - upto[:, None, 1:])[..., None] * x["a"])       # (b, t, t, d, n): from after j to i
    seen = ((i >= j) & (game[:, :, None] == game[:, None]))[..., None, None]
    h = torch.where(seen, span * gain[:, None], 0.0).sum(2)
    h = h + torch.where((game == 0)[..., None, None], torch.exp(upto[:, 1:, :, None] * x["a"]) * x["state"][:, None], 0.0)
    y = (h * x["c"].repeat_interleave(d // groups, 2)).sum(-1) + x["skip"] * x["u"]
    out = y * torch.nn.functional.silu(x["gate"]) * live[..., None]
    return out, h[:, -1]


def test_scan():
    x = _scan_inputs(1)
    want = O.scan(x)
    names = ("u", "delta", "gate", "b", "c", "a", "skip", "delta_bias", "state")
    leaves = {k: x[k].clone().requires_grad_() for k in names}
    out, state = _scan_plain({**x, **leaves})
    assert torch.allclose(out, want["out"], rtol=1e-11, atol=1e-12)
    assert torch.allclose(state, want["state"], rtol=1e-11, atol=1e-12)
    grads = torch.autograd.grad([out, state], list(leaves.values()), [x["d_out"], x["d_state"]])
    for k, g in zip(names, grads):
        assert torch.allclose(g, want["d_" + k], rtol=1e-9, atol=1e-11), k


def test_scan_differences():
    x = _scan_inputs(2, b=1, t=4, d=2, n=2, groups=1)
    want = O.scan(x)

    def value(y):
        r = O.scan({**y, "d_out": None})
        return (r["out"] * x["d_out"]).sum() + (r["state"] * x["d_state"]).sum()
    for k in ("u", "delta", "gate", "b", "c", "a", "skip", "delta_bias", "state"):
        for i in range(x[k].numel()):
            e = torch.zeros_like(x[k]).flatten()
            e[i] = 1e-6
            e = e.view_as(x[k])
            slope = (value({**x, k: x[k] + e}) - value({**x, k: x[k] - e})) / 2e-6
            assert abs(slope - want["d_" + k].flatten()[i]) < 1e-7, (k, i)


@pytest.mark.parametrize("taps", [1, 2, 4, 8])
def test_conv(taps):
    g = torch.Generator().manual_seed(taps)
    b, t, d = 4, 9, 3
    x = {"x": _rand(g, b, t, d), "weight": _rand(g, d, taps), "bias": _rand(g, d), "starts": torch.rand(b, t, generator=g) < 0.25,
         "lengths": torch.tensor([t, 0, 1, 5]), "state": _rand(g, b, taps - 1, d), "silu": True, "d_out": _rand(g, b, t, d),
         "d_state": _rand(g, b, taps - 1, d)}
    want = O.conv(x)
    names = ("x", "weight", "bias", "state")
    leaves = {k: x[k].clone().requires_grad_() for k in names}
    live = torch.arange(t) < x["lengths"][:, None]
    seen = torch.cat([leaves["state"], leaves["x"]], 1)
    game = torch.nn.functional.pad(x["starts"].cumsum(1), (taps - 1, 0))
    same = game.unfold(1, taps, 1) == game[:, taps - 1:, None]
    o = (seen.unfold(1, taps, 1) * same[:, :, None] * leaves["weight"]).sum(-1) + leaves["bias"]
    out = torch.nn.functional.silu(o) * live[..., None]
    at = x["lengths"][:, None] + torch.arange(taps - 1)
    last = game.gather(1, (x["lengths"] + taps - 2).clamp(min=0)[:, None])
    state = seen.gather(1, at[..., None].expand(-1, -1, d)) * (game.gather(1, at) == last)[..., None]
    assert torch.allclose(out, want["out"], atol=1e-12) and torch.allclose(state, want["state"], atol=1e-12)
    grads = torch.autograd.grad([out, state], list(leaves.values()), [x["d_out"], x["d_state"]], allow_unused=True)
    for k, got in zip(names, grads):
        assert got is None and not want["d_" + k].numel() or torch.allclose(got, want["d_" + k], atol=1e-11), k


def test_logits():
    x = {"logits": torch.tensor([[1.0, -2.0, 3.0, 0.5]], dtype=F64), "bias": torch.tensor([0.1, 0.2, 0.3, 0.4], dtype=F64),
         "legal": torch.tensor([[True, True, True, False]]), "recent": torch.tensor([[1, 0, 1, -1, 9, 2]]),
         "recent_lengths": torch.tensor([5]), "repetition": 2.0, "frequency": 0.25, "presence": 0.5,
         "d_out": torch.ones(1, 4, dtype=F64)}
    r = O.logits(x)
    assert r["out"].tolist() == [[0.5 - 0.75 + 0.1, -4.0 - 1.0 + 0.2, 3.3, -torch.inf]]
    assert r["d_logits"].tolist() == [[0.5, 2.0, 1.0, 0.0]] and r["d_bias"].tolist() == [1.0, 1.0, 1.0, 0.0]
