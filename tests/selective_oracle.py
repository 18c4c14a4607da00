"""The definitions of the selective scan, the causal convolution and the masked logits,
in 64 bits on the CPU, ply by ply, with their gradients by going back; and how far
results may be off.

A result that is a sum of terms is off by at most (number of roundings) * 2^-24 * (sum
of the terms' magnitudes), which the same definition gives with `size`: every factor by
its absolute value, the decays as they are. Rounding the result to its type adds half a
step of the value, finfo.eps / 2."""

from __future__ import annotations

import torch

EPS = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def silu_slope(z, size=False):
    s = torch.sigmoid(z)
    return s * (1 + (z.abs() if size else z) * (1 - s))


def scan(x, size=False):
    """x: u, delta, gate (B, T, D), b, c (B, T, G, N), a (D, N), skip, delta_bias (D,), starts, lengths,
    state (B, D, N), softplus, d_out, d_state: CPU doubles, None where absent."""
    f = torch.abs if size else (lambda v: v)
    u, (b_, c_), a = f(x["u"]), (f(x["b"]), f(x["c"])), x["a"]
    batch, plies, d = u.shape
    n, groups = b_.shape[-1], b_.shape[-2]
    per = d // groups
    b, c = b_.repeat_interleave(per, 2), c_.repeat_interleave(per, 2)
    pre = x["delta"] + (0.0 if x["delta_bias"] is None else x["delta_bias"])
    step = torch.nn.functional.softplus(pre, threshold=1e9) if x["softplus"] else pre
    rate = torch.sigmoid(pre) if x["softplus"] else torch.ones_like(pre)
    dt = f(step)
    skip = torch.zeros(d, dtype=torch.float64) if x["skip"] is None else f(x["skip"])
    z = x["gate"]
    gain = torch.ones_like(u) if z is None else f(z) * torch.sigmoid(z)
    starts = torch.zeros(batch, plies, dtype=torch.bool) if x["starts"] is None else x["starts"].bool()
    count = torch.full((batch,), plies) if x["lengths"] is None else x["lengths"].long().clamp(0, plies)
    h = torch.zeros(batch, d, n, dtype=torch.float64) if x["state"] is None else f(x["state"]).clone()
    out, y = torch.zeros_like(u), torch.zeros_like(u)
    before, after, keep = [], [], []
    for t in range(plies):
        on = (t < count)[:, None, None]
        k = torch.where(starts[:, t, None, None], 0.0, torch.exp(step[:, t, :, None] * a))
        old = torch.where(starts[:, t, None, None], 0.0, h)
        new = k * old + (dt[:, t] * u[:, t])[..., None] * b[:, t]
        before.append(old)
        keep.append(k)
        h = torch.where(on, new, h)
        after.append(new)
        y[:, t] = torch.where(on[..., 0], (new * c[:, t]).sum(-1) + skip * u[:, t], 0.0)
        out[:, t] = torch.where(on[..., 0], y[:, t] * gain[:, t], 0.0)
    res = {"out": out, "state": h}
    if x["d_out"] is None:
        return res
    d_out = f(x["d_out"])
    dh = torch.zeros_like(h) if x["d_state"] is None else f(x["d_state"]).clone()
    g = {k: torch.zeros_like(v) for k, v in (("u", u), ("delta", u), ("b", b_), ("c", c_), ("a", a), ("skip", skip),
                                            ("delta_bias", skip), ("gate", u))}
    for t in reversed(range(plies)):
        live = t < count
        on, on1 = live[:, None, None], live[:, None]
        dy = torch.where(on1, d_out[:, t] * gain[:, t], 0.0)
        full = torch.where(on, dh + c[:, t] * dy[..., None], 0.0)
        moved = torch.where(on, full * keep[t] * before[t], 0.0)
        through = (full * b[:, t]).sum(-1)
        d_pre = torch.where(on1, (u[:, t] * through + (moved * f(a)).sum(-1)) * rate[:, t], 0.0)
        g["u"][:, t] = torch.where(on1, dt[:, t] * through + skip * dy, 0.0)
        g["delta"][:, t] = d_pre
        g["delta_bias"] += d_pre.sum(0)
        g["skip"] += (dy * torch.where(on1, u[:, t], 0.0)).sum(0)
        g["a"] += (moved * dt[:, t, :, None]).sum(0)
        push = torch.where(on1, dt[:, t] * u[:, t], 0.0)
        g["b"][:, t] = (full * push[..., None]).unflatten(1, (groups, per)).sum(2)
        g["c"][:, t] = torch.where(on, dy[..., None] * after[t], 0.0).unflatten(1, (groups, per)).sum(2)
        if z is not None:
            g["gate"][:, t] = torch.where(on1, d_out[:, t] * y[:, t] * silu_slope(z[:, t], size), 0.0)
        dh = torch.where(on, torch.where(starts[:, t, None, None], 0.0, full * keep[t]), dh)
    g["state"] = dh
    return {**res, **{"d_" + k: v for k, v in g.items()}}


def scan_roundings(x):
    """How many roundings a term may go through: a decay's exponent is dt * a, of which dt is off
    by some ten (softplus), so a product of decays by that times the sum of the exponents, and
    by four for each ply; sums over states, channels and games; gates and rates, some thirty."""
    pre = x["delta"] + (0.0 if x["delta_bias"] is None else x["delta_bias"])
    dt = torch.nn.functional.softplus(pre) if x["softplus"] else pre.abs()
    batch, plies, d = x["u"].shape
    exponents = (dt[..., None] * x["a"].abs()).sum(1).max().item() if plies and batch else 0.0
    return 4 * plies + 12 * min(exponents, 90.0) + x["a"].shape[1] + d + batch * plies + 40


def conv(x, size=False):
    """x: x (B, T, D), weight (D, W), bias, starts, lengths, state (B, W - 1, D), silu, d_out, d_state."""
    f = torch.abs if size else (lambda v: v)
    v, w = f(x["x"]), f(x["weight"])
    batch, plies, d = v.shape
    taps = w.shape[1]
    bias = torch.zeros(d, dtype=torch.float64) if x["bias"] is None else f(x["bias"])
    starts = torch.zeros(batch, plies, dtype=torch.bool) if x["starts"] is None else x["starts"].bool()
    count = torch.full((batch,), plies) if x["lengths"] is None else x["lengths"].long().clamp(0, plies)
    state = torch.zeros(batch, taps - 1, d, dtype=torch.float64) if x["state"] is None else f(x["state"])
    true = None if not size else conv({**x, "silu": False, "d_out": None})["out"]
    out, pre = torch.zeros_like(v), torch.zeros_like(v)
    final = torch.zeros_like(state)
    g = {"x": torch.zeros_like(v), "weight": torch.zeros_like(w), "bias": torch.zeros_like(bias), "state": torch.zeros_like(state)}
    d_out = None if x["d_out"] is None else f(x["d_out"])
    for i in range(batch):
        for t in range(int(count[i])):
            seen = []
            for back in range(taps):
                if back and t - back + 1 >= 0 and starts[i, t - back + 1]:
                    break
                seen.append(back)
            o = bias.clone()
            for back in seen:
                o = o + w[:, taps - 1 - back] * (v[i, t - back] if t >= back else state[i, taps - 1 + t - back])
            pre[i, t] = o
            # off by its own error times the slope, at most 1.1, and by its own factors
            if x["silu"]:
                out[i, t] = 1.1 * o if size else o * torch.sigmoid(o)
            else:
                out[i, t] = o
            if d_out is None:
                continue
            slope = torch.ones(d, dtype=torch.float64)
            if x["silu"]:   # its slope's slope is at most 1/2
                slope = silu_slope(true[i, t], True) + 0.5 * o if size else silu_slope(o)
            ge = d_out[i, t] * slope
            g["bias"] += ge
            for back in seen:
                src = v[i, t - back] if t >= back else state[i, taps - 1 + t - back]
                g["weight"][:, taps - 1 - back] += ge * src
                to = g["x"][i, t - back] if t >= back else g["state"][i, taps - 1 + t - back]
                to += ge * w[:, taps - 1 - back]
        n = int(count[i])
        for back in range(1, taps):      # the input `back` plies before ply n
            if back > 1 and n - back + 1 >= 0 and n and starts[i, n - back + 1]:
                break
            src = v[i, n - back] if n >= back else state[i, taps - 1 + n - back]
            final[i, taps - 1 - back] = src
            if x["d_state"] is not None:
                to = g["x"][i, n - back] if n >= back else g["state"][i, taps - 1 + n - back]
                to += f(x["d_state"])[i, taps - 1 - back]
    res = {"out": out, "state": final}
    return res if d_out is None else {**res, **{"d_" + k: q for k, q in g.items()}}


def logits(x):
    """x: logits (N, A), bias, legal (N, A) bool, recent (N, L), recent_lengths, repetition, frequency,
    presence (numbers or (N,)), d_out. The result, its gradients, and the terms' magnitudes."""
    v = x["logits"]
    n, acts = v.shape
    count = torch.zeros(n, acts, dtype=torch.float64)
    if x["recent"] is not None:
        for i in range(n):
            for j in range(x["recent"].shape[1] if x["recent_lengths"] is None else int(x["recent_lengths"][i].clamp(0, x["recent"].shape[1]))):
                a = int(x["recent"][i, j])
                if 0 <= a < acts:
                    count[i, a] += 1

    def rows(p):
        return p.double()[:, None] if isinstance(p, torch.Tensor) else p
    rep, fre, pres = (rows(x[k]) for k in ("repetition", "frequency", "presence"))
    factor = torch.where(count > 0, torch.where(v > 0, 1.0 / rep + 0 * v, rep + 0 * v), 1.0)
    less = torch.where(count > 0, fre * count + pres, 0.0)
    bias = torch.zeros(acts, dtype=torch.float64) if x["bias"] is None else x["bias"]
    legal = torch.ones(n, acts, dtype=torch.bool) if x["legal"] is None else x["legal"]
    out = torch.where(legal, v * factor - less + bias, -torch.inf)
    size = v.abs() * factor + torch.where(count > 0, abs(fre) * count + abs(pres), 0.0) + bias.abs()
    g = torch.where(legal, x["d_out"], 0.0)
    return {"out": out, "d_logits": g * factor, "d_bias": g.sum(0), "size": size, "size_bias": g.abs().sum(0)}


def close(name, got, want, size, roundings, dtype, floor=1e-36):
    """got is within rounding to dtype of what float32 sums may be off from want; `floor`: what
    float32 cannot hold."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)}, not {tuple(want.shape)}"
    if not got.numel():
        return
    bound = want.abs() * half_step(dtype) * (1 if dtype != torch.float32 else 0) + (roundings + 1) * EPS * size + floor
    off = (got - want).abs()
    assert bool((off <= bound).all()), (
        f"{name}: off by {off.max().item():.3g} of {want.abs().max().item():.3g}, bound there "
        f"{bound.flatten()[(off - bound).argmax()].item():.3g}")
