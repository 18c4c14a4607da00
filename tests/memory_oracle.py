"""The definition of linear attention with a decay for each head, in 64 bits and
ply by ply, and how far results may be off it in the mean.

`check_rms` holds the root mean square of a result's errors. Roundings of a sum's
terms are independent of each other, so their mean grows with the root of the sum
of the terms' squares (`spread`), which the same definition gives on squares, and
not with the terms' magnitudes as a bound for every element has to."""

from __future__ import annotations

import torch

NAMES = ("out", "state", "dq", "dk", "dv", "d_state")
# Mean errors of float32 sums in units of `spread`. Roundings: some hundred in a row at
# most (a product's depth, a chunk, the chunks within a memory of 256 plies), 2^-24 each,
# independent: below 1e-6. The decays: exp2 of a chunk's exponent is off by 2^-23, the
# same in each of the 16 chunks of such a memory: 2e-6.
F32_MEAN = 4e-6
# A float32 operand as two bfloat16 terms: off by 2^-17.
PARTS_MEAN = 2.0 ** -17


def define(q, k, v, log_decay, starts, lengths, state, scale, d_out=None, d_state=None):
    """(out, state), or with d_out (out, state, dq, dk, dv, d_state). q, k, v (B, T, H, D)
    and the others in float64, on any one device."""
    b, t, h, dk = q.shape
    dv, dev = v.shape[-1], q.device
    lam = torch.exp(log_decay)[None, :, None, None]
    keep = torch.ones(b, t, dtype=torch.bool, device=dev) if starts is None else ~starts.bool()
    count = torch.full((b,), t, device=dev) if lengths is None else lengths.long().clamp(0, t)
    live = torch.arange(t, device=dev) < count[:, None]
    s = torch.zeros(b, h, dk, dv, dtype=torch.float64, device=dev) if state is None else state.clone()
    out = torch.zeros(b, t, h, dv, dtype=torch.float64, device=dev)
    dq, d_k, d_v = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(t):
        on, kept = live[:, i, None, None], keep[:, i, None, None, None]
        s = torch.where(on[..., None], torch.where(kept, lam * s, 0.0) + k[:, i, :, :, None] * v[:, i, :, None], s)
        out[:, i] = torch.where(on, scale * (q[:, i, :, :, None] * s).sum(-2), 0.0)
        if d_out is not None:
            dq[:, i] = torch.where(on, scale * (s * d_out[:, i, :, None]).sum(-1), 0.0)
    if d_out is None:
        return out, s
    ds = torch.zeros_like(s) if d_state is None else d_state.clone()
    for i in reversed(range(t)):
        on, kept = live[:, i, None, None], keep[:, i, None, None, None]
        full = ds + scale * q[:, i, :, :, None] * d_out[:, i, :, None]
        d_k[:, i] = torch.where(on, (full * v[:, i, :, None]).sum(-1), 0.0)
        d_v[:, i] = torch.where(on, (full * k[:, i, :, :, None]).sum(-2), 0.0)
        ds = torch.where(on[..., None], torch.where(kept, lam * full, 0.0), ds)
    return out, s, dq, d_k, d_v, ds


def spread(q, k, v, log_decay, starts, lengths, state, scale, d_out=None, d_state=None):
    """The roots of the sums of the squares of the terms of `define`'s results."""
    def square(x):
        return None if x is None else x * x
    r = define(square(q), square(k), square(v), 2 * log_decay, starts, lengths, square(state), scale * scale,
               square(d_out), square(d_state))
    return tuple(x.sqrt() for x in r)


def check_rms(name, got, want, terms, dtype):
    """The root mean square of got - want is at most that of rounding `want` to `dtype`, plus
    twice that of the sum's own errors (which move a rounded result by what they are, or to
    its neighbour where it was that near)."""
    delta = (F32_MEAN + (PARTS_MEAN if dtype == torch.bfloat16 else 0.0)) * terms.norm()
    bound = delta if got.dtype == torch.float32 else (want.to(got.dtype).double() - want).norm() + 2 * delta
    off = (got.double() - want).norm()
    assert off <= bound, (f"{name}: off by {(off / want.norm()).item():.4g} of the result in the mean, "
                          f"at most {(bound / want.norm()).item():.4g}")
