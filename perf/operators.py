"""Performance cases of the operators of a policy's memory over the plies of a
game (junqi_amd.memory): linear attention with a decay for each head, rotary
positions with several axes, layer norm.

Every case is one pass through one operator as a training or serving program
calls it. `run` computes it in plain 32-bit torch operations where `own` is
false, and through the package where it is true.

Kinds of cases (`kind`):
  attention  linear attention over segments of plies: forward, or forward and
             backward (`train`)
  step       linear attention of one new ply of every game, its state updated in
             place
  rotary     rotary positions of (ply, row, column) or (row, column), forward, or
             forward and backward (`train`)
  norm       layer norm, forward, or forward and backward (`train`)
"""

from __future__ import annotations

import numpy as np
import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}
MAX_PLIES = 1200   # the ply limit that the collector's games run under


def listed():
    return [
        # PPO update over 256-step rollout segments of 1,024 games, out of time-major buffers; games restart inside
        # a segment, and the memory of the step before it goes in
        {"name": "attention_train_bf16_1024x256", "kind": "attention", "train": True, "dtype": "bf16", "games": 1024,
         "plies": 256, "heads": 4, "key_dim": 64, "value_dim": 64, "time_major": True, "ragged": False, "state": True},
        # the same in float32 on a small rollout with odd sizes: games of different lengths, gradients of the states
        {"name": "attention_train_f32_96x77", "kind": "attention", "train": True, "dtype": "f32", "games": 96,
         "plies": 77, "heads": 3, "key_dim": 40, "value_dim": 56, "time_major": False, "ragged": True, "state": True},
        # two long records of games one after another, read once: few rows, a long axis
        {"name": "attention_bf16_2x65537", "kind": "attention", "train": False, "dtype": "bf16", "games": 2,
         "plies": 65537, "heads": 8, "key_dim": 128, "value_dim": 128, "time_major": False, "ragged": False,
         "state": False},
        # an evaluation match that catches up on its openings: launches and latency
        {"name": "attention_bf16_24x33", "kind": "attention", "train": False, "dtype": "bf16", "games": 24, "plies": 33,
         "heads": 4, "key_dim": 64, "value_dim": 64, "time_major": False, "ragged": True, "state": True},
        # one ply of the batch that the environment is built for
        {"name": "step_bf16_32768", "kind": "step", "dtype": "bf16", "games": 32768, "seats": 1, "heads": 4,
         "key_dim": 64, "value_dim": 64},
        # the acting seat's own memory out of four, in a match of a few dozen games
        {"name": "step_f32_24", "kind": "step", "dtype": "f32", "games": 24, "seats": 4, "heads": 4, "key_dim": 64,
         "value_dim": 64},
        # queries and keys of the rollout segments, at (ply, row, column), trained through
        {"name": "rotary_train_bf16_262144", "kind": "rotary", "train": True, "dtype": "bf16", "tokens": 262144,
         "heads": 8, "dim": 64, "axes": 3, "rotated": 64, "interleaved": False},
        # the 129 cells of every board of an odd batch, at (row, column); part of each head stays as it is
        {"name": "rotary_f32_4099x129", "kind": "rotary", "train": False, "dtype": "f32", "tokens": 4099 * 129,
         "heads": 2, "dim": 56, "axes": 2, "rotated": 40, "interleaved": True},
        # one ply of a match: queries and keys of 24 games
        {"name": "rotary_bf16_24", "kind": "rotary", "train": False, "dtype": "bf16", "tokens": 24, "heads": 8,
         "dim": 64, "axes": 3, "rotated": 64, "interleaved": False},
        # the rollout segments' tokens, trained
        {"name": "norm_train_bf16_262144x256", "kind": "norm", "train": True, "dtype": "bf16", "rows": 262144,
         "width": 256},
        # the 28 globals of every game's observation, trained
        {"name": "norm_train_f32_32768x28", "kind": "norm", "train": True, "dtype": "f32", "rows": 32768, "width": 28},
        # one ply of an odd batch with a wide odd row, served
        {"name": "norm_bf16_333x8191", "kind": "norm", "train": False, "dtype": "bf16", "rows": 333, "width": 8191},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; odd ones as likely as even."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    return max(lo, min(hi, v + rng.randrange(2)))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "step", "rotary", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind in ("attention", "step"):
        heads = rng.randrange(1, 9)
        key_dim = rng.choice([16, 32, 40, 50, 64, 64, 96, 128])
        value_dim = rng.choice([key_dim, key_dim, rng.choice([24, 36, 64, 128])])
        width = heads * max(key_dim, value_dim)
        if kind == "step":
            seats = rng.choice([1, 4])
            top = min(32000, int(4e8) // (seats * heads * key_dim * value_dim))
            return {"kind": kind, "dtype": dtype, "games": _size(rng, 8, max(9, top)), "seats": seats, "heads": heads,
                    "key_dim": key_dim, "value_dim": value_dim}
        plies = _size(rng, 1, 16000)
        top = max(1, min(2048, int(2.5e7) // (plies * width)))
        return {"kind": kind, "train": rng.random() < 0.6, "dtype": dtype, "games": _size(rng, 1, top), "plies": plies,
                "heads": heads, "key_dim": key_dim, "value_dim": value_dim, "time_major": rng.random() < 0.5,
                "ragged": rng.random() < 0.5, "state": rng.random() < 0.5}
    if kind == "rotary":
        heads, dim, axes = rng.randrange(1, 9), rng.choice([24, 32, 40, 64, 96, 128]), rng.randrange(1, 4)
        return {"kind": kind, "train": rng.random() < 0.5, "dtype": dtype,
                "tokens": _size(rng, 8, int(4e7) // (heads * dim)), "heads": heads, "dim": dim, "axes": axes,
                "rotated": rng.choice([dim, dim, 2 * rng.randrange(axes, dim // 2)]),
                "interleaved": rng.random() < 0.5}
    width = _size(rng, 16, 9000)
    return {"kind": kind, "train": rng.random() < 0.6, "dtype": dtype, "rows": _size(rng, 8, int(4e7) // width),
            "width": width}


# ------------------------------------------------------------------ inputs
def _sections(case):
    """How many pairs turn with each axis: even parts, the first the largest."""
    pairs, axes = case["rotated"] // 2, case["axes"]
    rest = [pairs // axes] * (axes - 1)
    return [pairs - sum(rest), *rest]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPE[case["dtype"]]
    kind, train = case["kind"], case.get("train", False)

    def randn(*shape, dtype=dt, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)

    def below(n, *shape):
        return torch.randint(0, n, shape, generator=g, device="cuda")

    s = {"kind": kind, "train": train}
    if kind in ("attention", "step"):
        b, h, dk, dv = case["games"], case["heads"], case["key_dim"], case["value_dim"]
        # memories of 8 to 1,024 plies
        s["log_decay"] = torch.log1p(-torch.exp2(-3 - 7 * torch.arange(h, device="cuda") / max(1, h - 1))).float()
        s["scale"] = dk ** -0.5
        if kind == "step":
            s["q"], s["k"], s["v"] = randn(b, h, dk), randn(b, h, dk), randn(b, h, dv)
            s["memory"] = randn(b * case["seats"], h, dk, dv, dtype=torch.float32, scale=3.0)
            s["starts"] = below(200, b) == 0
            acting = below(case["seats"], b)
            s["rows"] = torch.arange(b, device="cuda") * 4 + acting if case["seats"] == 4 else None
            return s
        t = case["plies"]
        shape = (t, b) if case["time_major"] else (b, t)
        s["time_major"] = case["time_major"]
        s["q"], s["k"], s["v"] = randn(*shape, h, dk), randn(*shape, h, dk), randn(*shape, h, dv)
        s["starts"] = below(200, *shape) == 0
        s["lengths"] = below(t + 1, b).to(torch.int32) if case["ragged"] else None
        s["state"] = randn(b, h, dk, dv, dtype=torch.float32, scale=3.0) if case["state"] else None
        if train:
            s["d_out"] = randn(*shape, h, dv)
            s["leaves"] = [s[x].requires_grad_() for x in ("q", "k", "v")]
            if case["state"]:
                s["leaves"].append(s["state"].requires_grad_())
                s["d_state"] = randn(b, h, dk, dv, dtype=torch.float32)
        return s
    if kind == "rotary":
        n, h, d = case["tokens"], case["heads"], case["dim"]
        s["x"] = randn(n, h, d)
        at = [below(17, n) for _ in range(case["axes"])]
        if case["axes"] != 2:
            at[0] = below(MAX_PLIES, n)
        s["positions"] = torch.stack(at, -1).to(torch.int32)
        s["sections"] = _sections(case)
        s["frequencies"] = torch.cat([10000.0 ** (-torch.arange(p, dtype=torch.float64) / p) for p in s["sections"]])
        s["frequencies"] = s["frequencies"].float().cuda()
        s["axis"] = torch.repeat_interleave(torch.arange(case["axes"]), torch.tensor(s["sections"])).cuda()
        s["interleaved"] = case["interleaved"]
        if train:
            s["x"].requires_grad_()
            s["d_out"] = randn(n, h, d)
        return s
    n, w = case["rows"], case["width"]
    s["x"] = torch.add(randn(n, w), 0.5)
    s["weight"] = randn(w, dtype=torch.float32, scale=0.1).add_(1.0)
    s["bias"] = randn(w, dtype=torch.float32, scale=0.1)
    s["eps"] = 1e-5
    if train:
        s["d_out"] = randn(n, w)
        s["leaves"] = [s[x].requires_grad_() for x in ("x", "weight", "bias")]
    return s


# ------------------------------------------------------------------ plain forms, in 32 bits
def _plain_attention(q, k, v, log_decay, starts, lengths, state, scale):
    b, t, h, dk = q.shape
    dv = v.shape[-1]
    c = min(t, 128 if t > 4096 else 64)
    n = -(-t // c)
    dev = q.device
    live = torch.arange(t, device=dev)[None] < (lengths[:, None] if lengths is not None else t)   # (b or 1, t)

    def chunks(x):
        x = torch.where(live[:, :, None, None], x.float(), 0.0).transpose(1, 2)
        return torch.nn.functional.pad(x, (0, 0, 0, n * c - t)).reshape(b, h, n, c, x.shape[-1])

    q, k, v = chunks(q), chunks(k), chunks(v)
    game = torch.nn.functional.pad(torch.cumsum(starts.int(), 1), (0, n * c - t), mode="replicate").reshape(b, 1, n, c)
    end = game[..., -1]                                                       # (b, 1, n)
    before = torch.nn.functional.pad(end[..., :-1], (1, 0))
    at = torch.arange(c, device=dev)
    apart = at[:, None] - at
    ld = log_decay[:, None, None, None]
    decay = torch.exp(ld * apart.clamp(min=0))
    seen = (apart >= 0) & (game[..., :, None] == game[..., None, :])
    out = (q @ k.transpose(-1, -2) * torch.where(seen, decay, 0.0)) @ v
    to_end = torch.where(game == end[..., None], torch.exp(ld[..., 0] * (c - 1 - at)), 0.0)
    gained = (k * to_end[..., None]).transpose(-1, -2) @ v                    # (b, h, n, dk, dv)
    m = torch.arange(n, device=dev)
    steps = m[:, None] - 1 - m
    carried = torch.where((steps >= 0) & (before[..., :, None] == end[..., None, :]),
                          torch.exp(ld[..., 0] * c * steps.clamp(min=0)), 0.0)   # (b, h, n, n)
    first = (carried @ gained.reshape(b, h, n, dk * dv)).reshape(b, h, n, dk, dv)
    if state is not None:
        kept = torch.where(before == 0, torch.exp(log_decay[:, None] * c * m), 0.0)
        first = first + kept[..., None, None] * state[:, :, None]
    since = torch.where(game == before[..., None], torch.exp(ld[..., 0] * (at + 1)), 0.0)
    out = (out + since[..., None] * (q @ first)) * scale
    out = torch.where(live[:, :, None, None], out.reshape(b, h, n * c, dv)[:, :, :t].transpose(1, 2), 0.0)
    # the state after the last live ply
    count = lengths.long()[:, None] if lengths is not None else torch.full((b, 1), t, device=dev)
    game = torch.nn.functional.pad(torch.cumsum(starts.int(), 1), (1, 0))     # (b, t + 1): games begun before each ply
    last = torch.gather(game, 1, count)
    ply = torch.arange(t, device=dev)
    weight = torch.where((game[:, 1:] == last) & (ply < count), 1.0, 0.0)[:, None]
    weight = weight * torch.exp(log_decay[:, None] * (count - 1 - ply).clamp(min=0)[:, None])     # (b, h, t)
    k, v = k.reshape(b, h, n * c, dk)[:, :, :t], v.reshape(b, h, n * c, dv)[:, :, :t]
    final = (k * weight[..., None]).transpose(-1, -2) @ v
    if state is not None:
        kept = torch.where(last == 0, torch.exp(log_decay * count), 0.0)
        final = final + kept[..., None, None] * state
    return out, final


def _plain_step(q, k, v, log_decay, memory, rows, starts, scale):
    s = memory if rows is None else memory[rows]
    s = torch.where(starts[:, None, None, None], 0.0, s * torch.exp(log_decay)[:, None, None])
    s = s + k.float()[..., :, None] * v.float()[..., None, :]
    if rows is None:
        memory.copy_(s)
    else:
        memory[rows] = s
    return ((q.float()[..., None, :] @ s)[..., 0, :] * scale).to(q.dtype)


def _plain_rotary(x, positions, frequencies, axis, interleaved):
    angle = positions[:, axis].float() * frequencies
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    r = 2 * frequencies.numel()
    y, rest = x.float()[..., :r], x.float()[..., r:]
    if interleaved:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, rest], -1).to(x.dtype)


def _plain_norm(x, weight, bias, eps):
    y = x.float()
    y = y - y.mean(-1, keepdim=True)
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps)
    return (y * weight + bias).to(x.dtype)


# ------------------------------------------------------------------ one pass
def run(state):
    s = state
    kind, train = s["kind"], s["train"]
    if own:
        from junqi_amd import memory
    if kind == "attention":
        q, k, v, starts = s["q"], s["k"], s["v"], s["starts"]
        if s["time_major"]:
            q, k, v, starts = (x.transpose(0, 1) for x in (q, k, v, starts))
        if own:
            out, final = memory.linear_attention(q, k, v, s["log_decay"], starts=starts, lengths=s["lengths"],
                                                 initial_state=s["state"], scale=s["scale"], return_state=True)
        else:
            out, final = _plain_attention(q, k, v, s["log_decay"], starts, s["lengths"], s["state"], s["scale"])
            out = out.to(q.dtype)
        if s["time_major"]:
            out = out.transpose(0, 1)
        if not train:
            return {"out": out, "state": final}
        results, grads = ([out, final], [s["d_out"], s["d_state"]]) if s["state"] is not None else ([out], [s["d_out"]])
        grads = torch.autograd.grad(results, s["leaves"], grads)
        return {"out": out.detach(), "state": final.detach(), "grads": grads}
    if kind == "step":
        step = memory.linear_attention_step if own else _plain_step
        out = step(s["q"], s["k"], s["v"], s["log_decay"], s["memory"], rows=s["rows"], starts=s["starts"],
                   scale=s["scale"])
        return {"out": out, "state": s["memory"]}
    if kind == "rotary":
        if own:
            out = memory.rotary(s["x"], s["positions"], s["frequencies"], s["sections"], interleaved=s["interleaved"])
        else:
            out = _plain_rotary(s["x"], s["positions"], s["frequencies"], s["axis"], s["interleaved"])
        if not train:
            return {"out": out}
        return {"out": out.detach(), "grads": torch.autograd.grad(out, [s["x"]], s["d_out"])}
    norm = memory.layer_norm if own else _plain_norm
    out = norm(s["x"], s["weight"], s["bias"], s["eps"])
    if not train:
        return {"out": out}
    return {"out": out.detach(), "grads": torch.autograd.grad(out, s["leaves"], s["d_out"])}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, e = case["kind"], BYTES[case["dtype"]]
    passes = 2 if case.get("train") else 1   # a gradient goes in and one comes out for each input and output
    if kind in ("attention", "step"):
        b, h, dk, dv = case["games"], case["heads"], case["key_dim"], case["value_dim"]
        state = b * h * dk * dv * 4
        if kind == "step":
            return {"bytes": b * h * (2 * dk + 2 * dv) * e + 2 * state + b, "flops": 4 * b * h * dk * dv}
        tokens = b * case["plies"] / (2 if case["ragged"] else 1)   # lengths are spread over 0 .. plies
        outputs = b * case["plies"] * h * ((2 * dk + 2 * dv) if case.get("train") else dv)
        inputs = tokens * h * (2 * dk + dv * passes)
        # the states before and after, and their gradients
        states = state * (passes if case["state"] else 0) + state * (passes if case["state"] else 1)
        # a product of the state's size each for the state and the output; the gradients take five
        return {"bytes": int((inputs + outputs) * e + states + b * case["plies"]),
                "flops": int(tokens * h * dk * dv * (14 if case.get("train") else 4))}
    if kind == "rotary":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * passes * n * e + case["tokens"] * case["axes"] * 4,
                "flops": 3 * passes * case["tokens"] * case["heads"] * case["rotated"]}
    n = case["rows"] * case["width"]
    return {"bytes": 2 * passes * n * e + case["width"] * 8 * passes, "flops": n * (20 if case.get("train") else 7)}


# ------------------------------------------------------------------ the definitions, in 64 bits
def _exact_attention(s):
    """Ply by ply: the state, what it answers, and the gradients by going back over the plies."""
    order = (lambda x: x) if s["time_major"] else (lambda x: x.transpose(0, 1))     # (t, b, ...)
    q, k, v = (order(s[x].detach()).double() for x in ("q", "k", "v"))
    starts = order(s["starts"])
    t, b, h, dk = q.shape
    dv = v.shape[-1]
    count = s["lengths"].long() if s["lengths"] is not None else torch.full((b,), t, device=q.device)
    lam = torch.exp(s["log_decay"].double())[None, :, None, None]
    scale = s["scale"]
    mem = torch.zeros(b, h, dk, dv, dtype=torch.float64, device=q.device)
    if s["state"] is not None:
        mem += s["state"].detach().double()
    d_out = order(s["d_out"]).double() if s["train"] else None
    # what a ply keeps of the memory before it: nothing if a game starts there
    keep = torch.where(starts[..., None, None, None], 0.0, lam)                     # (t, b, h, 1, 1)
    live = torch.arange(t, device=q.device)[:, None] < count
    out = torch.zeros(t, b, h, dv, dtype=torch.float64, device=q.device)
    dq = torch.zeros_like(q) if s["train"] else None
    on = live[..., None, None, None]
    for i in range(t):
        new = mem * keep[i]
        new = torch.where(on[i], torch.addcmul(new, k[i][..., None], v[i][..., None, :]), mem)
        mem = new
        out[i] = torch.where(on[i][..., 0], (q[i][..., None, :] @ mem)[..., 0, :] * scale, 0.0)
        if s["train"]:
            dq[i] = torch.where(on[i][..., 0], (mem @ d_out[i][..., None])[..., 0] * scale, 0.0)
    back = (lambda x: x) if s["time_major"] else (lambda x: x.transpose(0, 1))
    res = {"out": back(out), "state": mem}
    if not s["train"]:
        return res
    d_mem = torch.zeros_like(mem) if s["state"] is None else s["d_state"].double().clone()
    d_k, d_v = torch.zeros_like(k), torch.zeros_like(v)
    for i in reversed(range(t)):
        full = torch.addcmul(d_mem, q[i][..., None], d_out[i][..., None, :], value=scale)
        d_k[i] = torch.where(on[i][..., 0], (full @ v[i][..., None])[..., 0], 0.0)
        d_v[i] = torch.where(on[i][..., 0], (k[i][..., None, :] @ full)[..., 0, :], 0.0)
        d_mem = torch.where(on[i], full * keep[i], d_mem)
    return {**res, "grads": (back(dq), back(d_k), back(d_v)) + ((d_mem,) if s["state"] is not None else ())}


def exact(case, seed):
    s = prepare(case, seed)
    kind, train = s["kind"], s["train"]
    if kind == "attention":
        with torch.no_grad():
            return _exact_attention(s)
    if kind == "step":
        rows = s["rows"] if s["rows"] is not None else torch.arange(case["games"], device="cuda")
        mem = s["memory"].double()
        old = torch.where(s["starts"][:, None, None, None], 0.0, mem[rows])
        mem[rows] = torch.exp(s["log_decay"].double())[:, None, None] * old + torch.einsum(
            "bhk,bhv->bhkv", s["k"].double(), s["v"].double())
        return {"out": (s["q"].double()[..., None] * mem[rows]).sum(-2) * s["scale"], "state": mem}
    if kind == "rotary":
        x = s["x"].detach().double().cpu().numpy()
        pos, freq = s["positions"].cpu().numpy().astype(np.float64), s["frequencies"].cpu().numpy().astype(np.float64)
        axis = s["axis"].cpu().numpy()
        turn = np.exp(1j * pos[:, axis] * freq)[:, None, :]
        p = freq.size
        first = np.arange(p) * 2 if s["interleaved"] else np.arange(p)
        second = first + 1 if s["interleaved"] else first + p

        def turned(a, by):
            z = (a[..., first] + 1j * a[..., second]) * by
            y = a.copy()
            y[..., first], y[..., second] = z.real, z.imag
            return y

        out = {"out": turned(x, turn)}
        if train:
            out["grads"] = (turned(s["d_out"].double().cpu().numpy(), np.conj(turn)),)
        return out
    x, w, b = (s[n].detach().double() for n in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    r = 1.0 / torch.sqrt(var + s["eps"])
    hat = (x - mean) * r
    out = {"out": hat * w + b}
    if train:
        d = s["d_out"].double()
        gw = d * w
        dx = r * (gw - gw.mean(-1, keepdim=True) - hat * (gw * hat).mean(-1, keepdim=True))
        out["grads"] = (dx, (d * hat).sum(0), d.sum(0))
    return out
