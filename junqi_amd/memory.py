"""Operators of a policy's memory over the plies of a game: linear attention with
a decay for each head (segments of plies with their backward pass, and the step
of one ply), rotary positions with several axes, layer norm, and a selective state
space scan with its causal convolution (segments with their backward passes, and the
steps of one ply), through the jq_attention_*, jq_rotary, jq_layer_norm_*, jq_scan_*
and jq_conv_* kernels.

The opponents' pieces are hidden, so what a policy answers depends on the plies
before. A state of fixed size for each game and head keeps them: `linear_attention`
learns it from rollout segments, in which games end and start anew, and
`linear_attention_step` carries it along with the environment's games; so do
`selective_scan` and `causal_conv` with theirs, whose memory forgets as the plies
tell it to.

Tensors must be on the GPU (there is no host path), in float32 or bfloat16;
sums, statistics and states are float32. Where linear attention's bfloat16 results
are products with float32 operands (a state, the weights of the plies), these are
taken with 16 bits, so that the result's own rounding is what it is off by. Calls run
on torch's current stream and do not synchronise, and may be captured in graphs; a
backward pass is captured with leaves that no eager autograd graph still holds (detached
ones of its own), because autograd would wait for the eager graph's stream within the
capture. Wrong arguments raise ValueError.
"""

from __future__ import annotations

import contextlib
import ctypes as C

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _lib as L
from ._lib import check, lib

_DTYPES = {torch.float32: L.F32, torch.bfloat16: L.BF16}


_same_device = contextlib.nullcontext()


def _on(t: torch.Tensor):
    """The device of `t` made current, where it is not: the kernels launch there."""
    return _same_device if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def _stream(t: torch.Tensor) -> int:
    """torch.cuda.current_stream(t.device).cuda_stream without the Stream object: a
    tenth of its 3 us, which counts in a call of 15."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _rows(t: torch.Tensor) -> L.Rows:
    """A (batch, plies, heads, dim) tensor with adjacent elements for the C calls."""
    b, p, h, _ = t.stride()
    return L.Rows(t.data_ptr(), b, p, h)


def _adjacent(t: torch.Tensor) -> torch.Tensor:
    """`t`, or a copy of it, with the elements of its last dimension adjacent."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _like(t: torch.Tensor) -> torch.Tensor:
    """A new tensor of t's shape and, where it can be kept, t's order of dimensions."""
    out = torch.empty_like(t)
    return out if out.stride(-1) == 1 or t.shape[-1] == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _differentiated(*tensors: torch.Tensor | None) -> bool:
    """Whether autograd has to see the call: an input requires a gradient, or may have
    a forward-mode tangent, which the autograd functions refuse."""
    return forward_ad._current_level >= 0 or (
        torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


def _check_rows(name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have the type and device of the other tensors: "
                         f"{t.dtype} on {t.device}, not {like.dtype} on {like.device}")


def _check(name: str, t: torch.Tensor, shape: tuple[int, ...], dtypes: tuple[torch.dtype, ...], like: torch.Tensor) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, got {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d).removeprefix('torch.') for d in dtypes)}, got {t.dtype}")


def _check_decay(log_decay: torch.Tensor, heads: int, like: torch.Tensor) -> torch.Tensor:
    _check("log_decay", log_decay, (heads,), (torch.float32,), like)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("log_decay is a fixed schedule: it has no gradient (detach it)")
    return log_decay.contiguous()


_INT_MAX = 2 ** 31 - 1   # sizes past it would reach the C calls cut off
_MOST_STEPPED = _INT_MAX - 1024


def _check_dims(batch: int, plies: int, heads: int, key_dim: int, value_dim: int) -> None:
    if not (1 <= key_dim <= L.ATTENTION_MAX_DIM and 1 <= value_dim <= L.ATTENTION_MAX_DIM):
        raise ValueError(f"head dims must be in [1, {L.ATTENTION_MAX_DIM}], got {key_dim} for keys and {value_dim} for values")
    if heads < 1:
        raise ValueError("there must be a head")
    if batch * heads >= 1 << 23 or heads > _INT_MAX:   # heads of no game too
        raise ValueError(f"{batch} games of {heads} heads are too many")
    if plies > _MOST_STEPPED:
        raise ValueError(f"{plies} plies are too many")


# ------------------------------------------------------------------ linear attention
def _attention_args(q, k, v, log_decay, starts, lengths, initial, scale) -> L.Attention:
    b, t, h, dk = q.shape
    a = L.Attention(_DTYPES[q.dtype], b, t, h, dk, v.shape[-1], scale, log_decay.data_ptr())
    if starts is not None:
        a.starts = starts.data_ptr()
        a.starts_batch, a.starts_ply = starts.stride()
    a.lengths = _ptr(lengths)
    a.initial_state = _ptr(initial)
    a.q, a.k, a.v = _rows(q), _rows(k), _rows(v)
    return a


def _workspace(a: L.Attention, backward: bool, like: torch.Tensor) -> torch.Tensor | None:
    need = C.c_int64()
    check(lib.jq_attention_workspace(C.byref(a), backward, C.byref(need)))
    if not need.value:
        return None
    w = torch.empty(need.value, dtype=torch.uint8, device=like.device)
    a.workspace, a.workspace_bytes = w.data_ptr(), need.value
    return w


def _attention_forward(q, k, v, log_decay, starts, lengths, initial, scale, with_state):
    b, t, h, dk = q.shape
    a = _attention_args(q, k, v, log_decay, starts, lengths, initial, scale)
    out = _like(v)
    final = torch.empty((b, h, dk, v.shape[-1]), dtype=torch.float32, device=q.device) if with_state else None
    a.out, a.final_state = _rows(out), _ptr(final)
    with _on(q):
        work = _workspace(a, False, q)   # noqa: F841  (kept until the launch)
        check(lib.jq_attention_forward(C.byref(a), _stream(q)))
    return out, final


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, starts, lengths, initial, scale, with_state):
        out, final = _attention_forward(q, k, v, log_decay, starts, lengths, initial, scale, with_state)
        ctx.save_for_backward(q, k, v, log_decay, starts, lengths, initial)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_final):
        q, k, v, log_decay, starts, lengths, initial = ctx.saved_tensors
        if d_out is None and d_final is None:
            return (None,) * 9
        d_out = torch.zeros_like(v) if d_out is None else _adjacent(d_out)
        a = _attention_args(q, k, v, log_decay, starts, lengths, initial, ctx.scale)
        need = ctx.needs_input_grad
        dq = _like(q) if need[0] else None
        dk = dv = d_initial = None
        if need[1] or need[2] or need[6]:
            dk, dv = _like(k), _like(v)
        if need[6]:
            d_initial = torch.empty_like(initial)
        if d_final is not None:
            d_final = d_final.contiguous()
        a.d_out = _rows(d_out)
        if dq is not None:
            a.dq = _rows(dq)
        if dk is not None:
            a.dk, a.dv = _rows(dk), _rows(dv)
        a.d_final, a.d_initial = _ptr(d_final), _ptr(d_initial)
        with _on(q):
            work = _workspace(a, True, q)   # noqa: F841
            check(lib.jq_attention_backward(C.byref(a), _stream(q)))
        return dq, dk if need[1] else None, dv if need[2] else None, None, None, None, d_initial, None, None


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                     starts: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                     initial_state: torch.Tensor | None = None, scale: float | None = None,
                     return_state: bool = False):
    """Linear attention with a decay for each head, over segments of plies.

    For each game and head, with ``lambda = exp(log_decay)`` and a (key_dim,
    value_dim) state S that begins as ``initial_state`` (zeros if None):

        S = (0 if starts[t] else lambda * S) + k[t]^T v[t];   out[t] = scale * q[t] S

    ``q``, ``k`` (B, T, H, key_dim) and ``v`` (B, T, H, value_dim), float32 or
    bfloat16, dims up to 128, any strides (time-major rollout buffers go in as
    transposed views); ``log_decay`` (H,) float32, at most 0, a fixed schedule
    without a gradient; ``starts`` (B, T) bool or uint8, where a game starts: it
    sees nothing of the plies before; ``lengths`` (B,) int32 or int64: plies from
    there on (clamped to [0, T]) are padding, their ``out`` and gradients are 0.
    ``scale`` is key_dim ** -0.5 if None. Returns ``out`` (B, T, H, value_dim),
    or with ``return_state`` also the float32 state (B, H, key_dim, value_dim)
    after each game's last ply, to go on from.

    A ply's output depends only on the plies that it sees, also where others hold
    infinities or NaN. Differentiable in q, k, v and initial_state."""
    _check_rows("q", q)
    _check_rows("k", k, q)
    _check_rows("v", v, q)
    if q.ndim != 4 or k.shape != q.shape or v.ndim != 4 or v.shape[:3] != q.shape[:3]:
        raise ValueError("q and k must be (B, T, H, key_dim) and v (B, T, H, value_dim), got "
                         f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    b, t, h, dk = q.shape
    dv = v.shape[3]
    _check_dims(b, t, h, dk, dv)
    log_decay = _check_decay(log_decay, h, q)
    if starts is not None:
        _check("starts", starts, (b, t), (torch.bool, torch.uint8), q)
    if lengths is not None:
        _check("lengths", lengths, (b,), (torch.int32, torch.int64), q)
        lengths = (lengths if lengths.dtype == torch.int32 else lengths.clamp(0, t).to(torch.int32)).contiguous()
    if initial_state is not None:
        _check("initial_state", initial_state, (b, h, dk, dv), (torch.float32,), q)
        initial_state = initial_state.contiguous()
    scale = dk ** -0.5 if scale is None else float(scale)
    q, k, v = _adjacent(q), _adjacent(k), _adjacent(v)
    if _differentiated(q, k, v, initial_state):
        out, state = _Attention.apply(q, k, v, log_decay, starts, lengths, initial_state, scale, return_state)
    else:
        out, state = _attention_forward(q, k, v, log_decay, starts, lengths, initial_state, scale, return_state)
    return (out, state) if return_state else out


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, *, rows: torch.Tensor | None = None,
                          starts: torch.Tensor | None = None, scale: float | None = None,
                          out: torch.Tensor | None = None) -> torch.Tensor:
    """`linear_attention` of one new ply of each game, its state updated in place.

    ``q``, ``k`` (B, H, key_dim), ``v`` (B, H, value_dim); ``state`` (R, H,
    key_dim, value_dim) float32, contiguous. Game b's state is row ``rows[b]``
    (B,) int64 (row b if None, then R = B): for a memory of each seat, game * 4 +
    seat. A game whose row is outside [0, R) is left out, its output 0; no row may
    be named twice. ``starts`` (B,) bool or uint8: games that start with this ply.
    Returns (B, H, value_dim), written to ``out`` if given. Not differentiable."""
    _check_rows("q", q)
    _check_rows("k", k, q)
    _check_rows("v", v, q)
    if q.ndim != 3 or k.shape != q.shape or v.ndim != 3 or v.shape[:2] != q.shape[:2]:
        raise ValueError("q and k must be (B, H, key_dim) and v (B, H, value_dim), got "
                         f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    b, h, dk = q.shape
    dv = v.shape[2]
    _check_dims(b, 1, h, dk, dv)
    log_decay = _check_decay(log_decay, h, q)
    if not isinstance(state, torch.Tensor) or state.ndim != 4:
        raise ValueError("state must be an (R, H, key_dim, value_dim) tensor")
    _check("state", state, (state.shape[0], h, dk, dv), (torch.float32,), q)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise ValueError("linear_attention_step has no gradient: use linear_attention, or torch.no_grad()")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None
                                              for t in (q, k, v, log_decay, state)):
        raise ValueError("linear_attention_step has no forward-mode derivative")
    if rows is None:
        if state.shape[0] != b:
            raise ValueError(f"state must have a row for each of {b} games, got {state.shape[0]} (or rows to be given)")
    else:
        _check("rows", rows, (b,), (torch.int64,), q)
        rows = rows.contiguous()
    if starts is not None:
        _check("starts", starts, (b,), (torch.bool, torch.uint8), q)
        starts = starts.contiguous()
    if out is None:
        out = torch.empty((b, h, dv), dtype=q.dtype, device=q.device)
    else:
        _check("out", out, (b, h, dv), (q.dtype,), q)
        if dv > 1 and out.stride(2) != 1:
            raise ValueError("the elements of out's last dimension must be adjacent")
        if (b > 1 and out.stride(0) == 0) or (h > 1 and out.stride(1) == 0):
            raise ValueError("the rows of out must not share memory")
        if torch.is_grad_enabled() and out.requires_grad:
            raise ValueError("out must not require a gradient: what is written to it has none")
    q, k, v = _adjacent(q), _adjacent(k), _adjacent(v)
    r = [L.Rows(x.data_ptr(), x.stride(0), 0, x.stride(1)) for x in (q, k, v, out)]
    with _on(q):
        check(lib.jq_attention_step(_DTYPES[q.dtype], b, h, dk, dv, dk ** -0.5 if scale is None else float(scale),
                                    log_decay.data_ptr(), r[0], r[1], r[2], r[3], state.data_ptr(), state.shape[0],
                                    _ptr(rows), _ptr(starts), _stream(q)))
    increment_version((state, out))   # autograd: what saved them may not use them any more
    return out


# ------------------------------------------------------------------ rotary positions
def rotary_frequencies(sections, base: float = 10000.0, device=None) -> torch.Tensor:
    """Radians per unit of position for `rotary`: each axis with n pairs has its
    own ladder base ** (-i / n), i = 0 .. n - 1. (sum of sections,) float32."""
    f = [base ** (-torch.arange(n, dtype=torch.float64) / n) for n in sections]
    return torch.cat(f).to(torch.float32).to(device)


def _rotary_call(x, positions, frequencies, ends, interleaved, inverse):
    x = _adjacent(x)
    out = _like(x)
    x4, o4, p3 = (t if x.ndim == 4 else t.unsqueeze(0) for t in (x, out, positions))
    n0, n1, h, d = x4.shape
    with _on(x):
        check(lib.jq_rotary(_DTYPES[x.dtype], n0, n1, h, d, frequencies.numel(), _rows(x4), _rows(o4),
                            p3.data_ptr(), p3.dtype == torch.int64, p3.stride(0), p3.stride(1), len(ends), ends,
                            frequencies.data_ptr(), interleaved, inverse, _stream(x)))
    return out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, frequencies, ends, interleaved):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = ends, interleaved
        return _rotary_call(x, positions, frequencies, ends, interleaved, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        positions, frequencies = ctx.saved_tensors
        ends, interleaved = ctx.how
        return _rotary_call(d_out, positions, frequencies, ends, interleaved, True), None, None, None, None


def rotary(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, sections, *,
           interleaved: bool = False) -> torch.Tensor:
    """Rotary positions with several axes: a ply's token at (ply, row, column), a
    board cell's at (row, column).

    ``x`` (..., H, D) float32 or bfloat16 of any strides; ``positions`` (..., A)
    int32 or int64 of the same leading shape, at most 4 axes; ``frequencies``
    (P,) float32 radians per unit of position (`rotary_frequencies`), 2 P <= D;
    ``sections`` A whole numbers with the sum P: the first sections[0] pairs turn
    with axis 0, and so on. Pair p is elements (p, P + p), or (2p, 2p + 1) if
    ``interleaved``; the elements past 2 P stay as they are. Angles are taken in
    64 bits, so far plies lose nothing. Differentiable in x."""
    _check_rows("x", x)
    if x.ndim < 3:
        raise ValueError(f"x must be (..., H, D) with tokens before them, got {tuple(x.shape)}")
    sections = [int(n) for n in sections]
    axes, pairs, d = len(sections), sum(sections), x.shape[-1]
    if not 1 <= axes <= L.ROTARY_MAX_AXES or min(sections) < 0:
        raise ValueError(f"sections must be 1 to {L.ROTARY_MAX_AXES} counts of pairs, got {sections}")
    if not 0 < 2 * pairs <= d or pairs > L.ROTARY_MAX_PAIRS:
        raise ValueError(f"{pairs} pairs do not fit heads of {d} elements (at most {L.ROTARY_MAX_PAIRS} pairs)")
    if x.shape[-2] * d > _INT_MAX:
        raise ValueError(f"{x.shape[-2]} heads of {d} elements are too many")
    _check("positions", positions, (*x.shape[:-2], axes), (torch.int32, torch.int64), x)
    _check("frequencies", frequencies, (pairs,), (torch.float32,), x)
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise ValueError("frequencies are fixed: they have no gradient (detach them)")
    ends = (C.c_int32 * axes)(*(sum(sections[:i + 1]) for i in range(axes)))
    positions, frequencies = _adjacent(positions), frequencies.contiguous()
    shape = x.shape
    if x.ndim > 4:
        x, positions = x.flatten(0, -3), positions.flatten(0, -2)
    if _differentiated(x):
        out = _Rotary.apply(x, positions, frequencies, ends, bool(interleaved))
    else:
        out = _rotary_call(x, positions, frequencies, ends, bool(interleaved), False)
    return out.reshape(shape)


# ------------------------------------------------------------------ layer norm
def _norm_forward(x2, weight, bias, eps, with_stats):
    n, w = x2.shape
    out = torch.empty((n, w), dtype=x2.dtype, device=x2.device)
    mean = rstd = None
    if with_stats:
        mean, rstd = torch.empty((2, n), dtype=torch.float32, device=x2.device).unbind(0)
    wd = weight if weight is not None else bias
    with _on(x2):
        check(lib.jq_layer_norm_forward(_DTYPES[x2.dtype], _DTYPES[wd.dtype if wd is not None else x2.dtype], n, w,
                                        x2.data_ptr(), x2.stride(0), _ptr(weight), _ptr(bias), eps, out.data_ptr(), w,
                                        _ptr(mean), _ptr(rstd), _stream(x2)))
    return out, mean, rstd


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, weight, bias, eps):
        out, mean, rstd = _norm_forward(x2, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.weight_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else x2.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        x2, weight, mean, rstd = ctx.saved_tensors
        n, w = x2.shape
        need = ctx.needs_input_grad
        d_out = _adjacent(d_out)
        dx = torch.empty((n, w), dtype=x2.dtype, device=x2.device) if need[0] else None
        dw = torch.empty(w, dtype=ctx.weight_dtype, device=x2.device) if need[1] else None
        db = torch.empty(w, dtype=ctx.weight_dtype, device=x2.device) if need[2] else None
        size = C.c_int64()
        work = None
        if need[1] or need[2]:
            check(lib.jq_layer_norm_workspace(n, w, C.byref(size)))
            work = torch.empty(size.value, dtype=torch.uint8, device=x2.device)
        with _on(x2):
            check(lib.jq_layer_norm_backward(_DTYPES[x2.dtype], _DTYPES[ctx.weight_dtype], n, w, x2.data_ptr(),
                                             x2.stride(0), _ptr(weight), mean.data_ptr(), rstd.data_ptr(),
                                             d_out.data_ptr(), d_out.stride(0), _ptr(dx), w, _ptr(dw), _ptr(db),
                                             _ptr(work), size.value, _stream(x2)))
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension of ``x`` (..., width), float32 or
    bfloat16: (x - mean) / sqrt(variance + eps) * weight + bias, the statistics
    in float32. ``weight`` and ``bias`` (width,) are float32 or of x's type, both
    of one; None stands for ones and zeros. Differentiable in all three; the
    gradients of weight and bias are summed in a fixed order."""
    _check_rows("x", x)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be (..., width) with a positive width, got {tuple(x.shape)}")
    w = x.shape[-1]
    if w > _MOST_STEPPED:
        raise ValueError(f"rows of {w} elements are too wide")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check(name, t, (w,), (torch.float32, x.dtype), x)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    x2 = _adjacent(x).reshape(-1, w)
    if _differentiated(x, weight, bias):
        out = _Norm.apply(x2, weight, bias, float(eps))
    else:
        out = _norm_forward(x2, weight, bias, float(eps), False)[0]
    return out.reshape(x.shape)


# ------------------------------------------------------------------ what segments and steps of channels share
def _plies(t: torch.Tensor) -> L.Rows:
    """A (batch, plies, channels) tensor with adjacent elements for the C calls."""
    s = t.stride()
    return L.Rows(t.data_ptr(), s[0], s[1], 0)


def _ply(t: torch.Tensor) -> L.Rows:
    """A (batch, channels) tensor, or (batch, groups, states), with adjacent elements."""
    s = t.stride()
    return L.Rows(t.data_ptr(), s[0], 0, s[1] if len(s) == 3 else 0)


def _like_plies(t: torch.Tensor) -> torch.Tensor:
    """`_like` of rows that may be broadcast: no two elements of the result share memory."""
    return _like(t) if 0 not in t.stride() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _check_sizes(batch: int, plies: int, channels: int) -> None:
    if channels < 1:
        raise ValueError("there must be a channel")
    if batch > L.MOST_GAMES or plies > L.MOST_PLIES or channels > L.MOST_CHANNELS:
        raise ValueError(f"{batch} games of {plies} plies of {channels} channels are too many")


def _check_segments(starts, lengths, b: int, t: int, like: torch.Tensor):
    """lengths as the C calls take them."""
    if starts is not None:
        _check("starts", starts, (b, t), (torch.bool, torch.uint8), like)
    if lengths is not None:
        _check("lengths", lengths, (b,), (torch.int32, torch.int64), like)
        lengths = (lengths if lengths.dtype == torch.int32 else lengths.clamp(0, t).to(torch.int32)).contiguous()
    return lengths


def _set_segments(a, starts, lengths) -> None:
    if starts is not None:
        a.starts = starts.data_ptr()
        a.starts_batch, a.starts_ply = starts.stride()
    a.lengths = _ptr(lengths)


def _give_workspace(a, need: C.c_int64, like: torch.Tensor) -> torch.Tensor | None:
    if not need.value:
        return None
    w = torch.empty(need.value, dtype=torch.uint8, device=like.device)
    a.workspace, a.workspace_bytes = w.data_ptr(), need.value
    return w


def _check_step(name: str, x: torch.Tensor, state: torch.Tensor, state_shape: tuple[int, ...], dtype: torch.dtype,
                rows, starts, out, inputs):
    """rows, starts and out as the C calls take them, and the checks of a step that updates `state` in place."""
    b = x.shape[0]
    if not isinstance(state, torch.Tensor) or state.ndim != 3:
        raise ValueError(f"state must be an (R, {state_shape[0]}, {state_shape[1]}) tensor")
    _check("state", state, (state.shape[0], *state_shape), (dtype,), x)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is updated in place")
    grads = torch.is_grad_enabled()
    if grads:
        for t in (state, *inputs):
            if t is not None and t.requires_grad:
                raise ValueError(f"{name}_step has no gradient: use {name}, or torch.no_grad()")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in (*inputs, state)):
        raise ValueError(f"{name}_step has no forward-mode derivative")
    if rows is None:
        if state.shape[0] != b:
            raise ValueError(f"state must have a row for each of {b} games, got {state.shape[0]} (or rows to be given)")
    else:
        _check("rows", rows, (b,), (torch.int64,), x)
        rows = rows.contiguous()
    if starts is not None:
        _check("starts", starts, (b,), (torch.bool, torch.uint8), x)
        starts = starts.contiguous()
    if out is None:
        out = x.new_empty(x.shape)
    else:
        _check("out", out, tuple(x.shape), (x.dtype,), x)
        if x.shape[1] > 1 and out.stride(1) != 1:
            raise ValueError("the elements of out's last dimension must be adjacent")
        if b > 1 and out.stride(0) < x.shape[1]:
            raise ValueError("the rows of out must not share memory")
        if grads and out.requires_grad:
            raise ValueError("out must not require a gradient: what is written to it has none")
    return rows, starts, out


# ------------------------------------------------------------------ selective scan
def _near(t: torch.Tensor) -> torch.Tensor:
    """`t` with adjacent elements and plies that the scan's 32-bit offsets reach, or a copy that has them."""
    t = _adjacent(t)
    far = t.shape[1] > 1 and t.stride(1) * t.element_size() > L.SCAN_MAX_PLY_STRIDE
    return t.contiguous() if far else t


def _check_scan(u, delta, a, b, c, skip, gate, delta_bias, lead: int):
    """The checks that segments (lead 2) and steps (lead 1) share; the arguments with one
    group written out and adjacent elements."""
    _check_rows("u", u)
    if u.ndim != lead + 1:
        raise ValueError(f"u must be {'(B, T, D)' if lead == 2 else '(B, D)'}, got {tuple(u.shape)}")
    d = u.shape[-1]
    for name, t in (("delta", delta), ("gate", gate)):
        if t is not None:
            _check_rows(name, t, u)
            if t.shape != u.shape:
                raise ValueError(f"{name} must have u's shape {tuple(u.shape)}, got {tuple(t.shape)}")
    _check_rows("b", b, u)
    _check_rows("c", c, u)
    if b.shape != c.shape or b.ndim not in (lead + 1, lead + 2) or b.shape[:lead] != u.shape[:lead]:
        raise ValueError(f"b and c must be u's rows with (N) or (G, N) elements, got {tuple(b.shape)} and {tuple(c.shape)}")
    if b.ndim == lead + 1:
        b, c = b.unsqueeze(lead), c.unsqueeze(lead)
    groups, n = b.shape[lead:]
    if not 1 <= n <= L.SCAN_MAX_STATES:
        raise ValueError(f"there must be 1 to {L.SCAN_MAX_STATES} states, got {n}")
    if d < 1 or groups < 1 or d % groups:
        raise ValueError(f"{d} channels do not part into {groups} groups")
    _check_sizes(u.shape[0], u.shape[1] if lead == 2 else 1, d)
    _check("a", a, (d, n), (torch.float32,), u)
    for name, t in (("skip", skip), ("delta_bias", delta_bias)):
        if t is not None:
            _check(name, t, (d,), (torch.float32,), u)
    near = _near if lead == 2 else _adjacent
    return (near(u), near(delta), a.contiguous(), near(b), near(c),
            None if skip is None else skip.contiguous(), None if gate is None else near(gate),
            None if delta_bias is None else delta_bias.contiguous())


def _scan_args(u, delta, a, b, c, skip, gate, delta_bias, softplus, of=_plies, group_of=_rows) -> L.Scan:
    s = L.Scan(_DTYPES[u.dtype], u.shape[0], u.shape[1] if u.ndim == 3 else 1, u.shape[-1], b.shape[-1], b.shape[-2],
               softplus, a.data_ptr(), _ptr(skip), _ptr(delta_bias))
    s.u, s.delta, s.b, s.c = of(u), of(delta), group_of(b), group_of(c)
    if gate is not None:
        s.gate = of(gate)
    return s


def _scan_forward(u, delta, a, b, c, skip, gate, delta_bias, initial, starts, lengths, softplus, with_state, with_saved):
    s = _scan_args(u, delta, a, b, c, skip, gate, delta_bias, softplus)
    _set_segments(s, starts, lengths)
    out = _like_plies(u)
    final = torch.empty((u.shape[0], *a.shape), dtype=torch.float32, device=u.device) if with_state else None
    s.out, s.initial_state, s.final_state = _plies(out), _ptr(initial), _ptr(final)
    saved, need = None, C.c_int64()
    if with_saved:
        check(lib.jq_scan_saved(C.byref(s), C.byref(need)))
        saved = torch.empty(need.value // 4, dtype=torch.float32, device=u.device)
        s.saved = saved.data_ptr()
    with _on(u):
        check(lib.jq_scan_workspace(C.byref(s), 0, C.byref(need)))
        work = _give_workspace(s, need, u)   # noqa: F841  (kept until the launch)
        check(lib.jq_scan_forward(C.byref(s), _stream(u)))
    return out, final, saved


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, a, b, c, skip, gate, delta_bias, initial, starts, lengths, softplus, with_state):
        out, final, saved = _scan_forward(u, delta, a, b, c, skip, gate, delta_bias, initial, starts, lengths, softplus,
                                          with_state, True)
        ctx.save_for_backward(u, delta, a, b, c, skip, gate, delta_bias, starts, lengths, saved)
        ctx.softplus = softplus
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_final):
        u, delta, a, b, c, skip, gate, delta_bias, starts, lengths, saved = ctx.saved_tensors
        if d_out is None and d_final is None:
            return (None,) * 13
        d_out = torch.zeros_like(u) if d_out is None else _near(d_out)
        s = _scan_args(u, delta, a, b, c, skip, gate, delta_bias, ctx.softplus)
        _set_segments(s, starts, lengths)
        need = ctx.needs_input_grad
        grads = [None if x is None or not need[i] else
                 torch.empty_like(x) if i in (2, 5, 7) else _like_plies(x)
                 for i, x in enumerate((u, delta, a, b, c, skip, gate, delta_bias))]
        du, ddelta, da, db, dc, dskip, dgate, dbias = grads
        d_initial = torch.empty((u.shape[0], *a.shape), dtype=torch.float32, device=u.device) if need[8] else None
        if d_final is not None:
            d_final = d_final.contiguous()
        s.saved, s.d_out = saved.data_ptr(), _plies(d_out)
        for name, t in (("du", du), ("ddelta", ddelta), ("dgate", dgate)):
            if t is not None:
                setattr(s, name, _plies(t))
        for name, t in (("db", db), ("dc", dc)):
            if t is not None:
                setattr(s, name, _rows(t))
        s.da, s.dskip, s.ddelta_bias = _ptr(da), _ptr(dskip), _ptr(dbias)
        s.d_final, s.d_initial = _ptr(d_final), _ptr(d_initial)
        size = C.c_int64()
        with _on(u):
            check(lib.jq_scan_workspace(C.byref(s), 1, C.byref(size)))
            work = _give_workspace(s, size, u)   # noqa: F841
            check(lib.jq_scan_backward(C.byref(s), _stream(u)))
        return (*grads, d_initial, None, None, None, None)


def selective_scan(u: torch.Tensor, delta: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, *,
                   skip: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                   delta_bias: torch.Tensor | None = None, softplus: bool = False,
                   starts: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                   initial_state: torch.Tensor | None = None, return_state: bool = False):
    """A state space scan whose steps depend on the input, over segments of plies.

    For each game, channel d and state n, with ``dt = softplus(delta + delta_bias)``
    (without the softplus if not ``softplus``) and a state h that begins as
    ``initial_state`` (zeros if None):

        h = exp(dt[t] * a[d, n]) * (0 if starts[t] else h) + dt[t] * u[t] * b[t, n]
        out[t] = (sum over n of c[t, n] * h + skip[d] * u[t]) * silu(gate[t])

    ``u``, ``delta``, ``gate`` (B, T, D) and ``b``, ``c`` (B, T, N) or (B, T, G, N),
    all float32 or all bfloat16, up to 64 states, any strides (time-major rollout
    buffers go in as transposed views); with G groups, channel d has those of group
    d // (D / G). ``a`` (D, N), ``skip`` and ``delta_bias`` (D,) float32. ``starts``
    and ``lengths`` as in `linear_attention`: a game that starts sees nothing of the
    plies before, plies from a game's length on are padding, their ``out`` and
    gradients 0. A ply's decay below 2^-126 counts as 0, one past float32's end as
    infinite (it makes NaN of a state of 0). Returns ``out`` (B, T, D), or with
    ``return_state`` also the float32 state (B, D, N) after each game's last ply.

    Differentiable in u, delta, a, b, c, skip, gate, delta_bias and initial_state;
    sums over plies and channels are taken in a fixed order. The backward pass keeps the
    state before every eighth ply, B * ceil(T / 8) * D * N float32."""
    u, delta, a, b, c, skip, gate, delta_bias = _check_scan(u, delta, a, b, c, skip, gate, delta_bias, 2)
    lengths = _check_segments(starts, lengths, u.shape[0], u.shape[1], u)
    if initial_state is not None:
        _check("initial_state", initial_state, (u.shape[0], *a.shape), (torch.float32,), u)
        initial_state = initial_state.contiguous()
    args = (u, delta, a, b, c, skip, gate, delta_bias, initial_state, starts, lengths, bool(softplus), return_state)
    if _differentiated(*args[:9]):
        out, state = _Scan.apply(*args)
    else:
        out, state, _ = _scan_forward(*args, False)
    return (out, state) if return_state else out


def selective_scan_step(u: torch.Tensor, delta: torch.Tensor, a: torch.Tensor, b: torch.Tensor, c: torch.Tensor,
                        state: torch.Tensor, *, skip: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                        delta_bias: torch.Tensor | None = None, softplus: bool = False,
                        rows: torch.Tensor | None = None, starts: torch.Tensor | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """`selective_scan` of one new ply of each game, its state updated in place.

    ``u``, ``delta``, ``gate`` (B, D), ``b``, ``c`` (B, N) or (B, G, N); ``state``
    (R, D, N) float32, contiguous; ``rows``, ``starts`` and ``out`` as in
    `linear_attention_step`: a game whose row is outside [0, R) is left out, its output
    0, and no row may be named twice; the rows of ``out`` share no memory, and none with
    the other arguments. Returns (B, D). Not differentiable."""
    given = (u, delta, a, b, c, skip, gate, delta_bias)
    u, delta, a, b, c, skip, gate, delta_bias = _check_scan(*given, 1)
    rows, starts, out = _check_step("selective_scan", u, state, tuple(a.shape), torch.float32, rows, starts, out, given)
    s = _scan_args(u, delta, a, b, c, skip, gate, delta_bias, bool(softplus), _ply, _ply)
    s.out = _ply(out)
    with _on(u):
        check(lib.jq_scan_step(C.byref(s), state.data_ptr(), state.shape[0], _ptr(rows), _ptr(starts), _stream(u)))
    increment_version((state, out))   # autograd: what saved them may not use them any more
    return out


# ------------------------------------------------------------------ causal convolution
def _check_conv(x, weight, bias, lead: int):
    _check_rows("x", x)
    if x.ndim != lead + 1:
        raise ValueError(f"x must be {'(B, T, D)' if lead == 2 else '(B, D)'}, got {tuple(x.shape)}")
    d = x.shape[-1]
    _check_sizes(x.shape[0], x.shape[1] if lead == 2 else 1, d)
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2:
        raise ValueError("weight must be a (D, taps) tensor")
    taps = weight.shape[1]
    if not 1 <= taps <= L.CONV_MAX_TAPS:
        raise ValueError(f"there must be 1 to {L.CONV_MAX_TAPS} taps, got {taps}")
    _check("weight", weight, (d, taps), (torch.float32, x.dtype), x)
    if bias is not None:
        _check("bias", bias, (d,), (weight.dtype,), x)
        bias = bias.contiguous()
    return _adjacent(x), weight.contiguous(), bias


def _conv_args(x, weight, bias, silu, of=_plies) -> L.Conv:
    v = L.Conv(_DTYPES[x.dtype], _DTYPES[weight.dtype], x.shape[0], x.shape[1] if x.ndim == 3 else 1, x.shape[-1],
               weight.shape[1], silu, weight.data_ptr(), _ptr(bias))
    v.x = of(x)
    return v


def _conv_forward(x, weight, bias, initial, starts, lengths, silu, with_state):
    v = _conv_args(x, weight, bias, silu)
    _set_segments(v, starts, lengths)
    out = _like_plies(x)
    final = None
    if with_state:
        final = torch.empty((x.shape[0], weight.shape[1] - 1, x.shape[2]), dtype=x.dtype, device=x.device)
    v.out, v.initial_state, v.final_state = _plies(out), _ptr(initial), _ptr(final)
    with _on(x):
        check(lib.jq_conv_forward(C.byref(v), _stream(x)))
    return out, final


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial, starts, lengths, silu, with_state):
        out, final = _conv_forward(x, weight, bias, initial, starts, lengths, silu, with_state)
        ctx.save_for_backward(x, weight, bias, initial, starts, lengths)
        ctx.silu = silu
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_final):
        x, weight, bias, initial, starts, lengths = ctx.saved_tensors
        if d_out is None and d_final is None:
            return (None,) * 8
        d_out = torch.zeros_like(x) if d_out is None else _adjacent(d_out)
        v = _conv_args(x, weight, bias, ctx.silu)
        _set_segments(v, starts, lengths)
        need = ctx.needs_input_grad
        dx = _like_plies(x) if need[0] else None
        dw = torch.empty_like(weight) if need[1] else None
        db = torch.empty_like(bias) if need[2] else None
        d_initial = torch.empty_like(initial) if need[3] else None
        if d_final is not None:
            d_final = d_final.contiguous()
        v.initial_state, v.d_out = _ptr(initial), _plies(d_out)
        if dx is not None:
            v.dx = _plies(dx)
        v.dweight, v.dbias, v.d_final, v.d_initial = _ptr(dw), _ptr(db), _ptr(d_final), _ptr(d_initial)
        size = C.c_int64()
        with _on(x):
            check(lib.jq_conv_workspace(C.byref(v), C.byref(size)))
            work = _give_workspace(v, size, x)   # noqa: F841
            check(lib.jq_conv_backward(C.byref(v), _stream(x)))
        return dx, dw, db, d_initial, None, None, None, None


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, silu: bool = False,
                starts: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                initial_state: torch.Tensor | None = None, return_state: bool = False):
    """A causal convolution of each channel over its last few plies, as it stands before
    `selective_scan`.

        out[t] = bias[d] + sum over j < taps of weight[d, j] * x[t - taps + 1 + j],

    then silu(out) if ``silu``. ``x`` (B, T, D) float32 or bfloat16, any strides;
    ``weight`` (D, taps), up to 8 taps, and ``bias`` (D,) float32 or of x's type, both
    of one. Inputs before a game's start (``starts``) are 0, those before the first ply
    are ``initial_state`` (B, taps - 1, D) of x's type, the oldest first (zeros if
    None); ``lengths`` as in `linear_attention`. Returns ``out`` (B, T, D), or with
    ``return_state`` also the last taps - 1 inputs of each game, to go on from.

    Differentiable in x, weight, bias and initial_state; the gradients of weight and
    bias are summed in a fixed order."""
    x, weight, bias = _check_conv(x, weight, bias, 2)
    b, t, d = x.shape
    lengths = _check_segments(starts, lengths, b, t, x)
    if initial_state is not None:
        _check("initial_state", initial_state, (b, weight.shape[1] - 1, d), (x.dtype,), x)
        initial_state = initial_state.contiguous()
    args = (x, weight, bias, initial_state, starts, lengths, bool(silu), return_state)
    out, state = (_Conv.apply if _differentiated(*args[:4]) else _conv_forward)(*args)
    return (out, state) if return_state else out


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, state: torch.Tensor, bias: torch.Tensor | None = None, *,
                     silu: bool = False, rows: torch.Tensor | None = None, starts: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """`causal_conv` of one new ply of each game, its last inputs updated in place.

    ``x`` (B, D); ``state`` (R, taps - 1, D) of x's type, contiguous; ``rows``,
    ``starts`` and ``out`` as in `linear_attention_step`: a game whose row is outside
    [0, R) is left out, its output 0, and no row may be named twice; the rows of ``out``
    share no memory, and none with the other arguments. Returns (B, D). Not
    differentiable."""
    given = (x, weight, bias)
    x, weight, bias = _check_conv(*given, 1)
    rows, starts, out = _check_step("causal_conv", x, state, (weight.shape[1] - 1, x.shape[1]), x.dtype, rows, starts, out,
                                    given)
    v = _conv_args(x, weight, bias, bool(silu), _ply)
    v.out = _ply(out)
    with _on(x):
        check(lib.jq_conv_step(C.byref(v), state.data_ptr(), state.shape[0], _ptr(rows), _ptr(starts), _stream(x)))
    increment_version((state, out))
    return out
