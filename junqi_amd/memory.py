"""Operators of a policy's memory over the plies of a game: linear attention with
a decay for each head (segments of plies with their backward pass, and the step
of one ply), rotary positions with several axes, and layer norm, through the
jq_attention_*, jq_rotary and jq_layer_norm_* kernels.

The opponents' pieces are hidden, so what a policy answers depends on the plies
before. A state of fixed size for each game and head keeps them: `linear_attention`
learns it from rollout segments, in which games end and start anew, and
`linear_attention_step` carries it along with the environment's games.

Tensors must be on the GPU (there is no host path), in float32 or bfloat16;
sums, statistics and states are float32. Where linear attention's bfloat16 results
are products with float32 operands (a state, the weights of the plies), these are
taken with 16 bits, so that the result's own rounding is what it is off by. Calls run
on torch's current stream and do not synchronise. Wrong arguments raise ValueError.
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
