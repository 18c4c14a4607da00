"""Legal-support storage of rollout buffers: dense bool mask rows <-> per-row id
lists (junqi_rl/training/rollout_gpu.py:119-198), on the device through the
jq_mask_encode / jq_ids_to_mask kernels (jq_mask_count and jq_mask_to_ids where
memory is short).

Same arguments, shapes, dtypes and ValueError checks as the reference's
``_dense_mask_to_csr`` and ``_csr_to_dense_selected``; tensors must be on the
GPU (there is no host path).

`action_logits` puts such masks, or the packed ones of the environment, on a policy's
logits, with penalties of repeated actions and biases (the jq_logits_* kernels; no
counterpart in the reference).
"""

from __future__ import annotations

import ctypes as C
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from ._lib import check, lib
from .memory import _DTYPES, _adjacent, _check, _check_rows, _differentiated, _on, _ptr


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def dense_mask_to_csr(mask: torch.Tensor, out_ids: torch.Tensor, out_counts: torch.Tensor) -> None:
    """Write the True columns of each row of ``mask`` (N, FLAT) bool into
    ``out_ids`` (N, K_MAX) int32, in order, zero-padded, and the per-row count
    into ``out_counts`` (N,) int32. Overflow raises before any output changes."""
    if mask.ndim != 2 or mask.dtype != torch.bool or out_ids.ndim != 2:
        raise ValueError("CSR encoding requires a 2-D bool mask and 2-D ids")
    n, k_max = out_ids.shape
    if k_max <= 0 or mask.shape[0] != n or out_counts.shape != (n,):
        raise ValueError("CSR output shapes must be (N, K>0) and (N,)")
    if out_ids.dtype != torch.int32 or out_counts.dtype != torch.int32:
        raise ValueError("CSR ids and counts must be int32")
    if out_ids.device != mask.device or out_counts.device != mask.device:
        raise ValueError("CSR inputs and outputs must share a device")
    if mask.device.type != "cuda":
        raise ValueError("CSR encoding runs on the GPU: mask must be a CUDA tensor")
    mask = mask.contiguous()
    if not out_ids.is_contiguous() or not out_counts.is_contiguous():
        raise ValueError("CSR outputs must be contiguous")
    s, d = _stream(mask), int(mask.shape[1])
    # the rows are encoded into scratch and published on the device if they all
    # fit; only the largest count comes back, through pinned host memory
    rows = (n * k_max + 3) // 4 * 4
    try:
        work = torch.empty(rows + n, dtype=torch.int32, device=mask.device)
    except torch.OutOfMemoryError:   # no room for a second copy of the ids: count, test, then write them in place
        counts = torch.empty(n, dtype=torch.int32, device=mask.device)
        check(lib.jq_mask_count(mask.data_ptr(), n, d, counts.data_ptr(), s))
        _fits(int(counts.max()), k_max)   # synchronises
        out_counts.copy_(counts)
        check(lib.jq_mask_to_ids(mask.data_ptr(), n, d, k_max, out_ids.data_ptr(), s))
        return
    most = torch.empty(1, dtype=torch.int32, pin_memory=True)   # written by the kernel itself
    p = work.data_ptr()
    check(lib.jq_mask_encode(mask.data_ptr(), n, d, k_max, p, p + 4 * rows, out_ids.data_ptr(),
                             out_counts.data_ptr(), most.data_ptr(), s))
    torch.cuda.current_stream(mask.device).synchronize()   # like the reference's guard
    _fits(int(most), k_max)


def _fits(required: int, k_max: int) -> None:
    if required > k_max:
        raise ValueError(
            f"CSR legal-mask overflow: need {required} entries, capacity {k_max}; "
            "increase rollout.csr_k_max or disable CSR legal-mask storage")


def csr_to_dense_selected(legal_ids: torch.Tensor, legal_counts: torch.Tensor, idx: torch.Tensor,
                          flat_action_dim: int) -> torch.Tensor:
    """Dense (B, flat_action_dim) bool mask of the transitions ``idx`` (B,)
    int64 from (T*N, K_MAX) int32 id lists and their (T*N,) counts."""
    if legal_ids.ndim != 2 or legal_counts.shape != (legal_ids.shape[0],):
        raise ValueError("legal_ids must be (rows, K_MAX) with legal_counts (rows,)")
    if legal_ids.dtype != torch.int32 or legal_counts.dtype != torch.int32:
        raise ValueError("legal_ids and legal_counts must be int32")
    if legal_ids.device.type != "cuda" or legal_counts.device != legal_ids.device or idx.device != legal_ids.device:
        raise ValueError("legal ids, counts and indices must be CUDA tensors on one device")
    ids = legal_ids.contiguous()
    cnt = legal_counts.contiguous()
    sel = idx.to(torch.int64).contiguous().reshape(-1)
    b = int(sel.numel())
    out = torch.empty((b, int(flat_action_dim)), dtype=torch.bool, device=ids.device)
    check(lib.jq_ids_to_mask(ids.data_ptr(), cnt.data_ptr(), int(ids.shape[0]), int(ids.shape[1]), sel.data_ptr(),
                             b, int(flat_action_dim), out.data_ptr(), _stream(ids)))
    return out


# ------------------------------------------------------------------ masked logits
class _Penalties:
    """Each penalty as one number, or as a float32 tensor of the rows' own."""

    def __init__(self, logits, repetition, frequency, presence):
        self.numbers, self.tensors = [1.0, 0.0, 0.0], [None, None, None]
        for i, (name, v) in enumerate((("repetition", repetition), ("frequency", frequency), ("presence", presence))):
            if isinstance(v, torch.Tensor):
                _check(name, v, (logits.shape[0],), (torch.float32,), logits)
                if v.requires_grad and torch.is_grad_enabled():
                    raise ValueError(f"{name} has no gradient (detach it)")
                if forward_ad._current_level >= 0 and forward_ad.unpack_dual(v).tangent is not None:
                    raise ValueError(f"{name} has no forward-mode derivative")
                self.tensors[i] = v.contiguous()
            else:
                self.numbers[i] = C.c_float(float(v)).value   # as the kernel has it
                if not math.isfinite(self.numbers[i]):
                    raise ValueError(f"{name} must be finite in float32, got {v}")
        if self.numbers[0] <= 0.0:
            raise ValueError(f"repetition must be positive in float32, got {repetition}")


def _logits_args(like, logits, bias, legal, recent, lengths, numbers, tensors) -> L.Logits:
    """`like` has the logits' type and shape, where a backward pass has no use for them."""
    g = L.Logits(_DTYPES[like.dtype], L.MASK_BYTES, like.shape[0], like.shape[1])
    g.bias = _ptr(bias)
    if logits is not None:
        g.logits, g.logits_stride = logits.data_ptr(), logits.stride(0)
    if legal is not None:
        g.mask_kind = L.MASK_WORDS_PACKED if legal.dtype == torch.int32 else L.MASK_BYTES
        g.mask, g.mask_stride = legal.data_ptr(), legal.stride(0)
    if recent is not None:
        g.recent_count, g.recent64 = recent.shape[1], recent.dtype == torch.int64
        g.recent, g.recent_stride, g.recent_lengths = recent.data_ptr(), recent.stride(0), _ptr(lengths)
    g.repetition, g.frequency, g.presence = numbers
    g.repetitions, g.frequencies, g.presences = (_ptr(t) for t in tensors)
    return g


def _stream_of(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _logits_forward(logits, bias, legal, recent, lengths, penalties):
    out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    g = _logits_args(logits, logits, bias, legal, recent, lengths, penalties.numbers, penalties.tensors)
    with _on(logits):
        check(lib.jq_logits_forward(C.byref(g), out.data_ptr(), out.shape[1], _stream_of(logits)))
    return out


class _ActionLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, legal, recent, lengths, penalties):
        # only a repetition's gradient looks at the logits
        ctx.save_for_backward(None if recent is None else logits, bias, legal, recent, lengths, *penalties.tensors)
        ctx.numbers = penalties.numbers
        return _logits_forward(logits, bias, legal, recent, lengths, penalties)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        logits, bias, legal, recent, lengths, *tensors = ctx.saved_tensors
        d_out = _adjacent(d_out)
        g = _logits_args(d_out, logits, bias, legal, recent, lengths, ctx.numbers, tensors)
        need = ctx.needs_input_grad
        d_logits = torch.empty(d_out.shape, dtype=d_out.dtype, device=d_out.device) if need[0] else None
        d_bias = torch.empty_like(bias) if need[1] else None
        size, work = C.c_int64(), None
        if need[1]:
            check(lib.jq_logits_workspace(C.byref(g), C.byref(size)))
            work = torch.empty(size.value, dtype=torch.uint8, device=d_out.device)
        with _on(d_out):
            check(lib.jq_logits_backward(C.byref(g), d_out.data_ptr(), d_out.stride(0), _ptr(d_logits), d_out.shape[1],
                                         _ptr(d_bias), _ptr(work), size.value, _stream_of(d_out)))
        return d_logits, d_bias, None, None, None, None


def action_logits(logits: torch.Tensor, *, bias: torch.Tensor | None = None, legal: torch.Tensor | None = None,
                  recent: torch.Tensor | None = None, recent_lengths: torch.Tensor | None = None,
                  repetition: float | torch.Tensor = 1.0, frequency: float | torch.Tensor = 0.0,
                  presence: float | torch.Tensor = 0.0) -> torch.Tensor:
    """A policy's logits with penalties of repeated actions, a bias and the legal mask,
    ready for a softmax.

    ``logits`` (N, A) float32 or bfloat16. Where ``recent`` (N, L) int32 or int64, the
    first ``recent_lengths`` (N,) int32 of each row (all if None), names an action count
    times: x = (x / repetition if x > 0 else x * repetition) - frequency * count -
    presence; each penalty is a finite number, a repetition above 0, or an (N,) float32
    tensor, whose values are not looked at (that would wait for the GPU): the formula is
    taken with them as they are. Ids outside [0, A) are passed over (padding). Then ``bias`` (A,) float32 is added, and actions
    that ``legal`` does not have become -infinity: (N, A) bool, or (N, ceil(A / 32))
    int32 words, bit j of word i for action 32 i + j, as the environment packs them. A
    row without a legal action is all -infinity. Returns (N, A) of logits' type.

    Differentiable in logits and bias; an illegal action's gradient is 0 whatever comes
    in. The environment overwrites its masks in place: give a copy of them to a call
    whose backward pass comes after its next step."""
    _check_rows("logits", logits)
    if logits.ndim != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be (N, A) with an action, got {tuple(logits.shape)}")
    n, a = logits.shape
    if n > 2 ** 31 - 1 or a > 2 ** 31 - 1 - 4096:
        raise ValueError(f"{n} rows of {a} actions are too many")
    if bias is not None:
        _check("bias", bias, (a,), (torch.float32,), logits)
        bias = bias.contiguous()
    if legal is not None:
        if not isinstance(legal, torch.Tensor) or legal.dtype not in (torch.bool, torch.int32):
            raise ValueError("legal must be a bool mask or int32 mask words")
        _check("legal", legal, (n, a if legal.dtype == torch.bool else -(-a // 32)), (legal.dtype,), logits)
        legal = _adjacent(legal)
    if recent is None:
        if recent_lengths is not None:
            raise ValueError("recent_lengths without recent")
    else:
        if not isinstance(recent, torch.Tensor) or recent.ndim != 2 or recent.shape[1] > 2 ** 31 - 257:
            raise ValueError("recent must be an (N, L) tensor")
        _check("recent", recent, (n, recent.shape[1]), (torch.int32, torch.int64), logits)
        recent = _adjacent(recent)
        if recent_lengths is not None:
            _check("recent_lengths", recent_lengths, (n,), (torch.int32,), logits)
            recent_lengths = recent_lengths.contiguous()
    penalties = _Penalties(logits, repetition, frequency, presence)
    logits = _adjacent(logits)
    args = (logits, bias, legal, recent, recent_lengths, penalties)
    return _ActionLogits.apply(*args) if _differentiated(logits, bias) else _logits_forward(*args)
