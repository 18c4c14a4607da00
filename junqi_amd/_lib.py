"""ctypes binding of the C ABI in include/junqi_amd.h.

The shared library is built in-tree by ``junqi_amd/build.py``. If it is missing
this module raises at import time: there is no CPU fallback for any entry point.
"""

from __future__ import annotations

import ctypes as C
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "_build" / "libjunqi_amd.so"

JQ_OK = 0
JQ_E_ARG, JQ_E_STATE, JQ_E_HIP, JQ_E_OOM, JQ_E_CAPACITY = -1, -2, -3, -4, -5
SAMPLE_UNIFORM, SAMPLE_LOGITS = 0, 1
OBS_F32, OBS_BF16, OBS_U8 = 0, 1, 2
ACT_WORLD, ACT_CANONICAL = 0, 1
F32, BF16 = 0, 1
ATTENTION_MAX_DIM = 128
ROTARY_MAX_AXES = 4
ROTARY_MAX_PAIRS = 4096
SCAN_MAX_STATES = 64
CONV_MAX_TAPS = 8
SCAN_MAX_PLY_STRIDE = 1 << 28
MASK_WORDS_PACKED, MASK_BYTES = 0, 1
MOST_CHANNELS, MOST_PLIES, MOST_GAMES = 1 << 20, 1 << 30, 1 << 30
NUM_CELLS = 289
NUM_ON_BOARD = 129
NUM_PIDS = 120
ACTION_DIM = 16641
MASK_WORDS = 521
OBS_CHANNELS = 317
OBS_GLOBALS = 28
AUX_BYTES = 2320   # u8 aux row: float32[2] turn history + uint16[4][289] recency codes
MAX_LEGAL = 3200
SLOTS_PER_PIECE = 80
SETUP_CANONICAL, SETUP_MIXED = 1, 2
NOALLOC_MAX_ROWS = 1024
AUX_CHANNELS = (64, 65, 253, 254, 255, 256)

FIELDS = {
    "cell": 0, "ptype": 1, "pos": 2, "zero": 3, "move_count": 4, "active_eat": 5, "passive_surv": 6,
    "death_reason": 7, "death_step": 8, "death_loc": 9, "belief": 10, "remaining": 11, "rem_tracked": 12,
    "cm_direct_lo": 13, "cm_direct_hi": 14, "cm_direct_type": 15, "cm_last_direct": 16,
    "cm_other_count": 17, "cm_chain_lo": 18, "cm_chain_hi": 19, "cm_chain_type": 20,
    "cm_last_chain": 21, "cm_eaten_lo": 22, "cm_eaten_hi": 23, "cm_floor": 24, "cm_floor_step": 25,
    "cm_flags": 26, "hist": 27, "hist_meta": 28, "turn": 29, "terminated": 30, "winner": 31,
    "draw": 32, "seat_dead": 33, "flag_rev": 34, "move_counter": 35, "mslc": 36, "zobrist": 37,
}

_EXPORTS = [
    "jq_last_error", "jq_version", "jq_create", "jq_destroy", "jq_num_envs", "jq_upload_zobrist",
    "jq_upload_recency", "jq_upload_setup_pool", "jq_reset_lineups", "jq_reset_seeded",
    "jq_generate_lineups", "jq_generate_pool", "jq_generate_styled", "jq_board_tables", "jq_move_tables", "jq_reset_terminated", "jq_step",
    "jq_legal", "jq_legal_slots", "jq_observe", "jq_obs_timing", "jq_obs_timing_read", "jq_obs_decode_table",
    "jq_sample_uniform", "jq_sample_logits",
    "jq_env_step", "jq_field_info", "jq_get_field", "jq_set_field", "jq_field_ptr", "jq_finalize_import",
    "jq_finalize_import_masked", "jq_rehash", "jq_validate_lineup",
    "jq_sync", "jq_step_host", "jq_legal_dense_host", "jq_env_flags_host", "jq_history_create", "jq_history_destroy", "jq_history_bytes", "jq_history_snapshot",
    "jq_history_reconstruct", "jq_history_reconstruct_bf16", "jq_history_reconstruct_noalloc", "jq_mask_count", "jq_mask_to_ids", "jq_mask_encode", "jq_ids_to_mask", "jq_upload_beliefs",
    "jq_clear_beliefs", "jq_attention_workspace", "jq_attention_forward", "jq_attention_backward", "jq_attention_step",
    "jq_rotary", "jq_layer_norm_forward", "jq_layer_norm_workspace", "jq_layer_norm_backward",
    "jq_scan_workspace", "jq_scan_saved", "jq_scan_forward", "jq_scan_backward", "jq_scan_step", "jq_conv_workspace",
    "jq_conv_forward", "jq_conv_backward", "jq_conv_step", "jq_logits_forward", "jq_logits_workspace", "jq_logits_backward",
]


class Rows(C.Structure):
    """jq_rows: a (batch, plies, heads, dim) tensor, strides in elements."""
    _fields_ = [("data", C.c_void_p), ("batch", C.c_int64), ("ply", C.c_int64), ("head", C.c_int64)]


class Attention(C.Structure):
    """jq_attention."""
    _fields_ = [("dtype", C.c_int32), ("batch", C.c_int32), ("plies", C.c_int32), ("heads", C.c_int32),
                ("key_dim", C.c_int32), ("value_dim", C.c_int32), ("scale", C.c_float), ("log_decay", C.c_void_p),
                ("starts", C.c_void_p), ("starts_batch", C.c_int64), ("starts_ply", C.c_int64),
                ("lengths", C.c_void_p), ("initial_state", C.c_void_p), ("final_state", C.c_void_p),
                ("q", Rows), ("k", Rows), ("v", Rows), ("out", Rows),
                ("d_out", Rows), ("dq", Rows), ("dk", Rows), ("dv", Rows),
                ("d_final", C.c_void_p), ("d_initial", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_int64)]


class Scan(C.Structure):
    """jq_scan."""
    _fields_ = [("dtype", C.c_int32), ("batch", C.c_int32), ("plies", C.c_int32), ("channels", C.c_int32),
                ("states", C.c_int32), ("groups", C.c_int32), ("softplus", C.c_int32), ("a", C.c_void_p),
                ("skip", C.c_void_p), ("delta_bias", C.c_void_p), ("starts", C.c_void_p), ("starts_batch", C.c_int64),
                ("starts_ply", C.c_int64), ("lengths", C.c_void_p), ("initial_state", C.c_void_p),
                ("final_state", C.c_void_p), ("u", Rows), ("delta", Rows), ("gate", Rows), ("out", Rows), ("b", Rows),
                ("c", Rows), ("saved", C.c_void_p), ("d_out", Rows), ("du", Rows), ("ddelta", Rows), ("dgate", Rows),
                ("db", Rows), ("dc", Rows), ("da", C.c_void_p), ("dskip", C.c_void_p), ("ddelta_bias", C.c_void_p),
                ("d_final", C.c_void_p), ("d_initial", C.c_void_p), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_int64)]


class Conv(C.Structure):
    """jq_conv."""
    _fields_ = [("dtype", C.c_int32), ("weight_dtype", C.c_int32), ("batch", C.c_int32), ("plies", C.c_int32),
                ("channels", C.c_int32), ("taps", C.c_int32), ("silu", C.c_int32), ("weight", C.c_void_p),
                ("bias", C.c_void_p), ("starts", C.c_void_p), ("starts_batch", C.c_int64), ("starts_ply", C.c_int64),
                ("lengths", C.c_void_p), ("initial_state", C.c_void_p), ("final_state", C.c_void_p), ("x", Rows),
                ("out", Rows), ("d_out", Rows), ("dx", Rows), ("dweight", C.c_void_p), ("dbias", C.c_void_p),
                ("d_final", C.c_void_p), ("d_initial", C.c_void_p), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_int64)]


class Logits(C.Structure):
    """jq_logits."""
    _fields_ = [("dtype", C.c_int32), ("mask_kind", C.c_int32), ("rows", C.c_int64), ("actions", C.c_int32),
                ("recent_count", C.c_int32), ("recent64", C.c_int32), ("logits", C.c_void_p),
                ("logits_stride", C.c_int64), ("bias", C.c_void_p), ("mask", C.c_void_p), ("mask_stride", C.c_int64),
                ("recent", C.c_void_p), ("recent_stride", C.c_int64), ("recent_lengths", C.c_void_p),
                ("repetition", C.c_float), ("frequency", C.c_float), ("presence", C.c_float),
                ("repetitions", C.c_void_p), ("frequencies", C.c_void_p), ("presences", C.c_void_p)]


class JunqiError(RuntimeError):
    """A C-ABI call returned an error code."""


class ArgumentError(JunqiError, ValueError):
    """A call was given a bad argument (JQ_E_ARG): also a ValueError, which the
    reference raises for invalid setups and seats."""


class CapacityError(JunqiError):
    """An output buffer was smaller than the result (JQ_E_CAPACITY)."""


def _load() -> C.CDLL:
    if not LIB_PATH.exists():
        raise ImportError(
            f"junqi_amd HIP library not built: {LIB_PATH} is missing "
            "(run `python junqi_amd/build.py` or __graft_entry__.build())")
    return bind(C.CDLL(str(LIB_PATH)))


def bind(L: C.CDLL) -> C.CDLL:
    """Declare the C-ABI signatures of include/junqi_amd.h on a loaded library."""
    P, I32, I64, U64 = C.c_void_p, C.c_int32, C.c_int64, C.c_uint64
    F32T, R = C.c_float, C.POINTER(Rows)
    sig = {
        "jq_last_error": ([], C.c_char_p), "jq_version": ([], C.c_char_p),
        "jq_create": ([C.POINTER(P), I32, I32, I32, I32], C.c_int),
        "jq_destroy": ([P], C.c_int), "jq_num_envs": ([P], I32),
        "jq_upload_zobrist": ([P, P, I64], C.c_int), "jq_upload_recency": ([P, P], C.c_int),
        "jq_upload_setup_pool": ([P, P, I32], C.c_int), "jq_reset_lineups": ([P, P, P], C.c_int),
        "jq_reset_seeded": ([P, I64, P], C.c_int), "jq_generate_lineups": ([I64, I32, P], C.c_int),
        "jq_generate_pool": ([I64, I32, P], C.c_int),
        "jq_generate_styled": ([I32, I64, I32, I32, C.c_char_p, I32, P], C.c_int), "jq_board_tables": ([P, I64], C.c_int),
        "jq_move_tables": ([P, I64], C.c_int),
        "jq_reset_terminated": ([P, I64, P], C.c_int),
        "jq_step": ([P, P, P, I32, P, P, P, P, P, P, P, P, P, P], C.c_int),
        "jq_legal": ([P, P, P, P, P, I64, P, P, P], C.c_int),
        "jq_legal_slots": ([P, P, P, P], C.c_int),
        "jq_observe": ([P, P, I32, I32, P, P, P, P], C.c_int),
        "jq_obs_decode_table": ([P], C.c_int),
        "jq_obs_timing": ([P, I32], C.c_int),
        "jq_obs_timing_read": ([P, C.POINTER(C.c_double), C.POINTER(I64)], C.c_int),
        "jq_sample_uniform": ([P, P, P, P, I64, U64, U64, P, P], C.c_int),
        "jq_sample_logits": ([P, P, P, P, P, I64, U64, U64, P, P, P], C.c_int),
        "jq_env_step": ([P, P, I32, U64, U64, I64, P, P, P, I64, P, I32, P, P, P, P, P, P, P, P], C.c_int),
        "jq_validate_lineup": ([P], C.c_int),
        "jq_field_info": ([I32, C.POINTER(I32), C.POINTER(I32)], C.c_int),
        "jq_get_field": ([P, I32, P], C.c_int), "jq_set_field": ([P, I32, P], C.c_int),
        "jq_field_ptr": ([P, I32, C.POINTER(P), C.POINTER(I64), C.POINTER(I64)], C.c_int),
        "jq_finalize_import": ([P, P], C.c_int), "jq_finalize_import_masked": ([P, P, P], C.c_int),
        "jq_rehash": ([P, P], C.c_int),
        "jq_sync": ([P], C.c_int),
        "jq_step_host": ([P, P, P, P, P, P, P, P, P], C.c_int),
        "jq_legal_dense_host": ([P, P, P, P, P, I64, I32, P, P, P], C.c_int),
        "jq_env_flags_host": ([P, P, P, P, P], C.c_int),
        "jq_history_create": ([C.POINTER(P), I32, I32, I32, I32], C.c_int),
        "jq_history_destroy": ([P], C.c_int), "jq_history_bytes": ([P, C.POINTER(I64)], C.c_int),
        "jq_history_snapshot": ([P, P, P, I32, P], C.c_int),
        "jq_history_reconstruct": ([P, P, P, I32, I32, P, P, P, P, P, P], C.c_int),
        "jq_history_reconstruct_bf16": ([P, P, P, I32, P, P, P, P, P], C.c_int),
        "jq_history_reconstruct_noalloc": ([P, P, P, I32, I32, P, P, P, P, P, P], C.c_int),
        "jq_mask_count": ([P, I32, I32, P, P], C.c_int), "jq_mask_to_ids": ([P, I32, I32, I32, P, P], C.c_int),
        "jq_mask_encode": ([P, I32, I32, I32, P, P, P, P, P, P], C.c_int),
        "jq_ids_to_mask": ([P, P, I64, I32, P, I32, I32, P, P], C.c_int),
        "jq_upload_beliefs": ([P, P, I32, P], C.c_int), "jq_clear_beliefs": ([P], C.c_int),
        "jq_attention_workspace": ([C.POINTER(Attention), I32, C.POINTER(I64)], C.c_int),
        "jq_attention_forward": ([C.POINTER(Attention), P], C.c_int),
        "jq_attention_backward": ([C.POINTER(Attention), P], C.c_int),
        "jq_attention_step": ([I32, I32, I32, I32, I32, F32T, P, R, R, R, R, P, I64, P, P, P], C.c_int),
        "jq_rotary": ([I32, I64, I64, I32, I32, I32, R, R, P, I32, I64, I64, I32, C.POINTER(I32), P, I32, I32, P], C.c_int),
        "jq_layer_norm_forward": ([I32, I32, I64, I32, P, I64, P, P, F32T, P, I64, P, P, P], C.c_int),
        "jq_layer_norm_workspace": ([I64, I32, C.POINTER(I64)], C.c_int),
        "jq_layer_norm_backward": ([I32, I32, I64, I32, P, I64, P, P, P, P, I64, P, I64, P, P, P, I64, P], C.c_int),
    }
    S, V, G = C.POINTER(Scan), C.POINTER(Conv), C.POINTER(Logits)
    sig.update({
        "jq_scan_workspace": ([S, I32, C.POINTER(I64)], C.c_int), "jq_scan_saved": ([S, C.POINTER(I64)], C.c_int),
        "jq_scan_forward": ([S, P], C.c_int), "jq_scan_backward": ([S, P], C.c_int),
        "jq_scan_step": ([S, P, I64, P, P, P], C.c_int),
        "jq_conv_workspace": ([V, C.POINTER(I64)], C.c_int), "jq_conv_forward": ([V, P], C.c_int),
        "jq_conv_backward": ([V, P], C.c_int), "jq_conv_step": ([V, P, I64, P, P, P], C.c_int),
        "jq_logits_forward": ([G, P, I64, P], C.c_int), "jq_logits_workspace": ([G, C.POINTER(I64)], C.c_int),
        "jq_logits_backward": ([G, P, I64, P, I64, P, P, I64, P], C.c_int),
    })
    for name, (args, res) in sig.items():
        fn = getattr(L, name)
        fn.argtypes = args
        fn.restype = res
    return L


lib = _load()


def check(rc: int) -> None:
    """Raise for a failed call: ArgumentError (a ValueError) for bad arguments,
    CapacityError for a too small output buffer, JunqiError otherwise."""
    if rc != JQ_OK:
        msg = f"junqi_amd error {rc}: {lib.jq_last_error().decode()}"
        if rc == JQ_E_ARG:
            raise ArgumentError(msg)
        if rc == JQ_E_CAPACITY:
            raise CapacityError(msg)
        raise JunqiError(msg)


def exported_symbols() -> list[str]:
    return list(_EXPORTS)


def field_info(name: str) -> tuple[int, int]:
    e, b = C.c_int32(), C.c_int32()
    check(lib.jq_field_info(FIELDS[name], C.byref(e), C.byref(b)))
    return e.value, b.value
