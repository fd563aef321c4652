"""ctypes binding of libnemo.so (the C ABI declared in include/nemo.h).

The library is loaded from the package directory (next to ``csrc/``). There
is no fallback: if it is missing or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes
import os

PACKAGE_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(PACKAGE_DIR, "libnemo.so")

NEMO_OK = 0
STATUS_NAMES = {1: "invalid", 2: "missing", 3: "device", 4: "out of memory", 5: "unsupported"}

TYPE_F32, TYPE_F16, TYPE_Q4_0, TYPE_Q4_K, TYPE_Q6_K = 0, 1, 2, 12, 14
TYPE_Q4_0_TILE32 = 258  # wgpack q4_0-tile32-compact records (include/nemo.h)
TYPE_I8, TYPE_BF16, TYPE_F8_E4M3 = 24, 30, 259
ROPE_INTERLEAVED, ROPE_HALF = 0, 1
ROPE_NONE, ROPE_LINEAR, ROPE_YARN, ROPE_BANDS = 0, 1, 2, 3
MATMUL_AUTO, MATMUL_GEMM, MATMUL_GEMV, MATMUL_TWO_PASS, MATMUL_GEMM_MID, MATMUL_GEMM_SPLIT = 0, 1, 2, 3, 4, 5
STATIC_SCRATCH_BYTES = 64 << 20  # NEMO_STATIC_SCRATCH_BYTES

# Every symbol include/nemo.h declares.
EXPORTED = [
    "nemo_dims_reference", "nemo_last_error", "nemo_version", "nemo_debug_fail_after", "nemo_init", "nemo_shutdown",
    "nemo_model_create", "nemo_model_set_tensor", "nemo_model_synthesize", "nemo_model_finalize",
    "nemo_model_get_tensor", "nemo_model_destroy", "nemo_plan_create", "nemo_plan_run", "nemo_plan_run_device",
    "nemo_plan_profile", "nemo_profile_stage_count", "nemo_profile_stage_name", "nemo_plan_destroy",
    "nemo_plan_shape", "nemo_plan_read_buffer",
    "nemo_weight_create", "nemo_weight_destroy", "nemo_weight_matmul", "nemo_weight_matmul_static",
    "nemo_weight_dequantize", "nemo_dequantize",
    "nemo_requantize_q40", "nemo_probe_stream",
    "nemo_rope_config_default", "nemo_rope_create", "nemo_rope_destroy", "nemo_rope_apply",
    "nemo_window_attention_workspace", "nemo_window_attention", "nemo_rmsnorm", "nemo_model_set_attention",
    "nemo_plan_token_states8",
    "nemo_rope_norm_apply", "nemo_matmul8", "nemo_cache4_page_bytes", "nemo_cache4_append", "nemo_cache4_read",
    "nemo_cache4_attention_workspace", "nemo_cache4_attention",
]


class NemoError(RuntimeError):
    """A libnemo call failed; ``status`` is the nemo_status code."""

    def __init__(self, status: int, message: str):
        super().__init__(message)
        self.status = status


class Dims(ctypes.Structure):
    """nemo_dims (include/nemo.h)."""
    _fields_ = [
        ("hidden", ctypes.c_int32), ("q_heads", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32), ("intermediate", ctypes.c_int32), ("layers", ctypes.c_int32),
        ("vocab", ctypes.c_int32), ("merge_after_layer", ctypes.c_int32), ("rms_epsilon", ctypes.c_float),
        ("rope_theta", ctypes.c_float), ("kv_stride_threshold", ctypes.c_int32), ("kv_stride", ctypes.c_int32),
        ("kv_dense_before_merge", ctypes.c_int32),
    ]


class RopeConfig(ctypes.Structure):
    """nemo_rope_config (include/nemo.h)."""
    _fields_ = [
        ("head_dim", ctypes.c_int32), ("rotary_dim", ctypes.c_int32), ("layout", ctypes.c_int32),
        ("scaling", ctypes.c_int32), ("theta", ctypes.c_double), ("factor", ctypes.c_double),
        ("original_positions", ctypes.c_int32), ("beta_fast", ctypes.c_double), ("beta_slow", ctypes.c_double),
        ("low_band", ctypes.c_double), ("high_band", ctypes.c_double), ("magnitude", ctypes.c_double),
    ]


class RopeHeads(ctypes.Structure):
    """nemo_rope_heads (include/nemo.h)."""
    _fields_ = [
        ("x", ctypes.c_void_p), ("y", ctypes.c_void_p), ("x_row", ctypes.c_int64), ("x_head", ctypes.c_int64),
        ("y_row", ctypes.c_int64), ("y_head", ctypes.c_int64), ("heads", ctypes.c_int32),
    ]


class AttentionConfig(ctypes.Structure):
    """nemo_attention_config (include/nemo.h)."""
    _fields_ = [
        ("q_heads", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
        ("type", ctypes.c_int32), ("left", ctypes.c_int32), ("right", ctypes.c_int32), ("sinks", ctypes.c_int32),
        ("scale", ctypes.c_float),
    ]


class AttentionBatch(ctypes.Structure):
    """nemo_attention_batch (include/nemo.h)."""
    _fields_ = [
        ("count", ctypes.c_int32), ("q_rows", ctypes.c_int64), ("kv_rows", ctypes.c_int64),
        ("max_kv", ctypes.c_int64), ("q_start", ctypes.c_void_p), ("kv_start", ctypes.c_void_p),
        ("kv_len", ctypes.c_void_p), ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
        ("out", ctypes.c_void_p), ("q_row", ctypes.c_int64), ("q_head", ctypes.c_int64), ("k_row", ctypes.c_int64),
        ("k_head", ctypes.c_int64), ("v_row", ctypes.c_int64), ("v_head", ctypes.c_int64),
        ("out_row", ctypes.c_int64), ("out_head", ctypes.c_int64), ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class ModelAttention(ctypes.Structure):
    """nemo_model_attention (include/nemo.h)."""
    _fields_ = [
        ("left", ctypes.c_int32), ("right", ctypes.c_int32), ("sinks", ctypes.c_int32),
        ("global_every", ctypes.c_int32), ("rope", RopeConfig),
    ]


class NormArgs(ctypes.Structure):
    """nemo_norm_args (include/nemo.h)."""
    _fields_ = [
        ("type", ctypes.c_int32), ("hidden", ctypes.c_int32), ("rows", ctypes.c_int64), ("x", ctypes.c_void_p),
        ("delta", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("sum", ctypes.c_void_p), ("y", ctypes.c_void_p),
        ("y8", ctypes.c_void_p), ("scales", ctypes.c_void_p), ("x_row", ctypes.c_int64),
        ("delta_row", ctypes.c_int64), ("sum_row", ctypes.c_int64), ("y_row", ctypes.c_int64),
        ("y8_row", ctypes.c_int64), ("scales_row", ctypes.c_int64), ("type8", ctypes.c_int32),
        ("group", ctypes.c_int32), ("epsilon", ctypes.c_float),
    ]


class HeadNorm(ctypes.Structure):
    """nemo_head_norm (include/nemo.h)."""
    _fields_ = [
        ("q_weight", ctypes.c_void_p), ("k_weight", ctypes.c_void_p), ("q_weight_head", ctypes.c_int64),
        ("k_weight_head", ctypes.c_int64), ("epsilon", ctypes.c_float),
    ]


class Matmul8Args(ctypes.Structure):
    """nemo_matmul8_args (include/nemo.h)."""
    _fields_ = [
        ("type", ctypes.c_int32), ("n", ctypes.c_int32), ("k", ctypes.c_int32), ("m", ctypes.c_int64),
        ("x", ctypes.c_void_p), ("x_scale", ctypes.c_void_p), ("w", ctypes.c_void_p), ("w_scale", ctypes.c_void_p),
        ("bias", ctypes.c_void_p), ("y", ctypes.c_void_p), ("x_row", ctypes.c_int64), ("x_scale_row", ctypes.c_int64),
        ("w_row", ctypes.c_int64), ("y_row", ctypes.c_int64),
    ]


class Cache4Config(ctypes.Structure):
    """nemo_cache4_config (include/nemo.h)."""
    _fields_ = [("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("page", ctypes.c_int32)]


class Cache4Pages(ctypes.Structure):
    """nemo_cache4_pages (include/nemo.h)."""
    _fields_ = [
        ("count", ctypes.c_int32), ("pages", ctypes.c_int32), ("data", ctypes.c_void_p), ("table", ctypes.c_void_p),
        ("table_row", ctypes.c_int64), ("kv_len", ctypes.c_void_p),
    ]


class Cache4Rows(ctypes.Structure):
    """nemo_cache4_rows (include/nemo.h)."""
    _fields_ = [
        ("type", ctypes.c_int32), ("rows", ctypes.c_int64), ("q_start", ctypes.c_void_p),
        ("positions", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_row", ctypes.c_int64),
        ("k_head", ctypes.c_int64), ("v_row", ctypes.c_int64), ("v_head", ctypes.c_int64),
    ]


class Cache4Queries(ctypes.Structure):
    """nemo_cache4_queries (include/nemo.h)."""
    _fields_ = [
        ("q_rows", ctypes.c_int64), ("max_kv", ctypes.c_int64), ("q_start", ctypes.c_void_p), ("q", ctypes.c_void_p),
        ("out", ctypes.c_void_p), ("q_row", ctypes.c_int64), ("q_head", ctypes.c_int64), ("out_row", ctypes.c_int64),
        ("out_head", ctypes.c_int64), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
    ]


_lib = None


def load() -> ctypes.CDLL:
    """Load libnemo.so; raise if it was not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"libnemo.so not found at {LIB_PATH}; run __graft_entry__.build() first")
    L = ctypes.CDLL(LIB_PATH)
    vp, sz, i32, u64 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int32, ctypes.c_uint64
    u32p = ctypes.POINTER(ctypes.c_uint32)
    i64p = ctypes.POINTER(ctypes.c_int64)
    f32p = ctypes.POINTER(ctypes.c_float)
    pp = ctypes.POINTER(ctypes.c_void_p)
    sig = {
        "nemo_dims_reference": (None, [ctypes.POINTER(Dims)]),
        "nemo_last_error": (ctypes.c_char_p, []),
        "nemo_version": (ctypes.c_char_p, []),
        "nemo_debug_fail_after": (None, [i32]),
        "nemo_init": (i32, [i32, pp]),
        "nemo_shutdown": (i32, [vp]),
        "nemo_model_create": (i32, [vp, ctypes.POINTER(Dims), pp]),
        "nemo_model_set_tensor": (i32, [vp, ctypes.c_char_p, i32, i64p, i32, vp, sz]),
        "nemo_model_synthesize": (i32, [vp, u64, i32]),
        "nemo_model_finalize": (i32, [vp]),
        "nemo_model_get_tensor": (i32, [vp, ctypes.c_char_p, ctypes.POINTER(i32), i64p, vp, ctypes.POINTER(sz)]),
        "nemo_model_destroy": (i32, [vp]),
        "nemo_plan_create": (i32, [vp, i32, i32, pp]),
        "nemo_plan_run": (i32, [vp, u32p, sz, u32p, sz, f32p]),
        "nemo_plan_run_device": (i32, [vp, vp, u32p, sz, vp, vp]),
        "nemo_plan_profile": (i32, [vp, u32p, sz, u32p, sz, f32p, i32]),
        "nemo_profile_stage_count": (i32, []),
        "nemo_profile_stage_name": (ctypes.c_char_p, [i32]),
        "nemo_plan_destroy": (i32, [vp]),
        "nemo_plan_shape": (i32, [vp, ctypes.POINTER(i32), ctypes.POINTER(i32), ctypes.POINTER(i32)]),
        "nemo_plan_read_buffer": (i32, [vp, ctypes.c_char_p, vp, ctypes.POINTER(sz)]),
        "nemo_weight_create": (i32, [vp, i32, i32, i32, vp, sz, pp]),
        "nemo_weight_destroy": (i32, [vp]),
        "nemo_weight_matmul": (i32, [vp, vp, i32, vp, i32, vp]),
        "nemo_weight_matmul_static": (i32, [vp, vp, i32, vp, i32, vp]),
        "nemo_weight_dequantize": (i32, [vp, vp, vp]),
        "nemo_dequantize": (i32, [i32, vp, ctypes.c_int64, vp, vp, vp]),
        "nemo_requantize_q40": (i32, [vp, i32, vp, sz, ctypes.c_int64, ctypes.c_int64, vp, sz]),
        "nemo_probe_stream": (i32, [vp, sz, i32, vp, vp]),
        "nemo_rope_config_default": (None, [ctypes.POINTER(RopeConfig)]),
        "nemo_rope_create": (i32, [vp, ctypes.POINTER(RopeConfig), pp]),
        "nemo_rope_destroy": (i32, [vp]),
        "nemo_rope_apply": (i32, [vp, i32, ctypes.POINTER(RopeHeads), ctypes.POINTER(RopeHeads), ctypes.c_int64, vp,
                                  ctypes.c_int64, vp]),
        "nemo_window_attention_workspace": (i32, [ctypes.POINTER(AttentionConfig), i32, ctypes.c_int64,
                                                  ctypes.c_int64, ctypes.POINTER(sz)]),
        "nemo_window_attention": (i32, [vp, ctypes.POINTER(AttentionConfig), ctypes.POINTER(AttentionBatch), vp]),
        "nemo_rmsnorm": (i32, [vp, ctypes.POINTER(NormArgs), vp]),
        "nemo_model_set_attention": (i32, [vp, ctypes.POINTER(ModelAttention)]),
        "nemo_plan_token_states8": (i32, [vp, i32, i32, vp, vp, ctypes.c_int64, i64p, vp]),
        "nemo_rope_norm_apply": (i32, [vp, i32, ctypes.POINTER(RopeHeads), ctypes.POINTER(RopeHeads),
                                       ctypes.POINTER(HeadNorm), ctypes.c_int64, vp, ctypes.c_int64, vp]),
        "nemo_matmul8": (i32, [vp, ctypes.POINTER(Matmul8Args), vp]),
        "nemo_cache4_page_bytes": (i32, [ctypes.POINTER(Cache4Config), ctypes.POINTER(sz)]),
        "nemo_cache4_append": (i32, [vp, ctypes.POINTER(Cache4Config), ctypes.POINTER(Cache4Pages),
                                     ctypes.POINTER(Cache4Rows), vp, vp]),
        "nemo_cache4_read": (i32, [vp, ctypes.POINTER(Cache4Config), ctypes.POINTER(Cache4Pages),
                                   ctypes.POINTER(Cache4Rows), vp]),
        "nemo_cache4_attention_workspace": (i32, [ctypes.POINTER(AttentionConfig), i32, ctypes.c_int64,
                                                  ctypes.c_int64, ctypes.POINTER(sz)]),
        "nemo_cache4_attention": (i32, [vp, ctypes.POINTER(Cache4Config), ctypes.POINTER(AttentionConfig),
                                        ctypes.POINTER(Cache4Pages), ctypes.POINTER(Cache4Queries), vp]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def check(status: int) -> None:
    if status != NEMO_OK:
        msg = load().nemo_last_error().decode()
        raise NemoError(status, msg or STATUS_NAMES.get(status, str(status)))
