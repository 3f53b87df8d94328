"""ctypes binding of the C ABI declared in ``include/ai_attn.h``.

The shared library ``_ai_attn.so`` is built in-tree by
``autoindexer_b200.build`` (``nvcc -gencode arch=compute_100a,code=sm_100a``).
There is no fallback: if the library is missing or cannot be loaded every
attention call raises.
"""

from __future__ import annotations

import ctypes
import os
import threading

__all__ = [
    "LIB_PATH",
    "AiTensor4",
    "AiAttnLayout",
    "AiAttnFwdArgs",
    "AiAttnBwdArgs",
    "AiAttnDecodeArgs",
    "DTYPE_BF16",
    "DTYPE_F16",
    "DTYPE_F32",
    "EXPORTED_SYMBOLS",
    "lib",
    "check",
]

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_ai_attn.so")

DTYPE_BF16, DTYPE_F16, DTYPE_F32 = 0, 1, 2
# AiProfKind, in order: those that ai_attn_profile_read writes, and all.
PROF_KINDS = ("prerot", "fwd", "fwd_fill", "delta", "dq", "dkdv", "bwd_fill", "simt", "decode")
ALL_PROF_KINDS = PROF_KINDS + ("head_norm", "append", "prefix", "verify", "score", "distill", "paged4", "attn4")
ABI_VERSION = 9
BWD_DQ, BWD_DKDV = 1, 2
TAILS = {"bucket": 0, "renormalize": 1}  # AiTail
MAX_TOP = 128  # AI_SCORE_MAX_TOP, AI_DISTILL_MAX_TOP
MAX_ROW_BYTES = 3145728  # AI_DISTILL_MAX_ROW_BYTES

# Every function include/ai_attn.h declares.
EXPORTED_SYMBOLS = (
    "ai_attn_abi_version",
    "ai_attn_fwd_tile_rows",
    "ai_attn_kv_tile_rows",
    "ai_attn_fwd",
    "ai_attn_fwd_workspace",
    "ai_attn_bwd_workspace",
    "ai_attn_bwd",
    "ai_attn_bwd_noalloc",
    "ai_attn_decode_workspace",
    "ai_attn_decode",
    "ai_attn_profile_enable",
    "ai_attn_profile_read",
    "ai_attn_profile_read_all",
    "ai_attn_read_status",
    "ai_attn_selftest_wait",
    "ai_attn_strerror",
    "ai_attn_positions_from_ops_sizes",
    "ai_attn_positions_from_ops",
    "ai_attn_prep_sizes",
    "ai_attn_prep",
    "ai_index_fwd",
    "ai_index_bwd",
    "ai_index_rows_sizes",
    "ai_index_rows",
    "ai_head_norm_fwd",
    "ai_head_norm_bwd_workspace",
    "ai_head_norm_bwd",
    "ai_paged_append",
    "ai_prefix_attn_workspace",
    "ai_prefix_attn",
    "ai_verify_draft_workspace",
    "ai_verify_draft",
    "ai_token_logprobs",
    "ai_token_logprobs_bwd",
    "ai_distill",
    "ai_distill_bwd",
    "ai_paged_append_4bit",
    "ai_paged_read_4bit",
    "ai_paged_attn_4bit_workspace",
    "ai_paged_attn_4bit",
)

_i32p = ctypes.POINTER(ctypes.c_int32)
_f32p = ctypes.POINTER(ctypes.c_float)


class AiTensor4(ctypes.Structure):
    _fields_ = [
        ("ptr", ctypes.c_void_p),
        ("stride_b", ctypes.c_int64),
        ("stride_h", ctypes.c_int64),
        ("stride_t", ctypes.c_int64),
    ]


class AiAttnLayout(ctypes.Structure):
    _fields_ = [
        ("n_blocks", ctypes.c_int32),
        ("blocks", ctypes.c_void_p),
        ("row_blocks", ctypes.c_void_p),
        ("row_cov", ctypes.c_void_p),
        ("key_info", ctypes.c_void_p),
        ("n_keys", ctypes.c_int64),
        ("q_pos", ctypes.c_void_p),
        ("k_own", ctypes.c_void_p),
        ("rope_cos", ctypes.c_void_p),
        ("rope_sin", ctypes.c_void_p),
        ("rope_cs16", ctypes.c_void_p),
        ("n_pos", ctypes.c_int32),
        ("fwd_tile", ctypes.c_int32),
        ("fwd_items", ctypes.c_void_p),
        ("n_fwd_items", ctypes.c_int32),
        ("n_fwd_abs_items", ctypes.c_int32),
        ("kv_tile", ctypes.c_int32),
        ("kv_items", ctypes.c_void_p),
        ("n_kv_items", ctypes.c_int32),
        ("n_kv_abs_items", ctypes.c_int32),
        ("all_rows_owned", ctypes.c_int32),
        ("n_fwd_short_items", ctypes.c_int32),
        ("kv_chunks", ctypes.c_void_p),
        ("n_kv_chunks", ctypes.c_int32),
        ("n_kv_partials", ctypes.c_int32),
        ("kv_reduce", ctypes.c_void_p),
        ("n_kv_reduce", ctypes.c_int32),
        ("kv_cost_max", ctypes.c_int32),
        ("kv_cost_total", ctypes.c_int32),
        ("blk_cls", ctypes.c_void_p),
        ("chunk_cls", ctypes.c_void_p),
        ("n_chunk_cls", ctypes.c_int32),
        ("rot_classes", ctypes.c_void_p),
        ("n_rot_classes", ctypes.c_int32),
        ("n_fwd_abs_short_items", ctypes.c_int32),
    ]


class AiAttnFwdArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("q", AiTensor4),
        ("k", AiTensor4),
        ("v", AiTensor4),
        ("out", AiTensor4),
        ("lse", ctypes.c_void_p),
        ("layout", AiAttnLayout),
        ("status", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class AiAttnBwdArgs(ctypes.Structure):
    _fields_ = [
        ("fwd", AiAttnFwdArgs),
        ("dout", AiTensor4),
        ("dq", AiTensor4),
        ("dk", AiTensor4),
        ("dv", AiTensor4),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("fwd_rotated", ctypes.c_int32),
        ("parts", ctypes.c_int32),
    ]


class AiAttnDecodeArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("kv_len", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("q", AiTensor4),
        ("k", AiTensor4),
        ("v", AiTensor4),
        ("out", AiTensor4),
        ("key_rows", ctypes.c_void_p),
        ("key_rows_stride_b", ctypes.c_int64),
        ("key_ok", ctypes.c_void_p),
        ("key_ok_stride_b", ctypes.c_int64),
        ("rope_cs16", ctypes.c_void_p),
        ("n_pos", ctypes.c_int32),
        ("status", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class AiIndexArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("q", AiTensor4),
        ("k", AiTensor4),
        ("n_rows", ctypes.c_int32),
        ("rows", ctypes.c_void_p),
        ("targets", ctypes.c_void_p),
        ("n_keys", ctypes.c_int64),
        ("key_rows", ctypes.c_void_p),
        ("key_ok", ctypes.c_void_p),
        ("rope_cos", ctypes.c_void_p),
        ("rope_sin", ctypes.c_void_p),
        ("n_pos", ctypes.c_int32),
        ("logits", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
        ("loss", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
    ]


class AiIndexBwdArgs(ctypes.Structure):
    _fields_ = [
        ("fwd", AiIndexArgs),
        ("dloss", ctypes.c_void_p),
        ("dq", AiTensor4),
        ("dk", AiTensor4),
    ]


class AiPrepList(ctypes.Structure):
    _fields_ = [
        ("n_blocks", ctypes.c_int32),
        ("boundary", ctypes.c_void_p),
        ("n_query", ctypes.c_int64),
        ("query_pos", ctypes.c_void_p),
        ("n_keys", ctypes.c_int64),
        ("key_pos", ctypes.c_void_p),
        ("attn_mask", ctypes.c_void_p),
        ("abs_mask", ctypes.c_void_p),
    ]


class AiIndexRowsOut(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_void_p),
        ("key_rows", ctypes.c_void_p),
        ("key_ok", ctypes.c_void_p),
        ("rel_lo", ctypes.c_int64),
        ("rel_hi", ctypes.c_int64),
    ]


class AiPrepSizes(ctypes.Structure):
    _fields_ = [
        ("n_blocks", ctypes.c_int32),
        ("n_fwd_items", ctypes.c_int32),
        ("n_kv_items", ctypes.c_int32),
        ("n_kv_chunks", ctypes.c_int32),
        ("n_kv_reduce", ctypes.c_int32),
        ("n_chunk_cls", ctypes.c_int32),
        ("n_rot_classes", ctypes.c_int32),
        ("n_keys", ctypes.c_int64),
        ("p_min", ctypes.c_int64),
        ("p_max", ctypes.c_int64),
    ]


class AiPrepTables(ctypes.Structure):
    _fields_ = [
        ("blocks", ctypes.c_void_p),
        ("row_blocks", ctypes.c_void_p),
        ("row_cov", ctypes.c_void_p),
        ("key_info", ctypes.c_void_p),
        ("q_pos", ctypes.c_void_p),
        ("k_own", ctypes.c_void_p),
        ("fwd_items", ctypes.c_void_p),
        ("kv_items", ctypes.c_void_p),
        ("kv_chunks", ctypes.c_void_p),
        ("kv_reduce", ctypes.c_void_p),
        ("blk_cls", ctypes.c_void_p),
        ("chunk_cls", ctypes.c_void_p),
        ("rot_classes", ctypes.c_void_p),
        ("n_kv_partials", ctypes.c_int32),
        ("kv_cost_max", ctypes.c_int32),
        ("kv_cost_total", ctypes.c_int32),
        ("n_fwd_abs_items", ctypes.c_int32),
        ("n_fwd_short_items", ctypes.c_int32),
        ("n_fwd_abs_short_items", ctypes.c_int32),
        ("n_kv_abs_items", ctypes.c_int32),
        ("all_rows_owned", ctypes.c_int32),
        ("pairs_per_head", ctypes.c_int64),
    ]


class AiPositions(ctypes.Structure):
    _fields_ = [
        ("ptr", ctypes.c_void_p),
        ("stride_b", ctypes.c_int64),
        ("is_int64", ctypes.c_int32),
    ]


class AiHeadNormArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("weight_dtype", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("q", AiTensor4),
        ("k", AiTensor4),
        ("q_out", AiTensor4),
        ("k_out", AiTensor4),
        ("q_weight", ctypes.c_void_p),
        ("k_weight", ctypes.c_void_p),
        ("rope_cos", ctypes.c_void_p),
        ("rope_sin", ctypes.c_void_p),
        ("n_pos", ctypes.c_int32),
        ("pos", AiPositions),
        ("status", ctypes.c_void_p),
    ]


class AiHeadNormBwdArgs(ctypes.Structure):
    _fields_ = [
        ("fwd", AiHeadNormArgs),
        ("dq_out", AiTensor4),
        ("dk_out", AiTensor4),
        ("dq", AiTensor4),
        ("dk", AiTensor4),
        ("dq_weight", ctypes.c_void_p),
        ("dk_weight", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class AiPagedAppendArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("weight_dtype", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("k", AiTensor4),
        ("v", AiTensor4),
        ("k_pages", AiTensor4),
        ("v_pages", AiTensor4),
        ("n_pages", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("page_table", ctypes.c_void_p),
        ("page_table_stride", ctypes.c_int64),
        ("max_pages", ctypes.c_int32),
        ("lens", ctypes.c_void_p),
        ("new_lens", ctypes.c_void_p),
        ("k_weight", ctypes.c_void_p),
        ("rope_cos", ctypes.c_void_p),
        ("rope_sin", ctypes.c_void_p),
        ("n_pos", ctypes.c_int32),
        ("pos", AiPositions),
        ("status", ctypes.c_void_p),
    ]


class AiPrefixAttnArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("q", AiTensor4),
        ("out", AiTensor4),
        ("lse", ctypes.c_void_p),
        ("k_pages", AiTensor4),
        ("v_pages", AiTensor4),
        ("n_pages", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("prefix_pages", ctypes.c_void_p),
        ("prefix_len", ctypes.c_int32),
        ("page_table", ctypes.c_void_p),
        ("page_table_stride", ctypes.c_int64),
        ("max_pages", ctypes.c_int32),
        ("lens", ctypes.c_void_p),
        ("query_lens", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class AiVerifyArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("n_draft", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("target", ctypes.c_void_p),
        ("target_stride_b", ctypes.c_int64),
        ("target_stride_t", ctypes.c_int64),
        ("draft", ctypes.c_void_p),
        ("draft_stride_b", ctypes.c_int64),
        ("draft_stride_t", ctypes.c_int64),
        ("tokens", ctypes.c_void_p),
        ("uniforms", ctypes.c_void_p),
        ("noise", ctypes.c_void_p),
        ("temperature", ctypes.c_void_p),
        ("draft_lens", ctypes.c_void_p),
        ("accepted", ctypes.c_void_p),
        ("out_tokens", ctypes.c_void_p),
        ("logprobs", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class AiScoreArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("logits", ctypes.c_void_p),
        ("stride_b", ctypes.c_int64),
        ("stride_t", ctypes.c_int64),
        ("tokens", ctypes.c_void_p),
        ("temperature", ctypes.c_void_p),
        ("top_k", ctypes.c_int32),
        ("logprobs", ctypes.c_void_p),
        ("entropy", ctypes.c_void_p),
        ("top_logprobs", ctypes.c_void_p),
        ("top_tokens", ctypes.c_void_p),
        ("row_stats", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
    ]


class AiScoreBwdArgs(ctypes.Structure):
    _fields_ = [
        ("fwd", AiScoreArgs),
        ("g_logprobs", ctypes.c_void_p),
        ("g_entropy", ctypes.c_void_p),
        ("g_top", ctypes.c_void_p),
        ("dlogits", ctypes.c_void_p),
        ("dstride_b", ctypes.c_int64),
        ("dstride_t", ctypes.c_int64),
    ]


class AiDistillArgs(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("vocab", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("logits", ctypes.c_void_p),
        ("stride_b", ctypes.c_int64),
        ("stride_t", ctypes.c_int64),
        ("n_top", ctypes.c_int32),
        ("tail", ctypes.c_int32),
        ("top_tokens", ctypes.c_void_p),
        ("top_logprobs", ctypes.c_void_p),
        ("weights", ctypes.c_void_p),
        ("temperature", ctypes.c_void_p),
        ("losses", ctypes.c_void_p),
        ("dlogits", ctypes.c_void_p),
        ("dstride_b", ctypes.c_int64),
        ("dstride_t", ctypes.c_int64),
        ("row_stats", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
    ]


class AiDistillBwdArgs(ctypes.Structure):
    _fields_ = [
        ("fwd", AiDistillArgs),
        ("g_losses", ctypes.c_void_p),
        ("dlogits", ctypes.c_void_p),
        ("dstride_b", ctypes.c_int64),
        ("dstride_t", ctypes.c_int64),
    ]


class AiPool4(ctypes.Structure):
    _fields_ = [
        ("k_codes", AiTensor4),
        ("v_codes", AiTensor4),
        ("k_scales", AiTensor4),
        ("v_scales", AiTensor4),
        ("n_pages", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("page_table", ctypes.c_void_p),
        ("page_table_stride", ctypes.c_int64),
        ("max_pages", ctypes.c_int32),
    ]


class AiPaged4Args(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("k", AiTensor4),
        ("v", AiTensor4),
        ("pool", AiPool4),
        ("lens", ctypes.c_void_p),
        ("n", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
    ]


class AiPagedAttn4Args(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("q", AiTensor4),
        ("out", AiTensor4),
        ("lse", ctypes.c_void_p),
        ("pool", AiPool4),
        ("lens", ctypes.c_void_p),
        ("query_lens", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


_lock = threading.Lock()
_lib = None


def _bind(handle):
    P = ctypes.POINTER
    for name in ("ai_attn_fwd_tile_rows", "ai_attn_kv_tile_rows"):
        fn = getattr(handle, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [ctypes.c_int, ctypes.c_int]
    handle.ai_attn_fwd.restype = ctypes.c_int
    handle.ai_attn_fwd.argtypes = [P(AiAttnFwdArgs), ctypes.c_void_p]
    handle.ai_attn_fwd_workspace.restype = ctypes.c_int
    handle.ai_attn_fwd_workspace.argtypes = [P(AiAttnFwdArgs), P(ctypes.c_size_t)]
    handle.ai_attn_bwd_workspace.restype = ctypes.c_int
    handle.ai_attn_bwd_workspace.argtypes = [P(AiAttnBwdArgs), P(ctypes.c_size_t)]
    handle.ai_attn_bwd.restype = ctypes.c_int
    handle.ai_attn_bwd.argtypes = [P(AiAttnBwdArgs), ctypes.c_void_p]
    handle.ai_attn_bwd_noalloc.restype = ctypes.c_int
    handle.ai_attn_bwd_noalloc.argtypes = [P(AiAttnBwdArgs), ctypes.c_void_p]
    handle.ai_attn_decode_workspace.restype = ctypes.c_int
    handle.ai_attn_decode_workspace.argtypes = [P(AiAttnDecodeArgs), P(ctypes.c_size_t)]
    handle.ai_attn_decode.restype = ctypes.c_int
    handle.ai_attn_decode.argtypes = [P(AiAttnDecodeArgs), ctypes.c_void_p]
    handle.ai_attn_read_status.restype = ctypes.c_int
    handle.ai_attn_read_status.argtypes = [ctypes.c_void_p, ctypes.c_void_p, P(ctypes.c_int32)]
    handle.ai_attn_strerror.restype = ctypes.c_char_p
    handle.ai_attn_strerror.argtypes = [ctypes.c_int]
    handle.ai_attn_profile_enable.restype = ctypes.c_int
    handle.ai_attn_profile_enable.argtypes = [ctypes.c_int]
    handle.ai_attn_profile_read.restype = ctypes.c_int
    handle.ai_attn_profile_read.argtypes = [P(ctypes.c_float), P(ctypes.c_int32)]
    handle.ai_attn_profile_read_all.restype = ctypes.c_int
    handle.ai_attn_profile_read_all.argtypes = [P(ctypes.c_float), P(ctypes.c_int32), ctypes.c_int32]
    handle.ai_attn_selftest_wait.restype = ctypes.c_int
    handle.ai_attn_selftest_wait.argtypes = [ctypes.c_void_p, ctypes.c_longlong, ctypes.c_void_p]
    vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
    handle.ai_attn_positions_from_ops_sizes.restype = ctypes.c_int
    handle.ai_attn_positions_from_ops_sizes.argtypes = [vp, i32, P(i32), P(i64), P(i64)]
    handle.ai_attn_positions_from_ops.restype = ctypes.c_int
    handle.ai_attn_positions_from_ops.argtypes = [vp, i32, vp, vp, vp, vp, vp, vp]
    handle.ai_attn_prep_sizes.restype = ctypes.c_int
    handle.ai_attn_prep_sizes.argtypes = [P(AiPrepList), i32, vp, i32, i32, i32, i32, P(AiPrepSizes)]
    handle.ai_attn_prep.restype = ctypes.c_int
    handle.ai_attn_prep.argtypes = [P(AiPrepList), i32, vp, i32, i32, i32, i32, P(AiPrepTables)]
    handle.ai_index_fwd.restype = ctypes.c_int
    handle.ai_index_fwd.argtypes = [P(AiIndexArgs), vp]
    handle.ai_index_bwd.restype = ctypes.c_int
    handle.ai_index_bwd.argtypes = [P(AiIndexBwdArgs), vp]
    handle.ai_index_rows_sizes.restype = ctypes.c_int
    handle.ai_index_rows_sizes.argtypes = [P(AiPrepList), vp, P(i32), P(i64), vp]
    handle.ai_index_rows.restype = ctypes.c_int
    handle.ai_index_rows.argtypes = [P(AiPrepList), vp, i64, P(AiIndexRowsOut)]
    for name, args in (("ai_head_norm_fwd", AiHeadNormArgs), ("ai_head_norm_bwd", AiHeadNormBwdArgs),
                       ("ai_paged_append", AiPagedAppendArgs), ("ai_prefix_attn", AiPrefixAttnArgs),
                       ("ai_verify_draft", AiVerifyArgs), ("ai_token_logprobs", AiScoreArgs),
                       ("ai_token_logprobs_bwd", AiScoreBwdArgs), ("ai_distill", AiDistillArgs),
                       ("ai_distill_bwd", AiDistillBwdArgs),
                       ("ai_paged_append_4bit", AiPaged4Args), ("ai_paged_read_4bit", AiPaged4Args),
                       ("ai_paged_attn_4bit", AiPagedAttn4Args)):
        fn = getattr(handle, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [P(args), vp]
    for name, args in (("ai_head_norm_bwd_workspace", AiHeadNormBwdArgs),
                       ("ai_prefix_attn_workspace", AiPrefixAttnArgs),
                       ("ai_verify_draft_workspace", AiVerifyArgs),
                       ("ai_paged_attn_4bit_workspace", AiPagedAttn4Args)):
        fn = getattr(handle, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [P(args), P(ctypes.c_size_t)]
    return handle


def lib():
    """The loaded C library (loaded once).  Raises if it is missing."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                if not os.path.exists(LIB_PATH):
                    raise RuntimeError(
                        f"autoindexer_b200: CUDA library {LIB_PATH} is not built; "
                        "run `python -m autoindexer_b200.build` (nvcc, sm_100a)")
                handle = ctypes.CDLL(LIB_PATH)
                handle.ai_attn_abi_version.restype = ctypes.c_int
                handle.ai_attn_abi_version.argtypes = []
                ver = handle.ai_attn_abi_version()
                if ver != ABI_VERSION:
                    raise RuntimeError(f"autoindexer_b200: library ABI {ver} != expected {ABI_VERSION}; rebuild it")
                try:
                    _lib = _bind(handle)
                except AttributeError as e:  # (functions are added within an ABI)
                    raise RuntimeError(f"autoindexer_b200: the library lacks a function ({e}); rebuild it") from e
    return _lib


def strerror(code: int) -> str:
    return lib().ai_attn_strerror(int(code)).decode()


def check(code: int, what: str) -> None:
    if code != 0:
        raise RuntimeError(f"{what} failed ({code}): {strerror(code)}")
