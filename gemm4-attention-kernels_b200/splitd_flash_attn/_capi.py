"""ctypes binding of libsplitd_attn.so (the C-ABI declared in include/splitd_attn.h).

The library is built in-tree by ``build.py`` (nvcc, sm_100a). There is no fallback: if the
shared object is missing or a call fails, an exception is raised.
"""

from __future__ import annotations

import ctypes
import os
from typing import Optional

_PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(os.path.dirname(_PKG_DIR), "csrc", "libsplitd_attn.so")

SPLITD_DTYPE_BF16 = 0
SPLITD_DTYPE_FP16 = 1

EXPORTED_SYMBOLS = (
    "splitd_device_supported",
    "splitd_fwd",
    "splitd_fwd_workspace_bytes",
    "splitd_bwd_rowstat_elems",
    "splitd_out_resid_bytes",
    "splitd_bwd_workspace_bytes",
    "splitd_bwd_workspace_bytes_limit",
    "splitd_bwd_num_chunks",
    "splitd_bwd_chunk",
    "splitd_wait_probe",
    "splitd_bwd_preprocess",
    "splitd_bwd_dq",
    "splitd_bwd_dkdv",
    "splitd_bwd_tiles",
    "splitd_bwd_grads",
    "splitd_bwd",
    "splitd_bwd_static_scratch",
    "splitd_bwd_static_scratch_limit_rowstat",
    "splitd_bwd_static_scratch_limit_workspace",
    "splitd_paged_attn",
    "splitd_paged_attn_workspace_bytes",
    "splitd_rotary",
    "splitd_paged_append",
    "splitd_paged_evict",
    "splitd_last_error",
    "splitd_version",
)


class SplitdParams(ctypes.Structure):
    """Mirror of ``splitd_params`` (include/splitd_attn.h); field order must match."""

    _fields_ = [
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
        ("dout", ctypes.c_void_p),
        ("dlse", ctypes.c_void_p),
        ("dq", ctypes.c_void_p),
        ("dk", ctypes.c_void_p),
        ("dv", ctypes.c_void_p),
        ("dpsum", ctypes.c_void_p),
        ("lse_log2", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("cu_seqlens_q", ctypes.c_void_p),
        ("cu_seqlens_k", ctypes.c_void_p),
        ("batch", ctypes.c_int32),
        ("seqlen_q", ctypes.c_int32),
        ("seqlen_k", ctypes.c_int32),
        ("total_q", ctypes.c_int32),
        ("total_k", ctypes.c_int32),
        ("max_seqlen_q", ctypes.c_int32),
        ("max_seqlen_k", ctypes.c_int32),
        ("heads_q", ctypes.c_int32),
        ("heads_kv", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("q_strides", ctypes.c_int64 * 3),
        ("k_strides", ctypes.c_int64 * 3),
        ("v_strides", ctypes.c_int64 * 3),
        ("o_strides", ctypes.c_int64 * 3),
        ("do_strides", ctypes.c_int64 * 3),
        ("dq_strides", ctypes.c_int64 * 3),
        ("dk_strides", ctypes.c_int64 * 3),
        ("dv_strides", ctypes.c_int64 * 3),
        ("softmax_scale", ctypes.c_float),
        ("causal", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("status_flag", ctypes.c_void_p),
        ("debug", ctypes.c_void_p),
        ("softcap", ctypes.c_float),
        ("local", ctypes.c_int32),
        ("window_left", ctypes.c_int32),
        ("window_right", ctypes.c_int32),
        ("o_resid", ctypes.c_void_p),
        ("o_resid_all", ctypes.c_int32),
    ]


def _fields(text):
    """Fields of a parameter struct, one kind per line: ``kind: name name ...``; ``name*3`` is an array."""
    kinds = {
        "ptr": ctypes.c_void_p,
        "size": ctypes.c_size_t,
        "i32": ctypes.c_int32,
        "i64": ctypes.c_int64,
        "f32": ctypes.c_float,
    }
    out = []
    for line in text.strip().splitlines():
        kind, names = line.split(":")
        for name in names.split():
            name, _, n = name.partition("*")
            t = kinds[kind.strip()]
            out.append((name, t * int(n) if n else t))
    return out


class SplitdPagedParams(ctypes.Structure):
    """Mirror of ``splitd_paged_params``."""

    _fields_ = _fields(
        """
        ptr: q k_pages v_pages o lse key_weights page_table seqlens_k workspace
        size: workspace_bytes
        ptr: status_flag
        i32: batch seqlen_q heads_q heads_kv head_dim num_pages page_size max_pages key_weights_len dtype causal
        i32: local window_left window_right
        f32: softmax_scale softcap
        i64: page_table_stride key_weights_stride q_strides*3 o_strides*3 k_strides*3 v_strides*3
        """
    )


class SplitdRotaryParams(ctypes.Structure):
    """Mirror of ``splitd_rotary_params``."""

    _fields_ = _fields(
        """
        ptr: q k q_out k_out positions inv_freq
        i32: batch seqlen heads_q heads_kv head_dim rotary_dim interleaved backward positions_64bit dtype
        f32: factor
        i64: position_strides*2 q_strides*3 k_strides*3 q_out_strides*3 k_out_strides*3
        """
    )


class SplitdAppendParams(ctypes.Structure):
    """Mirror of ``splitd_append_params``."""

    _fields_ = _fields(
        """
        ptr: q k v q_out k_pages v_pages page_table seqlens_k cu_seqlens positions inv_freq status_flag
        i32: batch seqlen total_tokens heads_q heads_kv head_dim num_pages page_size max_pages
        i32: rotary_dim interleaved positions_64bit dtype
        f32: factor
        i64: page_table_stride position_strides*2 q_strides*3 k_strides*3 v_strides*3 q_out_strides*3
        i64: k_page_strides*3 v_page_strides*3
        """
    )


class SplitdEvictParams(ctypes.Structure):
    """Mirror of ``splitd_evict_params``."""

    _fields_ = _fields(
        """
        ptr: k_pages v_pages page_table new_page_table seqlens_k key_weights new_seqlens kept new_weights status_flag
        i32: batch heads_kv head_dim num_pages page_size max_pages new_max_pages
        i32: key_weights_len keep keep_first keep_recent new_weights_len
        i64: page_table_stride new_page_table_stride key_weights_stride k_strides*3 v_strides*3
        """
    )


class SplitdError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"splitd_attn error {code}: {message}")
        self.code = code


_lib: Optional[ctypes.CDLL] = None


def load_library() -> ctypes.CDLL:
    """Load the shared object once; raise if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} not found: build it with `python gemm4-attention-kernels_b200/build.py` "
            "(there is no CPU or PyTorch fallback for the attention kernels)"
        )
    lib = ctypes.CDLL(LIB_PATH)
    pp = ctypes.POINTER(SplitdParams)
    lib.splitd_device_supported.argtypes = [ctypes.c_int]
    lib.splitd_device_supported.restype = ctypes.c_int
    for name in (
        "splitd_fwd",
        "splitd_bwd_preprocess",
        "splitd_bwd_dq",
        "splitd_bwd_dkdv",
        "splitd_bwd_tiles",
        "splitd_bwd_grads",
        "splitd_bwd",
        "splitd_bwd_static_scratch",
    ):
        fn = getattr(lib, name)
        fn.argtypes = [pp, ctypes.c_void_p]
        fn.restype = ctypes.c_int
    for name in (
        "splitd_fwd_workspace_bytes",
        "splitd_bwd_rowstat_elems",
        "splitd_out_resid_bytes",
        "splitd_bwd_workspace_bytes",
    ):
        fn = getattr(lib, name)
        fn.argtypes = [pp]
        fn.restype = ctypes.c_size_t
    lib.splitd_bwd_workspace_bytes_limit.argtypes = [pp, ctypes.c_size_t]
    lib.splitd_bwd_workspace_bytes_limit.restype = ctypes.c_size_t
    lib.splitd_bwd_num_chunks.argtypes = [pp]
    lib.splitd_bwd_num_chunks.restype = ctypes.c_int
    lib.splitd_bwd_chunk.argtypes = [pp, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    lib.splitd_bwd_chunk.restype = ctypes.c_int
    lib.splitd_wait_probe.argtypes = [ctypes.c_void_p, ctypes.c_uint, ctypes.c_void_p, ctypes.c_void_p]
    lib.splitd_wait_probe.restype = ctypes.c_int
    for name in ("splitd_bwd_static_scratch_limit_rowstat", "splitd_bwd_static_scratch_limit_workspace"):
        fn = getattr(lib, name)
        fn.argtypes = []
        fn.restype = ctypes.c_size_t
    for name, params in (
        ("splitd_paged_attn", SplitdPagedParams),
        ("splitd_rotary", SplitdRotaryParams),
        ("splitd_paged_append", SplitdAppendParams),
        ("splitd_paged_evict", SplitdEvictParams),
    ):
        fn = getattr(lib, name)
        fn.argtypes = [ctypes.POINTER(params), ctypes.c_void_p]
        fn.restype = ctypes.c_int
    lib.splitd_paged_attn_workspace_bytes.argtypes = [ctypes.POINTER(SplitdPagedParams)]
    lib.splitd_paged_attn_workspace_bytes.restype = ctypes.c_size_t
    lib.splitd_last_error.restype = ctypes.c_char_p
    lib.splitd_version.restype = ctypes.c_char_p
    _lib = lib
    return lib


def check(code: int) -> None:
    if code != 0:
        msg = load_library().splitd_last_error().decode("utf-8", "replace")
        raise SplitdError(code, msg)
