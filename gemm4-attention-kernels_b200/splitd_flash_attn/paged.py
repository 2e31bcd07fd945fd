"""Generation with head_dim 512: a cache of keys and values in pages, the attention that reads it, the append that
fills it and the eviction that shortens it (no counterpart in the reference, which has no cache).

A cache is two tensors ``k_pages`` and ``v_pages`` of shape (num_pages, page_size, heads_kv, 512), bf16 or fp16, any page
size. ``page_table`` (B, max_pages) int32 names the pages of each sequence, ``seqlens_k`` (B,) int32 the slots in use;
slot j of sequence b is row ``j % page_size`` of page ``page_table[b, j // page_size]``. Both stay on the device: no call
here waits for the GPU, and all of them can be captured in a CUDA graph, with one exception: an append of packed tokens
reads ``cu_seqlens_q`` back to check it, unless ``cu_seqlens_validation(False)`` is in force. The kernels check every page
id and length before they use it; ``kernel_status()`` is 107 or 108 after a call that named a page the cache does not have
or a sequence longer than its row of the table (or than its weights).

One step of a decoder's layer::

    q = split_paged_append_func(q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq=inv_freq)
    out = split_flash_attn_paged_func(q, k_pages, v_pages, page_table, seqlens_k, causal=True)

with ``seqlens_k`` counting the new tokens already. Kernels: ``csrc/paged_attn_kernel.cu``, ``csrc/rotary_kernel.cu``,
``csrc/evict_kernel.cu``.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _capi
from .interface import (
    SUPPORTED_HEAD_DIM,
    _dec,
    _enc,
    _refuse_derivatives,
    _resolve_causal_local_window,
    _status_flag,
    _validate_cu_seqlens,
)
from .rotary import (
    _DTYPES,
    _Plans,
    _check_heads,
    _check_inv_freq,
    _check_positions,
    _check_same,
    _copied,
    _launch,
    _meta,
    _model,
    _position_strides,
    _rows_fit,
    _token_strides,
    _traced,
)

_SCALE = 1.0 / math.sqrt(SUPPORTED_HEAD_DIM)

__all__ = ["split_flash_attn_paged_func", "split_paged_append_func", "split_paged_evict_func"]


# ---------------------------------------------------------------------------
# argument checks
# ---------------------------------------------------------------------------


def _check_cache(k_pages, v_pages, page_table, seqlens_k, page_table_name="page_table") -> None:
    _check_heads(k_pages, "k_pages", 4)
    _check_heads(v_pages, "v_pages", 4)
    if v_pages.shape != k_pages.shape:
        raise ValueError(f"v_pages has shape {tuple(v_pages.shape)}, expected {tuple(k_pages.shape)}")
    device = k_pages.device
    _check_same(v_pages, "v_pages", k_pages.dtype, device)
    if k_pages.shape[1] == 0 or k_pages.shape[2] == 0:
        raise ValueError(f"k_pages has shape {tuple(k_pages.shape)}: page_size and heads_kv must not be 0")
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        # a cache is not copied: its rows have to be where 16-byte accesses can reach them
        s = t.stride()
        if s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8:
            raise ValueError(f"{name} needs an innermost stride of 1 and other strides that are multiples of 8, got {s}")
    if seqlens_k.ndim != 1:
        raise ValueError(f"seqlens_k must be a 1D tensor, got rank {seqlens_k.ndim}")
    _check_same(seqlens_k, "seqlens_k", torch.int32, device)
    _check_table(page_table, page_table_name, seqlens_k.shape[0], device)


def _check_written(k_pages, v_pages) -> None:
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"{name} is written and must not be an expanded tensor, got strides {t.stride()}")


def _check_table(page_table, name, batch, device) -> None:
    if page_table.ndim != 2 or page_table.shape[0] != batch:
        raise ValueError(f"{name} has shape {tuple(page_table.shape)}, expected ({batch}, pages per sequence)")
    _check_same(page_table, name, torch.int32, device)


def _page_pointers(k_pages, v_pages):
    k_at, v_at = k_pages.data_ptr(), v_pages.data_ptr()
    if k_at % 16 or v_at % 16:
        raise ValueError(("k_pages" if k_at % 16 else "v_pages") + " must start at a 16-byte boundary")
    return k_at or _NO_MEMORY, v_at or _NO_MEMORY


# Stands for the pointer of a tensor without elements, of which nothing is touched; the C-ABI refuses NULL.
_NO_MEMORY = 256


def _fill_cache(p, k_pages, page_table) -> None:
    """What the parameter structs have in common."""
    p.batch = page_table.shape[0]
    p.heads_kv, p.head_dim = k_pages.shape[2], SUPPORTED_HEAD_DIM
    p.num_pages, p.page_size = k_pages.shape[:2]
    p.max_pages, p.page_table_stride = page_table.shape[1], page_table.stride(0)


def _check_weights(key_weights, batch, device) -> None:
    if key_weights.ndim != 2 or key_weights.shape[0] != batch:
        raise ValueError(f"key_weights has shape {tuple(key_weights.shape)}, expected ({batch}, slots)")
    _check_same(key_weights, "key_weights", torch.float32, device)
    if key_weights.shape[1] > 1 and key_weights.stride(1) != 1:
        raise ValueError("key_weights must have an innermost stride of 1")
    if batch > 1 and key_weights.stride(0) < key_weights.shape[1]:
        raise ValueError("the rows of key_weights must not overlap")


def _unit_rows(*tensors) -> bool:
    # of a tensor without elements contiguous() would not change the strides
    return all(t.stride(-1) == 1 or t.shape[-1] < 2 or t.numel() == 0 for t in tensors)


def _written(*tensors) -> None:
    """For autograd, as after an in-place operation of torch: a backward that saved one of them has to notice."""
    torch.autograd.graph.increment_version(tensors)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


def _check_paged_attn(q, k_pages, v_pages, page_table, seqlens_k, key_weights) -> None:
    _check_heads(q, "q", 4)
    _check_cache(k_pages, v_pages, page_table, seqlens_k)
    _check_same(k_pages, "k_pages", q.dtype, q.device)
    if q.shape[0] != seqlens_k.shape[0]:
        raise ValueError(f"q has shape {tuple(q.shape)}, but seqlens_k names {seqlens_k.shape[0]} sequences")
    if q.shape[2] == 0 or q.shape[2] % k_pages.shape[2]:
        raise ValueError(f"num_head ({q.shape[2]}) must be divisible by num_head_kv ({k_pages.shape[2]})")
    if key_weights is not None:
        _check_weights(key_weights, q.shape[0], q.device)


class _PagedAttnPlan:
    def __init__(self, q, k_pages, v_pages, page_table, seqlens_k, key_weights, softmax_scale, causal, left, right, softcap):
        _check_paged_attn(q, k_pages, v_pages, page_table, seqlens_k, key_weights)
        causal, local = _resolve_causal_local_window(causal, left, right)
        batch, sq, hq, _ = q.shape
        self.index = q.get_device()
        self.fits = _rows_fit(q) and _unit_rows(page_table, seqlens_k)
        self.empty = q.numel() == 0
        self.counted = key_weights is not None and key_weights.shape[1] > 0
        self.out_model = _model(q.shape, q.dtype, q.device)
        self.lse_model = _model((batch, hq, sq), torch.float32, q.device)
        p = _capi.SplitdPagedParams()
        _fill_cache(p, k_pages, page_table)
        p.seqlen_q, p.heads_q, p.dtype = sq, hq, _DTYPES[q.dtype]
        p.causal, p.local = int(causal), int(local)
        p.window_left = -1 if left is None or left < 0 else min(left, 2**31 - 1)
        p.window_right = -1 if right is None or right < 0 else min(right, 2**31 - 1)
        p.softmax_scale, p.softcap = softmax_scale, softcap
        p.q_strides, p.o_strides = _token_strides(q), _token_strides(torch.empty_like(self.out_model))
        p.k_strides, p.v_strides = k_pages.stride()[:3], v_pages.stride()[:3]
        if self.counted:
            p.key_weights, p.key_weights_len, p.key_weights_stride = _NO_MEMORY, key_weights.shape[1], key_weights.stride(0)
        n = 0 if self.empty else _capi.load_library().splitd_paged_attn_workspace_bytes(ctypes.byref(p))
        p.workspace_bytes = n
        self.workspace_model = _model((n,), torch.uint8, q.device)
        self.params = bytes(p)


_paged_attn_plans = _Plans()


def _paged_attn(q, k_pages, v_pages, page_table, seqlens_k, key_weights, softmax_scale, causal, left, right, softcap, want_lse):
    how = softmax_scale, causal, left, right, softcap
    key = (_meta(q), _meta(k_pages), _meta(v_pages), _meta(page_table), _meta(seqlens_k), _meta(key_weights), how)
    plan = _paged_attn_plans.find(key)
    if plan is None:
        plan = _paged_attn_plans.keep(key, _PagedAttnPlan(q, k_pages, v_pages, page_table, seqlens_k, key_weights, *how))
    q_at = q.data_ptr()
    if not plan.fits or q_at % 16:
        return _paged_attn(
            _copied(q), k_pages, v_pages, page_table.contiguous(), seqlens_k.contiguous(), key_weights, *how, want_lse
        )
    out = torch.empty_like(plan.out_model)
    lse = torch.empty_like(plan.lse_model) if want_lse else None
    if plan.empty:
        return out, lse
    workspace = torch.empty_like(plan.workspace_model)
    p = _capi.SplitdPagedParams.from_buffer_copy(plan.params)
    p.status_flag = _status_flag(q.device).data_ptr()
    p.q, p.o, p.workspace = q_at, out.data_ptr(), workspace.data_ptr()
    p.k_pages, p.v_pages = _page_pointers(k_pages, v_pages)
    p.page_table, p.seqlens_k = page_table.data_ptr() or _NO_MEMORY, seqlens_k.data_ptr()
    if want_lse:
        p.lse = lse.data_ptr()
    if plan.counted:
        p.key_weights = key_weights.data_ptr()
    _launch(_capi.load_library().splitd_paged_attn, p, plan.index)
    if plan.counted:
        _written(key_weights)
    return out, lse


@torch.library.custom_op("splitd_flash_attn::paged_attn", mutates_args=("key_weights",))
def _paged_attn_custom(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    seqlens_k: torch.Tensor,
    key_weights: Optional[torch.Tensor],
    softmax_scale: float,
    causal: bool,
    window_size_left: int,
    window_size_right: int,
    softcap: float,
) -> tuple[torch.Tensor, torch.Tensor]:
    return _paged_attn(
        q, k_pages, v_pages, page_table, seqlens_k, key_weights, softmax_scale, causal, _dec(window_size_left),
        _dec(window_size_right), softcap, True,
    )


@torch.library.register_fake("splitd_flash_attn::paged_attn")
def _paged_attn_fake(
    q, k_pages, v_pages, page_table, seqlens_k, key_weights, softmax_scale, causal, window_size_left, window_size_right, softcap
):
    _check_paged_attn(q, k_pages, v_pages, page_table, seqlens_k, key_weights)
    return q.new_empty(q.shape), q.new_empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32)


def split_flash_attn_paged_func(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    seqlens_k: torch.Tensor,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    window_size: Tuple[Optional[int], Optional[int]] = (None, None),
    softcap: float = 0.0,
    key_weights: Optional[torch.Tensor] = None,
    return_lse: bool = False,
):
    """Attention of a few query tokens per sequence (one when decoding, a few when verifying drafted tokens) over a
    paged cache. Forward only. Returns ``out`` or ``(out, lse)``.

    q (B, Sq, Hq, 512) with Hq % heads_kv == 0, in the cache's dtype. ``seqlens_k[b]`` counts the sequence's slots with
    its Sq new tokens: query i stands at slot ``seqlens_k[b] - Sq + i``, and ``causal``, ``window_size`` and ``softcap``
    mean what they mean in ``split_flash_attn_func`` (bottom-right alignment; causal changes nothing for Sq = 1). A row
    that sees no slot, as in a sequence of length 0, gets out 0 and lse -inf. Slots that no row of a sequence may see
    are not read, and one that only some rows may see leaves the others alone, whatever it holds.

    ``key_weights`` (B, slots) float32, optional: every slot's softmax weight, summed over all query heads and tokens,
    is added to it in place, in a fixed order (what ``split_paged_evict_func`` ranks by). Slots behind its end are not
    counted (status 108). Costs a workspace of Hq * Sq * 4 bytes per slot of it.

    The cache is read once for up to 32 rows (Sq * Hq / heads_kv); more rows take as many passes. In fp16 a weight loses up
    to 2^-41 of its row's largest one in the output.
    """
    if not isinstance(window_size, tuple) or len(window_size) != 2:
        raise TypeError("window_size must be a tuple of (left, right)")
    _refuse_derivatives("paged attention", q, k_pages, v_pages, key_weights)
    softmax_scale = _SCALE if softmax_scale is None else float(softmax_scale)
    left, right = (None if w is None else int(w) for w in window_size)
    causal, softcap = bool(causal), float(softcap)
    if _traced(q, k_pages):
        _check_paged_attn(q, k_pages, v_pages, page_table, seqlens_k, key_weights)
        out, lse = torch.ops.splitd_flash_attn.paged_attn(
            q, k_pages, v_pages, page_table, seqlens_k, key_weights, softmax_scale, causal, _enc(left), _enc(right), softcap
        )
    else:
        out, lse = _paged_attn(
            q, k_pages, v_pages, page_table, seqlens_k, key_weights, softmax_scale, causal, left, right, softcap, return_lse
        )
    return (out, lse) if return_lse else out


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


def _check_append(q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q) -> None:
    rank = 4 if cu_seqlens_q is None else 3
    _check_heads(k, "k", rank)
    _check_heads(v, "v", rank)
    _check_cache(k_pages, v_pages, page_table, seqlens_k)
    _check_written(k_pages, v_pages)
    if v.shape != k.shape:
        raise ValueError(f"v has shape {tuple(v.shape)}, expected {tuple(k.shape)}")
    if k.shape[-2] != k_pages.shape[2]:
        raise ValueError(f"k has {k.shape[-2]} heads, the cache {k_pages.shape[2]}")
    for name, t in (("v", v), ("k_pages", k_pages)):
        _check_same(t, name, k.dtype, k.device)
    if q is not None:
        _check_heads(q, "q", rank)
        if q.shape[:-2] != k.shape[:-2]:
            raise ValueError(f"q has shape {tuple(q.shape)}, expected the tokens of k, {tuple(k.shape)}")
        _check_same(q, "q", k.dtype, k.device)
        if q.shape[-2] == 0 or q.shape[-2] % k.shape[-2]:
            raise ValueError(f"num_head ({q.shape[-2]}) must be divisible by num_head_kv ({k.shape[-2]})")
    batch = seqlens_k.shape[0]
    if cu_seqlens_q is None:
        if k.shape[0] != batch:
            raise ValueError(f"k has shape {tuple(k.shape)}, but seqlens_k names {batch} sequences")
    elif tuple(cu_seqlens_q.shape) != (batch + 1,):
        raise ValueError(f"cu_seqlens_q must have shape ({batch + 1},), got {tuple(cu_seqlens_q.shape)}")
    else:
        _check_same(cu_seqlens_q, "cu_seqlens_q", torch.int32, k.device)
    if inv_freq is not None:
        _check_inv_freq(inv_freq, k.device)
    elif positions is not None:
        raise ValueError("positions is given without inv_freq: there is nothing to rotate")
    if positions is not None:
        _check_positions(positions, k.shape[:-2], k.device)


class _AppendPlan:
    def __init__(self, q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q, interleaved, factor):
        _check_append(q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q)
        packed = cu_seqlens_q is not None
        self.index = k.get_device()
        self.pairs = 0 if inv_freq is None else inv_freq.numel()
        self.fits = (
            _rows_fit(q) and _rows_fit(k) and _rows_fit(v) and _unit_rows(page_table, seqlens_k)
            and (self.pairs < 2 or inv_freq.stride(0) == 1)
        )
        self.empty = k.numel() == 0
        self.q_model = None if q is None else _model(q.shape, q.dtype, q.device)
        p = _capi.SplitdAppendParams()
        _fill_cache(p, k_pages, page_table)
        p.seqlen, p.total_tokens = (0, k.shape[0]) if packed else (k.shape[1], 0)
        p.dtype, p.rotary_dim, p.interleaved, p.factor = _DTYPES[k.dtype], 2 * self.pairs, int(interleaved), factor
        if positions is not None:
            p.positions_64bit, p.position_strides = int(positions.dtype == torch.int64), _position_strides(positions, packed)
        if q is not None:
            p.heads_q, p.q_strides, p.q_out_strides = q.shape[-2], _token_strides(q), _token_strides(torch.empty_like(self.q_model))
        p.k_strides, p.v_strides = _token_strides(k), _token_strides(v)
        p.k_page_strides, p.v_page_strides = k_pages.stride()[:3], v_pages.stride()[:3]
        self.params = bytes(p)


_append_plans = _Plans()


def _paged_append(q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q, interleaved, factor):
    key = (
        _meta(q), _meta(k), _meta(v), _meta(k_pages), _meta(v_pages), _meta(page_table), _meta(seqlens_k), _meta(inv_freq),
        _meta(positions), _meta(cu_seqlens_q), interleaved, factor,
    )
    plan = _append_plans.find(key)
    if plan is None:
        plan = _append_plans.keep(
            key,
            _AppendPlan(q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q, interleaved, factor),
        )
    q_at, k_at, v_at = 0 if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr()
    if not plan.fits or q_at % 16 or k_at % 16 or v_at % 16:
        return _paged_append(
            None if q is None else _copied(q), _copied(k), _copied(v), k_pages, v_pages, page_table.contiguous(),
            seqlens_k.contiguous(), None if inv_freq is None else inv_freq.contiguous(), positions, cu_seqlens_q, interleaved,
            factor,
        )
    if cu_seqlens_q is not None:
        _validate_cu_seqlens(cu_seqlens_q, "cu_seqlens_q", seqlens_k.shape[0], total_tokens=k.shape[0])
    q_out = None if q is None else torch.empty_like(plan.q_model)
    if plan.empty:
        return q_out
    p = _capi.SplitdAppendParams.from_buffer_copy(plan.params)
    p.status_flag = _status_flag(k.device).data_ptr()
    p.k, p.v = k_at, v_at
    p.k_pages, p.v_pages = _page_pointers(k_pages, v_pages)
    if p.k_pages == p.v_pages and k_pages.numel():
        raise ValueError("k_pages and v_pages must not be the same memory: both are written")
    p.page_table, p.seqlens_k = page_table.data_ptr() or _NO_MEMORY, seqlens_k.data_ptr() or _NO_MEMORY
    if q is not None:
        p.q, p.q_out = q_at, q_out.data_ptr()
    if plan.pairs:
        p.inv_freq = inv_freq.data_ptr()
        if positions is not None:
            p.positions = positions.data_ptr()
    if cu_seqlens_q is not None:
        p.cu_seqlens = cu_seqlens_q.data_ptr()
    _launch(_capi.load_library().splitd_paged_append, p, plan.index)
    _written(k_pages, v_pages)
    return q_out


@torch.library.custom_op("splitd_flash_attn::paged_append", mutates_args=("k_pages", "v_pages"))
def _paged_append_custom(
    q: Optional[torch.Tensor],
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    seqlens_k: torch.Tensor,
    inv_freq: Optional[torch.Tensor],
    positions: Optional[torch.Tensor],
    cu_seqlens_q: Optional[torch.Tensor],
    interleaved: bool,
    factor: float,
) -> torch.Tensor:
    """The rotated q; an empty tensor if there is none."""
    out = _paged_append(
        q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q, interleaved, factor
    )
    return k.new_empty((0,)) if out is None else out


@torch.library.register_fake("splitd_flash_attn::paged_append")
def _paged_append_fake(
    q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q, interleaved, factor
):
    _check_append(q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q)
    return k.new_empty((0,) if q is None else q.shape)


def split_paged_append_func(
    q: Optional[torch.Tensor],
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    seqlens_k: torch.Tensor,
    inv_freq: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    factor: float = 1.0,
):
    """New tokens into a paged cache, in place, in one launch with the rotation of their queries and keys. Returns the
    rotated q (None if q is None). Forward only.

    Batched: q (B, S, Hq, 512), k and v (B, S, heads_kv, 512), S new tokens per sequence. Packed: (T, heads, 512) and
    ``cu_seqlens_q`` int32 of B + 1 entries, any number of tokens per sequence (its values are checked as in
    ``split_flash_attn_varlen_func``, which waits for the GPU and cannot be captured; ``cu_seqlens_validation(False)``
    leaves that out). ``seqlens_k[b]`` is the length of sequence b WITH its new tokens, which fill its last slots. Tokens
    whose slot would be negative are not stored (length 0: a row that only pads the batch); two tokens must not share a
    slot, nor ``k_pages`` and ``v_pages`` memory.

    ``inv_freq``, ``interleaved``, ``factor``: as in ``split_rotary_func``; without ``inv_freq`` nothing is rotated.
    Positions are the slots, unless ``positions`` (one per token, int32 or int64) says otherwise, as it has to after an
    eviction.
    """
    _refuse_derivatives("paged append", q, k, v, k_pages, v_pages, inv_freq)
    interleaved, factor = bool(interleaved), float(factor)
    if _traced(k, k_pages):
        args = (q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q)
        _check_append(*args)
        out = torch.ops.splitd_flash_attn.paged_append(*args, interleaved, factor)
        return None if q is None else out
    return _paged_append(
        q, k, v, k_pages, v_pages, page_table, seqlens_k, inv_freq, positions, cu_seqlens_q, interleaved, factor
    )


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------


def _check_evict(
    k_pages, v_pages, page_table, seqlens_k, key_weights, new_page_table, keep, keep_first, keep_recent, weights_len
) -> None:
    _check_cache(k_pages, v_pages, page_table, seqlens_k)
    _check_written(k_pages, v_pages)
    batch = seqlens_k.shape[0]
    _check_weights(key_weights, batch, k_pages.device)
    _check_table(new_page_table, "new_page_table", batch, k_pages.device)
    counts = ("keep", keep), ("keep_first", keep_first), ("keep_recent", keep_recent), ("weights_len", weights_len)
    for name, n in counts if weights_len is not None else counts[:3]:
        if isinstance(n, bool) or not isinstance(n, (int, torch.SymInt)):
            raise TypeError(f"{name} must be an int, got {type(n).__name__}")
        if n < 0:
            raise ValueError(f"{name} must be non-negative, got {n}")
    if keep < 1 or keep < keep_first + keep_recent:
        raise ValueError(f"keep ({keep}) must be at least 1 and at least keep_first + keep_recent ({keep_first} + {keep_recent})")
    if keep > 2**30:
        raise ValueError(f"keep ({keep}) must be at most 2^30")
    if weights_len is not None and not keep <= weights_len <= 2**30:
        raise ValueError(f"weights_len ({weights_len}) must be at least keep ({keep}) and at most 2^30")
    if new_page_table.shape[1] * k_pages.shape[1] < keep:
        raise ValueError(
            f"new_page_table has {new_page_table.shape[1]} pages of {k_pages.shape[1]} slots per sequence, too few for {keep}"
        )


class _EvictPlan:
    def __init__(
        self, k_pages, v_pages, page_table, seqlens_k, key_weights, new_page_table, keep, keep_first, keep_recent, weights_len
    ):
        _check_evict(
            k_pages, v_pages, page_table, seqlens_k, key_weights, new_page_table, keep, keep_first, keep_recent, weights_len
        )
        device, batch = k_pages.device, seqlens_k.shape[0]
        self.index = k_pages.get_device()
        self.fits = _unit_rows(page_table, new_page_table, seqlens_k)
        self.empty = batch == 0
        self.seqlens_model = _model((batch,), torch.int32, device)
        self.kept_model = _model((batch, keep), torch.int32, device)
        self.weights_model = _model((batch, keep if weights_len is None else weights_len), torch.float32, device)
        p = _capi.SplitdEvictParams()
        _fill_cache(p, k_pages, page_table)
        p.new_max_pages, p.new_page_table_stride = new_page_table.shape[1], new_page_table.stride(0)
        p.key_weights_len, p.key_weights_stride = key_weights.shape[1], key_weights.stride(0)
        p.keep, p.keep_first, p.keep_recent = keep, keep_first, keep_recent
        p.new_weights_len = 0 if weights_len is None else weights_len
        p.k_strides, p.v_strides = k_pages.stride()[:3], v_pages.stride()[:3]
        self.params = bytes(p)


_evict_plans = _Plans()


def _paged_evict(
    k_pages, v_pages, page_table, seqlens_k, key_weights, new_page_table, keep, keep_first, keep_recent, weights_len
):
    how = keep, keep_first, keep_recent, weights_len
    key = (
        _meta(k_pages), _meta(v_pages), _meta(page_table), _meta(seqlens_k), _meta(key_weights), _meta(new_page_table), how,
        type(keep), type(keep_first), type(keep_recent), type(weights_len),
    )
    plan = _evict_plans.find(key)
    if plan is None:
        plan = _evict_plans.keep(key, _EvictPlan(k_pages, v_pages, page_table, seqlens_k, key_weights, new_page_table, *how))
    if not plan.fits:
        return _paged_evict(
            k_pages, v_pages, page_table.contiguous(), seqlens_k.contiguous(), key_weights, new_page_table.contiguous(), *how
        )
    new_seqlens = torch.empty_like(plan.seqlens_model)
    kept, new_weights = torch.empty_like(plan.kept_model), torch.empty_like(plan.weights_model)
    if plan.empty:
        return new_seqlens, kept, new_weights
    p = _capi.SplitdEvictParams.from_buffer_copy(plan.params)
    p.status_flag = _status_flag(k_pages.device).data_ptr()
    p.k_pages, p.v_pages = _page_pointers(k_pages, v_pages)
    p.page_table, p.new_page_table = page_table.data_ptr() or _NO_MEMORY, new_page_table.data_ptr()
    p.seqlens_k, p.key_weights = seqlens_k.data_ptr(), key_weights.data_ptr() or _NO_MEMORY
    p.new_seqlens, p.kept, p.new_weights = new_seqlens.data_ptr(), kept.data_ptr(), new_weights.data_ptr()
    _launch(_capi.load_library().splitd_paged_evict, p, plan.index)
    _written(k_pages, v_pages)
    return new_seqlens, kept, new_weights


@torch.library.custom_op("splitd_flash_attn::paged_evict", mutates_args=("k_pages", "v_pages"))
def _paged_evict_custom(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    seqlens_k: torch.Tensor,
    key_weights: torch.Tensor,
    new_page_table: torch.Tensor,
    keep: int,
    keep_first: int,
    keep_recent: int,
    weights_len: Optional[int] = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return _paged_evict(
        k_pages, v_pages, page_table, seqlens_k, key_weights, new_page_table, keep, keep_first, keep_recent, weights_len
    )


@torch.library.register_fake("splitd_flash_attn::paged_evict")
def _paged_evict_fake(
    k_pages, v_pages, page_table, seqlens_k, key_weights, new_page_table, keep, keep_first, keep_recent, weights_len=None
):
    _check_evict(
        k_pages, v_pages, page_table, seqlens_k, key_weights, new_page_table, keep, keep_first, keep_recent, weights_len
    )
    batch = seqlens_k.shape[0]
    width = keep if weights_len is None else weights_len
    return seqlens_k.new_empty((batch,)), seqlens_k.new_empty((batch, keep)), key_weights.new_empty((batch, width))


def split_paged_evict_func(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    seqlens_k: torch.Tensor,
    key_weights: torch.Tensor,
    new_page_table: torch.Tensor,
    keep: int,
    keep_first: int = 0,
    keep_recent: int = 0,
    weights_len: Optional[int] = None,
):
    """Shortens every sequence to at most ``keep`` slots: its first ``keep_first``, its last ``keep_recent``, and of the
    others those with the largest ``key_weights`` (of equal ones the lower slot; NaN counts as the largest). The kept keys
    and values are copied, in slot order, to the pages of ``new_page_table`` (B, new pages per sequence), which no
    sequence may be using: pages are often shared between sequences, so none is changed in place. Sequences that are
    short enough already are copied as they are; leave them out of the call to leave them alone.

    ``key_weights`` (B, slots) has to reach as far as the sequences do: one that is longer is cut to it first, which
    loses its last slots, ``keep_recent`` or not (status 108).

    Returns ``(new_seqlens, kept, new_weights)``: (B,) int32 lengths; (B, keep) int32 old slots, ascending, -1 behind
    the last; (B, weights_len) float32 their weights, 0 behind the last. ``weights_len`` is ``keep`` if not given. To go
    on with them as ``key_weights`` of the new cache, ask for as many as that may grow to: slots behind the end of
    ``key_weights`` are not counted. Keys keep the rotation of the position they had, so tokens that follow need
    ``positions`` in ``split_paged_append_func``.
    """
    args = (k_pages, v_pages, page_table, seqlens_k, key_weights, new_page_table, keep, keep_first, keep_recent, weights_len)
    _refuse_derivatives("paged eviction", k_pages, v_pages, key_weights)
    if _traced(k_pages):
        _check_evict(*args)
        return torch.ops.splitd_flash_attn.paged_evict(*args)
    return _paged_evict(*args)
