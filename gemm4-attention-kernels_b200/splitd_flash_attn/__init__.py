"""B200 (sm_100a) SplitD FlashAttention for head_dim 512; same import surface as the reference's
``splitd_flash_attn`` package (splitd-flash-attn/src/__init__.py:3-10), plus rotary positions and the operators of
generation from a paged cache, which the reference does not have."""

from .interface import split_flash_attn_func, split_flash_attn_varlen_func
from .paged import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func
from .rotary import split_rotary_frequencies, split_rotary_func

__version__ = "0.1.0"

__all__ = [
    "split_flash_attn_func",
    "split_flash_attn_varlen_func",
    "split_flash_attn_paged_func",
    "split_paged_append_func",
    "split_paged_evict_func",
    "split_rotary_frequencies",
    "split_rotary_func",
]
