"""CPU: the width of the eviction's new weights, and what of it is refused."""
import ctypes

import pytest
import torch

from splitd_flash_attn import _capi
from test_paged_cpu import D, _cache, _refused, fake  # noqa: F401


def test_width_of_the_new_weights(fake):  # noqa: F811
    from splitd_flash_attn import split_paged_evict_func as fn

    k, v, t, n = _cache()
    w = torch.empty(3, 64, device="cuda")
    new = torch.empty(3, 2, dtype=torch.int32, device="cuda")
    for width in (32, 33, 1000):
        a, b, c = fn(k, v, t, n, w, new, 32, 2, 3, weights_len=width)
        assert a.shape == (3,) and b.shape == (3, 32) and c.shape == (3, width) and c.dtype == torch.float32
    assert fn(k, v, t, n, w, new, 32, 2, 3, weights_len=None)[2].shape == (3, 32)
    for width in (31, 0, -1, 2**30 + 1, 2**31 - 1, 2**31):
        with pytest.raises(ValueError, match="weights_len"):
            fn(k, v, t, n, w, new, 32, weights_len=width)
    for width in (40.0, True, "40"):
        with pytest.raises(TypeError, match="weights_len"):
            fn(k, v, t, n, w, new, 32, weights_len=width)


def test_entry_point_refuses_a_narrow_one():
    fn = _capi.load_library().splitd_paged_evict
    for width in (31, -1, 2**30 + 1, 2**31 - 1):
        p = _capi.SplitdEvictParams()
        for n in ("k_pages", "v_pages", "page_table", "new_page_table", "seqlens_k", "key_weights", "new_seqlens", "kept", "new_weights"):
            setattr(p, n, 1 << 20)
        p.batch, p.heads_kv, p.head_dim, p.num_pages, p.page_size, p.max_pages, p.new_max_pages = 2, 2, D, 10, 16, 4, 2
        p.key_weights_len, p.keep, p.new_weights_len = 64, 32, width
        _refused(fn, p, "new_weights_len")
    assert ctypes.sizeof(_capi.SplitdEvictParams) % 8 == 0
