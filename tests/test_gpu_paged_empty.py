"""GPU: calls without sequences, tokens or pages, whatever the strides of what they are given."""
import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import D, make_cache
from test_gpu_paged_cache import freq, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [0, 2])
def test_no_sequences_and_no_slots_with_strided_tables(batch):
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func

    k, v, _, _, _ = make_cache([20], 16, 2, torch.bfloat16, 12, fill=1.0)
    k0 = k.clone()
    wide = torch.zeros(3, 40, dtype=torch.int32, device="cuda")
    lens = torch.zeros(6, dtype=torch.int32, device="cuda")[::2][:batch]
    tables = [wide[:, ::2][:batch], wide.T[:3, :3][:batch], wide[:, 5:5][:batch], wide[:, ::2][:batch, :0]]
    q, kk = tokens((batch, 1), 8, torch.bfloat16, 1), tokens((batch, 1), 2, torch.bfloat16, 2)
    w = torch.zeros(batch, 9, device="cuda")
    f = freq(1024)[::2][:256]
    for t in tables:
        out, lse = split_flash_attn_paged_func(q, k, v, t, lens, key_weights=w, return_lse=True)
        assert out.shape == q.shape and (out == 0).all() and (lse == float("-inf")).all() and (w == 0).all()
        assert split_paged_append_func(q, kk, kk, k, v, t, lens, inv_freq=f).shape == q.shape
        new = wide[:, ::2][:batch]
        n, kept, nw = split_paged_evict_func(k, v, t, lens, w, new, 7)
        assert n.shape == (batch,) and (kept == -1).all() and kept.shape == (batch, 7) and (nw == 0).all()
    assert torch.equal(k, k0)
    assert_status_ok()


def test_no_tokens_with_odd_strides():
    from splitd_flash_attn import split_paged_append_func, split_rotary_func

    k, v, table, lens, _ = make_cache([20, 3], 16, 2, torch.bfloat16, 12, fill=1.0)
    odd = torch.zeros(2, 3, 8, D + 1, dtype=torch.bfloat16, device="cuda")[..., 1:]
    none = torch.zeros(0, device="cuda").long()
    assert split_rotary_func(odd[:, :0], odd[:, :0, :2], none, freq(512))[0].shape == (2, 0, 8, D)
    assert split_rotary_func(odd[:0], None, torch.zeros(3, device="cuda").long(), freq(512)[::2][:0])[0].shape == (0, 3, 8, D)
    assert split_paged_append_func(odd[:, :0], odd[:, :0, :2], odd[:, :0, :2], k, v, table, lens).shape == (2, 0, 8, D)
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    flat = odd.flatten(0, 1)[:0]
    assert split_paged_append_func(flat, flat[:, :2], flat[:, :2], k, v, table, lens, cu_seqlens_q=cu).shape == (0, 8, D)
    assert_status_ok()
