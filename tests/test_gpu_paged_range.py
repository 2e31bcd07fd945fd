"""GPU: attention over a paged cache where the values in it, or the spread of a row's weights, are extreme."""
import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import make_cache
from test_gpu_paged_attn import make_q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,sq", [((8, 1), 1), ((8, 1), 3), ((8, 1), 4)])
def test_rows_that_are_not_there_count_as_zeros_whatever_the_stage_held(dtype, heads, sq):
    """Sequences of nothing but infinities and NaN take turns with short ones, whose last tiles fill stages that those left
    behind: the places behind a sequence's last key have to be zeros in time."""
    from splitd_flash_attn import split_flash_attn_paged_func

    lens = [320, 33, 64, 1, 96, 5] * 60
    k, v, table, seqlens, _ = make_cache(lens, 16, heads[1], dtype, 31)
    q = make_q(len(lens), sq, heads[0], dtype, 31)
    clean = split_flash_attn_paged_func(q, k, v, table, seqlens, causal=True)
    for b in range(0, len(lens), 2):
        pages = table[b, : -(-lens[b] // 16)].long()
        v[pages], k[pages] = float("inf"), float("nan")
    for _ in range(5):
        out = split_flash_attn_paged_func(q, k, v, table, seqlens, causal=True)
        assert torch.equal(out[1::2], clean[1::2])
    assert_status_ok()
