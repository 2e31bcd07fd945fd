"""GPU: eviction next to what goes on around it: weights that change meanwhile, and decoding before and after."""
import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import D
from test_gpu_paged_cache import some_weights

pytestmark = pytest.mark.gpu


def test_weights_that_change_during_the_call_lead_out_of_no_tensor():
    """A sequence whose keys do not fit in shared memory, so that its weights are read several times, while another stream
    writes them: which slots stay is open then, but the lengths are as asked for, only the new pages are written, and
    places of `kept` that nobody filled (made to hold the largest number here) are not followed."""
    from splitd_flash_attn import split_paged_evict_func

    n, keep = 800001, 5000
    k = torch.randn(14, 1000, 1, D, device="cuda").to(torch.bfloat16)
    v = torch.randn(14, 1000, 1, D, device="cuda").to(torch.bfloat16)
    k0, v0 = k.clone(), v.clone()
    table = (torch.arange(801, device="cuda", dtype=torch.int32) % 8)[None]
    new = torch.arange(8, 13, device="cuda", dtype=torch.int32)[None]
    seqlens = torch.tensor([n], device="cuda", dtype=torch.int32)
    w = some_weights([n], "plain", 5)
    others = [some_weights([n], "plain", 6 + i) for i in range(2)]
    writer = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        full = torch.full((1, keep), 2**31 - 1, dtype=torch.int32, device="cuda")
        del full  # `kept` gets this memory
        with torch.cuda.stream(writer):
            for i in range(20):
                w.copy_(others[i % 2])
        m, _, _ = split_paged_evict_func(k, v, table, seqlens, w, new, keep, 1, 2)
        torch.cuda.synchronize()
        assert int(m) == keep
    assert torch.equal(k[:8], k0[:8]) and torch.equal(v[:8], v0[:8]) and torch.equal(k[13], k0[13]) and torch.equal(v[13], v0[13])
    assert_status_ok()
