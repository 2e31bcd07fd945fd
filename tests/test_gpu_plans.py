"""GPU: what the operators on a paged cache and rotary positions keep between calls, and where their status goes."""
import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import make_cache
from test_gpu_paged_cache import freq, tokens

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh_status():
    """A status word of its own for the test, so that the next call has to make one."""
    from splitd_flash_attn import interface

    torch.cuda.synchronize()
    saved = interface._status_flags.copy()
    interface._status_flags.clear()
    yield
    torch.cuda.synchronize()
    interface._status_flags.clear()
    interface._status_flags.update(saved)
    assert_status_ok()


def cache():
    k, v, table, seqlens, free = make_cache([21, 5], 16, 1, torch.bfloat16, 1, spare=4, fill=0.0)
    bad = table.clone()
    bad[0, 0] = k.shape[0]  # no page of the cache: the kernels check it and leave 107
    return k, v, table, bad, seqlens, free[:4].view(2, 2)


def test_the_status_word_of_now_is_used(fresh_status):
    """Not the one of the call that had the same shapes before."""
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func
    from splitd_flash_attn import interface
    from splitd_flash_attn.interface import kernel_status, reset_kernel_status

    k, v, table, bad, seqlens, new = cache()
    q, kk, w = tokens((2, 1), 5, torch.bfloat16, 2), tokens((2, 1), 1, torch.bfloat16, 3), torch.ones(2, 40, device="cuda")
    calls = (
        lambda t: split_flash_attn_paged_func(q, k, v, t, seqlens),
        lambda t: split_paged_append_func(q[:, :, :3], kk, kk, k, v, t, torch.ones_like(seqlens)),
        lambda t: split_paged_evict_func(k, v, t, seqlens, w, new, 10),
    )
    for call in calls:
        call(table)
        torch.cuda.synchronize()
        before = interface._status_flags.copy()
        interface._status_flags.clear()
        assert kernel_status() == 0
        call(bad)
        assert kernel_status() == 107
        assert all(int(f) == 0 for f in before.values())
        reset_kernel_status()


def test_plans_hold_no_device_memory():
    """Prompts of ever new lengths leave nothing on the device, in a capture neither."""
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_rotary_func
    from splitd_flash_attn.interface import cu_seqlens_validation

    k, v, table, _, seqlens, _ = cache()
    pos, f = torch.zeros(1000, dtype=torch.int32, device="cuda"), freq(64)
    q = tokens((1000,), 2, torch.bfloat16, 2)
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")

    def calls(n):
        split_rotary_func(q[:n], q[:n, :1], pos[:n], f)
        with cu_seqlens_validation(False):
            split_paged_append_func(q[:n], q[:n, :1], q[:n, :1], k, v, table, seqlens, cu_seqlens_q=cu)
        split_flash_attn_paged_func(q[:2, None], k, v, table.repeat(1, 1 + n), seqlens)

    calls(999)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for n in range(1, 60):
        calls(n)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(100)
    graph.replay()
    torch.cuda.synchronize()
    del graph
    assert torch.cuda.memory_allocated() == before
    assert_status_ok()
