"""CPU: gradients that the operators on a paged cache and rotary positions do not have are refused, whichever argument asks
for them. Under FakeTensorMode, so that what is not refused ends in a fake kernel."""
import pytest
import torch

from test_paged_cpu import D, _cache, fake  # noqa: F401


def test_no_argument_loses_its_gradient(fake):  # noqa: F811
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func, split_rotary_func

    k, v, t, n = _cache()
    q, kk = (torch.empty(3, 1, h, D, dtype=torch.bfloat16, device="cuda") for h in (8, 2))
    w = torch.empty(3, 64, device="cuda")
    f = torch.empty(256, dtype=torch.float64, device="cuda")
    new = torch.empty(3, 2, dtype=torch.int32, device="cuda")
    pos = torch.empty(1, dtype=torch.int64, device="cuda")
    calls = {
        "attention": (lambda q, k, v, w: split_flash_attn_paged_func(q, k, v, t, n, key_weights=w), (q, k, v, w)),
        "append": (lambda q, kk, vv, k, v, f: split_paged_append_func(q, kk, vv, k, v, t, n, inv_freq=f), (q, kk, kk, k, v, f)),
        "eviction": (lambda k, v, w: split_paged_evict_func(k, v, t, n, w, new, 32), (k, v, w)),
        "inv_freq": (lambda f: split_rotary_func(q, kk, pos, f), (f,)),
    }
    for name, (call, args) in calls.items():
        call(*args)
        for i in range(len(args)):
            some = [a.detach().requires_grad_(i == j) for j, a in enumerate(args)]
            with pytest.raises(NotImplementedError, match=name):
                call(*some)
            with torch.no_grad():
                call(*some)
