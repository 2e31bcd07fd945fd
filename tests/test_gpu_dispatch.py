"""GPU: what torch can see of the operators on a paged cache and of rotary positions: tracing, dispatch modes, version
counters, forward mode, and gradients that would be lost."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from gpu_utils import assert_status_ok
from paged_utils import D, assert_within, make_cache, rotate_ref
from test_gpu_paged_cache import freq, tokens

pytestmark = pytest.mark.gpu


def setup(seed=51):
    k, v, table, seqlens, free = make_cache([40, 21], 16, 2, torch.bfloat16, seed, spare=4, fill=0.0)
    q, kk, vv = (tokens((2, 1), h, torch.bfloat16, seed + h) for h in (8, 2, 3))
    return q, kk, vv[:, :, :2], k, v, table, seqlens, free[:4].view(2, 2)


def step(q, kk, vv, k, v, table, seqlens, new_table, w, f):
    """All four operators."""
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func, split_rotary_func

    pos = (seqlens - 1)[:, None]
    qr, kr = split_rotary_func(q, kk, pos, f)
    split_paged_append_func(None, kr, vv, k, v, table, seqlens)
    out, lse = split_flash_attn_paged_func(qr, k, v, table, seqlens, causal=True, key_weights=w, return_lse=True)
    return (out, lse) + tuple(split_paged_evict_func(k, v, table, seqlens, w, new_table, 24, 2, 2))


OPS = {"splitd_flash_attn." + n for n in ("rotary", "paged_append", "paged_attn", "paged_evict")}


def check_traced(trace):
    args = [*setup(), torch.zeros(2, 40, device="cuda"), freq(512)]
    want_state = [a.clone() for a in args]
    want = step(*want_state)
    traced = trace(step, [a.clone() for a in args])
    got_state = [a.clone() for a in args]
    got = traced(*got_state)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(got_state, want_state))
    return traced


@pytest.mark.parametrize("pre_dispatch", [False, True])
def test_make_fx_records_the_operators(pre_dispatch):
    from torch.fx.experimental.proxy_tensor import make_fx

    graph = check_traced(lambda fn, args: make_fx(fn, pre_dispatch=pre_dispatch)(*args)).graph
    names = {str(n.target) for n in graph.nodes}
    assert all(any(n.startswith(op) for n in names) for op in OPS), names


def test_jit_trace_records_the_operators():
    check_traced(lambda fn, args: torch.jit.trace(fn, args, check_trace=False))


class Names(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


def test_dispatch_modes_see_the_operators_forward_and_backward():
    from splitd_flash_attn import split_rotary_func

    args = [*setup(), torch.zeros(2, 40, device="cuda"), freq(512)]
    with Names() as names:
        step(*args)
    assert all(any(n.startswith(op) for n in names.seen) for op in OPS), names.seen
    q, f, pos = args[0].clone().requires_grad_(), freq(512), torch.arange(1, device="cuda")
    dy = tokens((2, 1), 8, torch.bfloat16, 3)
    want = torch.autograd.grad(split_rotary_func(q, None, pos, f)[0], q, dy)[0]
    y, _ = split_rotary_func(q, None, pos, f)
    with Names() as names:  # the forward ran outside
        got = torch.autograd.grad(y, q, dy)[0]
    assert torch.equal(got, want) and any(n.startswith("splitd_flash_attn.rotary") for n in names.seen)
    with Names():
        y, _ = split_rotary_func(q, None, pos, f)
    assert torch.equal(torch.autograd.grad(y, q, dy)[0], want)
    assert_status_ok()


# ---------------------------------------------------------------------------
# version counters
# ---------------------------------------------------------------------------


def test_writes_raise_the_version_counters():
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func

    q, kk, vv, k, v, table, seqlens, new_table = setup()
    w = torch.zeros(2, 40, device="cuda")

    def versions():
        return k._version, v._version, w._version, q._version, kk._version, seqlens._version, table._version

    before = versions()
    split_paged_append_func(q, kk, vv, k, v, table, seqlens)
    after = versions()
    assert after[0] > before[0] and after[1] > before[1] and after[2:] == before[2:]
    before = after
    split_flash_attn_paged_func(q, k, v, table, seqlens)
    assert versions() == before
    split_flash_attn_paged_func(q, k, v, table, seqlens, key_weights=w)
    after = versions()
    assert after[2] > before[2] and after[:2] == before[:2] and after[3:] == before[3:]
    before = after
    split_paged_evict_func(k, v, table, seqlens, w, new_table, 24)
    after = versions()
    assert after[0] > before[0] and after[1] > before[1] and after[2:] == before[2:]
    # of the tensor that a view belongs to
    kv = torch.stack((k, v), 1)
    before = kv._version
    split_paged_append_func(q, kk, vv, kv[:, 0], kv[:, 1], table, seqlens)
    assert kv._version > before


def test_autograd_notices_that_a_saved_cache_was_written():
    from splitd_flash_attn import split_paged_append_func

    q, kk, vv, k, v, table, seqlens, _ = setup()
    x = torch.ones(1, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = (x * k).sum()  # saves k
    split_paged_append_func(q, kk, vv, k, v, table, seqlens)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_caches_made_in_inference_mode():
    """They have no version counter."""
    with torch.inference_mode():
        args = [*setup(), torch.zeros(2, 40, device="cuda"), freq(512)]
        want = step(*[a.clone() for a in args])
        got = step(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert_status_ok()
