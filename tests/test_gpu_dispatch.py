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


# ---------------------------------------------------------------------------
# forward mode
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("interleaved", [False, True])
def test_tangents_are_rotated(interleaved):
    """Against the 64-bit form of the tangent's rotation; and against differences: the map is linear."""
    from torch.autograd import forward_ad
    from splitd_flash_attn import split_rotary_func

    q, k, tq = (tokens((2, 5), h, torch.float16, s) for h, s in ((4, 1), (2, 2), (4, 3)))
    pos, f = torch.arange(5, device="cuda") + 1000, freq(256)
    plain = split_rotary_func(q, k, pos, f, interleaved=interleaved, factor=1.25)
    ref, tol = rotate_ref(tq, pos.expand(2, 5), f, interleaved, 1.25)
    for grad in (False, True):
        x = q.clone().requires_grad_(grad)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, tq)
            y, z = split_rotary_func(dual, k, pos, f, interleaved=interleaved, factor=1.25)
            y, t = forward_ad.unpack_dual(y)
            assert forward_ad.unpack_dual(z).tangent is None
            assert torch.equal(y, plain[0]) and torch.equal(z, plain[1])
            assert_within(t, ref, tol, "tangent")
            assert y.requires_grad == grad
            y2, z2 = split_rotary_func(q, forward_ad.make_dual(k, k), pos, f, interleaved=interleaved, factor=1.25)
            assert forward_ad.unpack_dual(y2).tangent is None
            assert torch.equal(forward_ad.unpack_dual(z2).tangent, plain[1])
    moved, _ = split_rotary_func(q + tq, None, pos, f, interleaved=interleaved, factor=1.25)
    # q + tq, both results and their difference are rounded to fp16: half a step of each
    u = 2.0**-11 * 1.01
    bound = u * (moved.abs() + plain[0].abs()).double() + tol + 2.0**-24
    bound += 1.25 * u * 2 * (q + tq).abs().double().amax(-1, keepdim=True)
    assert ((moved.double() - plain[0].double() - ref).abs() <= bound).all()
    assert_status_ok()


def test_reverse_over_forward():
    """The tangent is itself differentiable: its gradient is the rotation backwards."""
    from torch.autograd import forward_ad
    from splitd_flash_attn import split_rotary_func

    q, dy = tokens((1, 9), 2, torch.bfloat16, 1), tokens((1, 9), 2, torch.bfloat16, 2)
    tq = tokens((1, 9), 2, torch.bfloat16, 3).requires_grad_()
    pos, f = torch.arange(9, device="cuda"), freq(512)
    with forward_ad.dual_level():
        y, _ = split_rotary_func(forward_ad.make_dual(q, tq), None, pos, f)
        (g,) = torch.autograd.grad(forward_ad.unpack_dual(y).tangent, tq, dy)
    x = q.clone().requires_grad_()
    (want,) = torch.autograd.grad(split_rotary_func(x, None, pos, f)[0], x, dy)
    assert torch.equal(g, want)


def test_tangents_that_would_be_lost_are_refused():
    from torch.autograd import forward_ad
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func, split_rotary_func

    q, kk, vv, k, v, table, seqlens, new_table = setup()
    w, f, pos = torch.zeros(2, 40, device="cuda"), freq(512), torch.arange(1, device="cuda")
    k0 = k.clone()
    with forward_ad.dual_level():
        def d(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = (
            [lambda a=a: split_flash_attn_paged_func(*a, table, seqlens) for a in ((d(q), k, v), (q, d(k), v), (q, k, d(v)))]
            + [lambda a=a: split_paged_append_func(*a, table, seqlens) for a in (
                (d(q), kk, vv, k, v), (q, d(kk), vv, k, v), (q, kk, d(vv), k, v), (q, kk, vv, d(k), v), (q, kk, vv, k, d(v)))]
            + [lambda a=a: split_paged_evict_func(*a[:2], table, seqlens, a[2], new_table, 24) for a in ((d(k), v, w), (k, d(v), w), (k, v, d(w)))]
            + [lambda: split_flash_attn_paged_func(q, k, v, table, seqlens, key_weights=d(w)),
               lambda: split_paged_append_func(q, kk, vv, k, v, table, seqlens, inv_freq=d(f)),
               lambda: split_rotary_func(q, None, pos, d(f))]
        )
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with Names(), pytest.raises(NotImplementedError, match="forward mode"):
            split_rotary_func(d(q), None, pos, f)
        # without a tangent everything goes on as ever
        out = split_flash_attn_paged_func(q, k, v, table, seqlens)
        assert torch.equal(split_rotary_func(q, None, pos, f)[0], split_rotary_func(q.clone(), None, pos, f)[0])
    assert torch.equal(out, split_flash_attn_paged_func(q, k, v, table, seqlens)) and torch.equal(k, k0)
    assert_status_ok()


def test_function_transforms_are_right_or_refused():
    from splitd_flash_attn import split_rotary_func

    q, dy = tokens((3, 5), 4, torch.bfloat16, 1), tokens((3, 5), 4, torch.bfloat16, 2)
    pos, f = torch.arange(5, device="cuda"), freq(512)
    want = split_rotary_func(q, None, pos, f)[0]
    x = q.clone().requires_grad_()
    (grad,) = torch.autograd.grad(split_rotary_func(x, None, pos, f)[0], x, dy)

    def fn(x):
        return split_rotary_func(x, None, pos, f)[0]

    def either(call, value):
        try:
            got = call()
        except (RuntimeError, NotImplementedError):
            return
        assert torch.equal(got, value)

    either(lambda: torch.func.functionalize(fn)(q), want)
    either(lambda: torch.vmap(lambda x: fn(x[None])[0])(q), want)
    either(lambda: torch.func.vjp(fn, q)[1](dy)[0], grad)
    either(lambda: torch.func.jvp(fn, (q,), (dy,))[1], split_rotary_func(dy, None, pos, f)[0])
    assert_status_ok()
