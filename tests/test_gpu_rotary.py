"""GPU: rotary positions, forward and backward, against the plain form in 64 bits (bounds: paged_utils)."""
import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import D, assert_within, rotate_ref

pytestmark = pytest.mark.gpu


def make(shape, dtype, seed, grad=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype).requires_grad_(grad)


def freq(r, base=10000.0):
    return torch.pow(torch.tensor(base, dtype=torch.float64, device="cuda"), -torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / max(r, 1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("r", [512, 256, 128, 64, 16, 2, 510, 250, 34, 6, 0])
def test_forward_and_gradients(dtype, interleaved, r):
    from splitd_flash_attn import split_rotary_func

    q, k = make((2, 37, 6, D), dtype, 1, True), make((2, 37, 3, D), dtype, 2, True)
    dq, dk = make((2, 37, 6, D), dtype, 3), make((2, 37, 3, D), dtype, 4)
    pos = torch.randint(0, 200000, (2, 37), device="cuda", dtype=torch.int32)
    f = freq(r)
    qo, ko = split_rotary_func(q, k, pos, f, interleaved=interleaved, factor=1.25)
    gq, gk = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    for name, got, x, sign in (("q", qo, q, 1.0), ("k", ko, k, 1.0), ("dq", gq, dq, -1.0), ("dk", gk, dk, -1.0)):
        ref, tol = rotate_ref(x, pos, f, interleaved, 1.25, sign)
        assert got.dtype == dtype and got.is_contiguous()
        assert_within(got.detach(), ref, tol, name)
        assert torch.equal(got[..., r:], x[..., r:])  # behind the rotated part: bit for bit
    assert_status_ok()


def test_gradient_against_differences():
    """The map is linear: sum(dy * f(x)) changes by sum(dx * e) when x changes by e. In fp16 with 32-bit sums; both sides
    carry a rounding of each output, at most 2^-11 of it."""
    from splitd_flash_attn import split_rotary_func

    q = make((1, 20, 4, D), torch.float16, 5, True)
    dy = make((1, 20, 4, D), torch.float16, 6)
    pos = torch.arange(20, device="cuda", dtype=torch.int64) + 7
    f = freq(512)
    y, none = split_rotary_func(q, None, pos, f)
    assert none is None
    (g,) = torch.autograd.grad(y, q, dy)
    for seed in range(3):
        e = make((1, 20, 4, D), torch.float16, 10 + seed)
        ye, _ = split_rotary_func(e, None, pos, f)
        left, right = (dy.double() * ye.double()), (g.double() * e.double())
        bound = 2.0**-11 * 1.01 * (left.abs().sum() + right.abs().sum())
        assert (left.sum() - right.sum()).abs() <= bound


def test_far_positions_and_their_types():
    """Angles are formed in 64 bits. At position 2^40 those leave an error of their own, 2^40 * 2^-52 turns at most here and
    in the oracle each: 2^-12 * 2 pi * 2 = 3e-3 rad."""
    from splitd_flash_attn import split_rotary_func

    q = make((5, 3, D), torch.bfloat16, 7)
    pos = torch.tensor([0, 3, 10**6, 2**31 + 5, 2**40 + 1], device="cuda")
    f = freq(512)
    y, _ = split_rotary_func(q, None, pos, f)
    ref, tol = rotate_ref(q, pos, f)
    far = (pos > 2**35)[:, None, None] * 3.1e-3 * q.abs().amax(-1, keepdim=True).double() * 2
    assert_within(y, ref, tol + far, "q")
    neg, _ = split_rotary_func(q, None, -pos[:3].repeat(2)[:5], f)
    ref, tol = rotate_ref(q, -pos[:3].repeat(2)[:5], f)
    assert_within(neg, ref, tol, "q")
    y32, _ = split_rotary_func(q[:3], None, pos[:3].to(torch.int32), f)
    assert torch.equal(y32, y[:3])


def test_layouts_strides_and_shared_positions():
    from splitd_flash_attn import split_rotary_func

    f = freq(256)
    qkv = make((2, 11, 16, D), torch.bfloat16, 8)
    q, k = qkv[:, :, :8], qkv[:, :, 8:12]
    pos = torch.arange(11, device="cuda", dtype=torch.int32)
    a = split_rotary_func(q, k, pos, f)
    b = split_rotary_func(q.contiguous(), k.contiguous(), pos.expand(2, 11), f)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c = split_rotary_func(q.flatten(0, 1), k.flatten(0, 1), pos.repeat(2), f)
    assert torch.equal(a[0].flatten(0, 1), c[0]) and torch.equal(a[1].flatten(0, 1), c[1])
    wide = torch.arange(22, device="cuda", dtype=torch.int32)
    d = split_rotary_func(q, k, wide[::2], f)
    e = split_rotary_func(q, k, wide[::2].contiguous(), f)
    assert torch.equal(d[0], e[0])
    odd = make((1, 5, 2, D + 1), torch.bfloat16, 9)[..., 1:]
    assert torch.equal(split_rotary_func(odd, None, pos[:5], f)[0], split_rotary_func(odd.contiguous(), None, pos[:5], f)[0])
    # one head broadcast over four: the gradient is the sum over them
    x = make((2, 11, 1, D), torch.bfloat16, 10, True)
    y, _ = split_rotary_func(x.expand(2, 11, 4, D), None, pos, f)
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    ref, tol = rotate_ref(torch.ones_like(x), pos.expand(2, 11), f, sign=-1.0)
    assert_within(g, 4 * ref, 4 * tol + 2.0**-8 * 4 * ref.abs(), "broadcast")


def test_special_values_stay_in_their_pair():
    from splitd_flash_attn import split_rotary_func

    for interleaved in (False, True):
        for r in (256, 250):
            q = make((1, 2, 2, D), torch.bfloat16, 11)
            f, pos = freq(r), torch.tensor([5, 6], device="cuda", dtype=torch.int32)
            clean, _ = split_rotary_func(q, None, pos, f, interleaved=interleaved)
            q[0, 0, 0, 4] = float("nan")
            q[0, 1, 1, 300] = float("inf")
            got, _ = split_rotary_func(q, None, pos, f, interleaved=interleaved)
            mate = 5 if interleaved else 4 + r // 2
            assert torch.isnan(got[0, 0, 0, [4, mate]]).all() and got[0, 1, 1, 300] == float("inf")
            got[0, 0, 0, [4, mate]] = clean[0, 0, 0, [4, mate]]
            got[0, 1, 1, 300] = clean[0, 1, 1, 300]
            assert torch.equal(got, clean)


def test_one_input_one_gradient_and_second_derivatives():
    from splitd_flash_attn import split_rotary_func

    f, pos = freq(512), torch.arange(9, device="cuda")
    q, k = make((1, 9, 2, D), torch.bfloat16, 12, True), make((1, 9, 1, D), torch.bfloat16, 13)
    qo, ko = split_rotary_func(q, k, pos, f)
    assert qo.requires_grad
    (g,) = torch.autograd.grad(qo.float().sum() + ko.float().sum(), q)
    alone, _ = split_rotary_func(q, None, pos, f)
    assert torch.equal(alone, qo)
    (g2,) = torch.autograd.grad(alone.float().sum(), q)
    assert torch.equal(g, g2)
    none, ko2 = split_rotary_func(None, k, pos, f)
    assert none is None and torch.equal(ko2, ko)
    # the gradient of the gradient is the forward map again
    y, _ = split_rotary_func(q, None, pos, f)
    dy = make((1, 9, 2, D), torch.bfloat16, 14, True)
    (gx,) = torch.autograd.grad(y, q, dy, create_graph=True)
    t = make((1, 9, 2, D), torch.bfloat16, 15)
    (back,) = torch.autograd.grad(gx, dy, t)
    assert torch.equal(back, split_rotary_func(t, None, pos, f)[0])


@pytest.mark.parametrize("shape", [(0, 5, 4), (2, 0, 4), (2, 5, 0), (1, 1, 1), (3, 2000, 40)])
def test_sizes(shape):
    from splitd_flash_attn import split_rotary_func

    q = make((*shape, D), torch.bfloat16, 16)
    pos = torch.arange(shape[1], device="cuda")
    y, _ = split_rotary_func(q, None, pos, freq(512))
    ref, tol = rotate_ref(q, pos.expand(shape[:2]), freq(512))
    assert_within(y, ref, tol, "q")


def test_captured_and_compiled_with_attention():
    """Rotary positions in front of the training attention: eager, captured forward and backward, and compiled."""
    from splitd_flash_attn import split_flash_attn_func, split_rotary_func

    f, pos = freq(512), torch.arange(128, device="cuda")
    q, k, v = (make((1, 128, h, D), torch.bfloat16, 17 + h, True) for h in (8, 2, 2))
    do = make((1, 128, 8, D), torch.bfloat16, 30)

    def step(q, k, v):
        qr, kr = split_rotary_func(q, k, pos, f)
        return split_flash_attn_func(qr, kr, v, causal=True)

    def grads():
        return torch.autograd.grad(step(q, k, v), (q, k, v), do)

    want = grads()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grads()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    compiled = torch.autograd.grad(torch.compile(step, fullgraph=True)(q, k, v), (q, k, v), do)
    assert all(torch.equal(a, b) for a, b in zip(want, compiled))
    # the gradients of the whole against 64 bits: softmax attention of rotated inputs
    qd, kd, vd = (t.detach().double().requires_grad_() for t in (q, k, v))

    def rot(x):
        ang = pos.double()[:, None, None] * f
        a, b = x[..., :256], x[..., 256:]
        return torch.cat((a * torch.cos(ang) - b * torch.sin(ang), a * torch.sin(ang) + b * torch.cos(ang)), -1)

    s = torch.einsum("bihgd,bjhd->bhgij", rot(qd).view(1, 128, 2, 4, D), rot(kd)) * D**-0.5
    s = s.masked_fill(~torch.ones(128, 128, device="cuda").tril().bool(), float("-inf"))
    o = torch.einsum("bhgij,bjhd->bihgd", torch.softmax(s, -1), vd).reshape(1, 128, 8, D)
    ref = torch.autograd.grad(o, (qd, kd, vd), do.double())
    # the rotated q, k and each gradient are rounded to bf16 once or twice on the way: a few times 2^-9, in norm
    for a, r in zip(want, ref):
        assert (a.double() - r).norm() <= 4 * 2.0**-8 * r.norm()
    assert_status_ok()
