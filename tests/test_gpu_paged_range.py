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


# ---------------------------------------------------------------------------
# one key far above all others
# ---------------------------------------------------------------------------


def far_cache(lens, page, hkv, dtype, nats, sink_value, seed):
    """Scores are q . k with q = (8, 0, ...): the first key of a sequence at `nats`, the others around 0 (spread 0.05)."""
    k, v, table, seqlens, _ = make_cache(lens, page, hkv, dtype, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    first = torch.randn(k.shape[:-1], device="cuda", generator=g) * (0.05 / 8)
    k.zero_()
    k[..., 0] = first.to(dtype)
    v.copy_((1 + 0.1 * torch.randn(v.shape, device="cuda", generator=g)).to(dtype))
    page0 = table[:, 0].long()
    k[page0, 0, :, 0] = nats / 8
    v[page0, 0] = sink_value
    return k, v, table, seqlens


def far_bounds(q, k, v, table, lens, out, p_floor):
    """Out and its bound, in 64 bits. Per key the weight is off by 2 delta + 8 u from its score (one exact product: delta = 4 u
    of the largest score) and by 2^-16 (bf16) or 2^-22 (fp16) as two 16-bit numbers, or p_floor of the largest weight where
    that is more. A tile adds 4 matrix instructions of 16 terms, cut at 2 u of the sum each, and one addition to the
    denominator; a share of the line has at most ceil(tiles / CTAs) + 1 of them, and at most all CTAs are joined."""
    u = 2.0**-24
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    hkv, sq, hq = k.shape[2], q.shape[1], q.shape[2]
    tiles = sum(-(-n // 32) for n in lens) * hkv * -(-sq * hq // hkv // 32)
    chain = (-(-tiles // sms) + 1) * (4 * 17 * 2 + 4) + sms + 40
    two = 2.0**-16 if q.dtype == torch.bfloat16 else 2.0**-22
    info = torch.finfo(q.dtype)
    for b, n in enumerate(lens):
        j = torch.arange(n, device="cuda")
        at = table[b].long()[j // k.shape[1]], j % k.shape[1]
        for h in range(hkv):
            x = 8 * k[at[0], at[1], h, 0].double()
            p = torch.softmax(x, 0)
            vv = v[at[0], at[1], h].double()
            ref = p @ vv
            rel = 2 * (8 * u * x.abs().max() + two + 8 * u + chain * u)
            bound = info.eps / 2 * 1.01 * ref.abs() + rel * (p @ vv.abs()) + info.smallest_normal * info.eps
            bound = bound + p_floor * p.max() * (vv.abs().sum(0) + n * ref.abs())
            got = out[b, :, h * (hq // hkv) : (h + 1) * (hq // hkv)].double()
            err = (got - ref).abs()
            assert (err <= bound).all(), (b, h, float((err / bound).max()), float((err / ref.abs()).max()))


# weights of the others: e^-14 = 2^-20 .. e^-22 = 2^-32. fp16 holds what is above 2^-41 of the largest (as 2^16 times the weight,
# in numbers that are multiples of 2^-24), bf16 whatever 32 bits hold
P_FLOOR = {torch.bfloat16: 0.0, torch.float16: 2.0**-41}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nats", [14.0, 16.0, 17.5, 18.0, 22.0])
@pytest.mark.parametrize("rows", [8, 16, 24, 32])
def test_many_keys_far_below_one(dtype, nats, rows):
    """One key's weight is nearly all of the row's, and its value 0: what comes out is what the others carry."""
    from splitd_flash_attn import split_flash_attn_paged_func

    lens = [131072]
    k, v, table, seqlens = far_cache(lens, 64, 1, dtype, nats, 0.0, 41)
    q = torch.zeros(1, rows // 8, 8, 512, dtype=dtype, device="cuda")
    q[..., 0] = 8
    out = split_flash_attn_paged_func(q, k, v, table, seqlens, softmax_scale=1.0)
    far_bounds(q, k, v, table, lens, out, P_FLOOR[dtype])
    assert_status_ok()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [[32], [20], [70] * 300, [3000, 40, 900]])
def test_keys_far_below_one_in_short_caches(dtype, lens):
    """Finished by the CTA that read them, or joined by the second launch."""
    from splitd_flash_attn import split_flash_attn_paged_func

    k, v, table, seqlens = far_cache(lens, 16, 2, dtype, 17.75, 0.0, 43)
    v.mul_(100)
    q = torch.zeros(len(lens), 1, 8, 512, dtype=dtype, device="cuda")
    q[..., 0] = 8
    out = split_flash_attn_paged_func(q, k, v, table, seqlens, softmax_scale=1.0)
    far_bounds(q, k, v, table, lens, out, P_FLOOR[dtype])
    assert_status_ok()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinity_at_a_key_far_below_another(dtype):
    """Its weight is small, not 0: the infinity comes through as one, in its column alone."""
    from splitd_flash_attn import split_flash_attn_paged_func

    lens = [500, 30]
    k, v, table, seqlens = far_cache(lens, 16, 1, dtype, 18.0, 0.0, 45)
    for b, n in enumerate(lens):
        v[table[b, (n - 5) // 16].long(), (n - 5) % 16, 0, 9] = float("inf")
    q = torch.zeros(2, 2, 8, 512, dtype=dtype, device="cuda")
    q[..., 0] = 8
    out = split_flash_attn_paged_func(q, k, v, table, seqlens, softmax_scale=1.0)
    assert (out[..., 9] == float("inf")).all()
    out[..., 9] = 0
    assert torch.isfinite(out).all()
    assert_status_ok()
