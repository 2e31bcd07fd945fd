"""GPU: drawn shapes, masks and layouts of the paged operators and of rotary positions (fixed seeds), against their plain
forms in 64 bits."""
import random

import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import D, assert_within, rotate_ref
from test_gpu_paged_attn import check as check_attention
from test_gpu_paged_cache import check_append, check_evict, some_weights
from test_gpu_rotary import freq, make

pytestmark = pytest.mark.gpu

HEADS = [(1, 1), (2, 1), (3, 1), (8, 1), (12, 2), (32, 4), (6, 6), (20, 4), (9, 3), (16, 1), (40, 2)]


def lengths(rng, n, longest):
    return [rng.choice((0, 1, rng.randint(1, longest), rng.randint(1, longest))) for _ in range(n - 1)] + [rng.randint(1, longest)]


@pytest.mark.parametrize("seed", range(24))
def test_attention(seed):
    rng = random.Random(seed)
    hq, hkv = rng.choice(HEADS)
    sq = rng.choice((1, 1, 1, 2, 3, 4, 7, 16))
    lens = lengths(rng, rng.choice((1, 2, 5, 33, 70)), rng.choice((40, 300, 2000)))
    mask = rng.choice(("none", "causal", "window", "window"))
    window = (rng.choice((None, 0, 5, 100, 1000)), rng.choice((None, 0, 0, 3))) if mask == "window" else (None, None)
    check_attention(
        lens, sq, hq, hkv, rng.choice((1, 5, 16, 32, 50, 64, 300)), rng.choice((torch.bfloat16, torch.float16)), seed=seed,
        causal=mask == "causal", window=window, softcap=rng.choice((0.0, 0.0, 20.0)), weights=rng.random() < 0.5,
        qscale=rng.choice((1.0, 4.0)),
    )


@pytest.mark.parametrize("seed", range(12))
def test_append(seed):
    rng = random.Random(100 + seed)
    hq, hkv = rng.choice(HEADS)
    packed = rng.random() < 0.5
    B = rng.choice((1, 2, 9, 40))
    new = [rng.randint(0, 30) for _ in range(B)] if packed else [rng.randint(1, 30)] * B
    if sum(new) == 0:
        new[0] = 1
    check_append(
        new, [rng.choice((0, rng.randint(0, 200))) for _ in range(B)], hq, hkv, rng.choice((1, 7, 16, 64)),
        rng.choice((torch.bfloat16, torch.float16)), packed, 2 * rng.randint(0, 256), rng.random() < 0.5, seed=seed,
        with_q=rng.random() < 0.8,
    )


@pytest.mark.parametrize("seed", range(12))
def test_evict(seed):
    rng = random.Random(200 + seed)
    lens = lengths(rng, rng.choice((1, 3, 20)), rng.choice((50, 700, 20000)))
    keep = rng.randint(1, max(lens) + 5)
    first = rng.randint(0, keep // 3)
    kind = rng.choice(("plain", "ties", "zeros", "signs", "special"))
    check_evict(
        lens, keep, first, rng.randint(0, keep - first), rng.choice((1, 2, 3, 5)), rng.choice((1, 16, 60)),
        rng.choice((torch.bfloat16, torch.float16)), some_weights(lens, kind, seed), seed=seed,
    )


@pytest.mark.parametrize("seed", range(12))
def test_rotary(seed):
    from splitd_flash_attn import split_rotary_func

    rng = random.Random(300 + seed)
    dtype, interleaved = rng.choice((torch.bfloat16, torch.float16)), rng.random() < 0.5
    lead = rng.choice(((rng.randint(1, 4), rng.randint(1, 500)), (rng.randint(1, 900),)))
    hq, hk = rng.randint(1, 45), rng.randint(1, 9)
    q, k = make((*lead, hq, D), dtype, seed, True), make((*lead, hk, D), dtype, seed + 1)
    pos = torch.randint(-50, 10**6, lead, device="cuda")
    f = freq(2 * rng.randint(0, 256), 1e6)
    y, z = split_rotary_func(q, k, pos, f, interleaved=interleaved, factor=0.7)
    dy = make((*lead, hq, D), dtype, seed + 2)
    (g,) = torch.autograd.grad(y, q, dy)
    for name, got, x, sign in (("q", y, q, 1.0), ("k", z, k, 1.0), ("dq", g, dy, -1.0)):
        ref, tol = rotate_ref(x, pos, f, interleaved, 0.7, sign)
        assert_within(got.detach(), ref, tol, name)
    assert_status_ok()


def test_many_sequences():
    """More sequences than any block has threads, most of them empty or of a few slots."""
    lens = [(b * 7919) % 5 for b in range(3000)]
    check_attention(lens, 1, 2, 1, 4, torch.bfloat16, seed=1, weights=False)


def test_more_rows_than_a_block_holds_share_a_cache():
    check_attention([600, 31], 20, 16, 1, 32, torch.bfloat16, seed=2, causal=True)
