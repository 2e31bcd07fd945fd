"""GPU: attention over a paged cache against its plain form in 64 bits (bounds: paged_utils)."""
import math

import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import D, assert_within, attention_ref, make_cache

pytestmark = pytest.mark.gpu


def make_q(B, sq, hq, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000)
    return (torch.randn(B, sq, hq, D, device="cuda", generator=g) * scale).to(dtype)


def check(lens, sq, hq, hkv, page, dtype, seed=0, causal=False, window=(None, None), softcap=0.0, weights=True, scale=None, qscale=1.0):
    from splitd_flash_attn import split_flash_attn_paged_func

    k, v, table, seqlens, _ = make_cache(lens, page, hkv, dtype, seed)
    q = make_q(len(lens), sq, hq, dtype, seed, qscale)
    w0 = torch.rand(len(lens), max(lens) + 3, device="cuda") if weights else None
    w = w0.clone() if weights else None
    out, lse = split_flash_attn_paged_func(
        q, k, v, table, seqlens, softmax_scale=scale, causal=causal, window_size=window, softcap=softcap, key_weights=w, return_lse=True
    )
    ref, lref, wref, otol, ltol, wtol = attention_ref(q, k, v, table, lens, scale, causal, window, softcap)
    assert out.dtype == dtype and out.shape == q.shape and lse.dtype == torch.float32
    assert_within(out, ref, otol, "out")
    assert_within(lse, lref, ltol, "lse")
    if weights:
        n = wref.shape[1]
        assert_within(w[:, : max(lens)], w0[:, : max(lens)].double() + wref[:, : max(lens)], wtol[:, : max(lens)] + 2.0**-22, "weights")
        for b, length in enumerate(lens):  # slots behind a sequence are left as they were
            assert torch.equal(w[b, length:], w0[b, length:])
    assert_status_ok()


def test_one_sequence_one_tile():
    check([20], 1, 8, 1, 16, torch.bfloat16, weights=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 100, 1000, 4097])
@pytest.mark.parametrize("page", [16, 48])
def test_lengths(length, dtype, page):
    check([length], 1, 8, 1, page, dtype, seed=length)


@pytest.mark.parametrize("heads", [(1, 1), (6, 6), (6, 3), (32, 4), (10, 2), (20, 1), (33, 1), (64, 2), (128, 1)])
@pytest.mark.parametrize("sq", [1, 3])
def test_head_layouts(heads, sq):
    check([130, 77], sq, heads[0], heads[1], 32, torch.bfloat16, seed=heads[0], causal=True)


@pytest.mark.parametrize("page", [1, 3, 7, 16, 100, 256, 1000])
def test_page_sizes(page):
    check([301, 64, 1], 1, 8, 2, page, torch.bfloat16, seed=page)


@pytest.mark.parametrize(
    "lens", [[0], [0, 0], [0, 5, 0, 0, 700, 0], [1] * 40, list(range(70)), [5000, 1, 3, 2500, 40] * 3, [17] * 200]
)
def test_ragged_batches(lens):
    check(lens, 1, 8, 2, 16, torch.bfloat16, seed=len(lens))


@pytest.mark.parametrize("sq", [1, 2, 5, 16, 40])
@pytest.mark.parametrize("mask", ["causal", "none", (20, 0), (0, 0), (7, 3), (None, 2), (30, None), (100000, 0), (2**31 - 1, 2**31 - 1)])
def test_masks_and_several_tokens(sq, mask):
    # lengths below sq: the first rows see nothing under the causal mask
    causal, window = (mask == "causal"), (mask if isinstance(mask, tuple) else (None, None))
    check([90, 3, 41, 0, 33], sq, 8, 2, 16, torch.float16, seed=sq, causal=causal, window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("softcap", [0.0, 15.0, 50.0])
def test_softcap_and_concentrated_rows(dtype, softcap):
    check([700, 33], 2, 32, 4, 64, dtype, seed=9, causal=True, softcap=softcap, qscale=6.0)


@pytest.mark.parametrize("scale", [1e-4, 1.0])
def test_softmax_scale(scale):
    check([300], 1, 8, 1, 64, torch.bfloat16, seed=2, scale=scale)


def test_long_sequence():
    check([40000, 12], 1, 8, 1, 64, torch.bfloat16, seed=4)


def test_keys_of_the_types_lowest_value():
    """Scores of -inf in 32 bits for two whole tiles, then ordinary ones."""
    from splitd_flash_attn import split_flash_attn_paged_func

    lens = [200]
    k, v, table, seqlens, _ = make_cache(lens, 16, 1, torch.bfloat16, 3)
    q = make_q(1, 1, 8, torch.bfloat16, 3).abs()
    j = torch.arange(64, device="cuda")
    k[table[0].long()[j // 16], j % 16] = torch.finfo(torch.bfloat16).min
    out, lse = split_flash_attn_paged_func(q, k, v, table, seqlens, return_lse=True)
    j2 = torch.arange(64, 200, device="cuda")
    kk, vv = k[table[0].long()[j2 // 16], j2 % 16, 0].double(), v[table[0].long()[j2 // 16], j2 % 16, 0].double()
    x = q[0, 0].double() @ kk.T * D**-0.5
    p = torch.softmax(x, 1)
    assert (out[0, 0].double() - p @ vv).abs().max() <= 2.0**-8 * (p @ vv).abs().max() + 1e-3
    assert (lse[0, :, 0].double() - torch.logsumexp(x, 1)).abs().max() <= 1e-4
    # nothing but scores of -inf: like a row without keys
    out, lse = split_flash_attn_paged_func(q, k, v, table, torch.tensor([64], dtype=torch.int32, device="cuda"), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert_status_ok()


def test_nan_and_infinity_of_a_visible_key_reach_the_rows_that_see_it_only():
    from splitd_flash_attn import split_flash_attn_paged_func

    lens = [100, 100]
    k, v, table, seqlens, _ = make_cache(lens, 16, 2, torch.bfloat16, 5)
    q = make_q(2, 1, 8, torch.bfloat16, 5)
    clean = split_flash_attn_paged_func(q, k, v, table, seqlens)
    k[table[0].long()[2], 3, 1, 7] = float("nan")
    out, lse = split_flash_attn_paged_func(q, k, v, table, seqlens, return_lse=True)
    assert torch.isnan(out[0, :, 4:]).all() and torch.isnan(lse[0, 4:]).all()
    assert torch.equal(out[0, :, :4], clean[0, :, :4]) and torch.equal(out[1], clean[1])
    # all keys of a row NaN
    k[:] = float("nan")
    assert torch.isnan(split_flash_attn_paged_func(q, k, v, table, seqlens)).all()
    # values: a NaN stays in its column
    k, v, table, seqlens, _ = make_cache(lens, 16, 2, torch.bfloat16, 5)
    v[table[1].long()[0], 0, 0, 11] = float("inf")
    out = split_flash_attn_paged_func(q, k, v, table, seqlens)
    assert (out[1, :, :4, 11] == float("inf")).all()
    out[1, :, :4, 11] = clean[1, :, :4, 11]
    assert torch.equal(out, clean)
    # slots outside the window are not read
    v[:] = float("nan")
    k2, v2, _, _, _ = make_cache(lens, 16, 2, torch.bfloat16, 5)
    for b in range(2):
        j = torch.arange(90, 100, device="cuda")
        v[table[b].long()[j // 16], j % 16] = v2[table[b].long()[j // 16], j % 16]
    out = split_flash_attn_paged_func(q, k, v, table, seqlens, window_size=(9, 0))
    assert torch.isfinite(out).all()
    assert_status_ok()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,sq", [((8, 1), 2), ((8, 2), 4), ((8, 1), 3), ((8, 1), 4), ((4, 4), 40)])
def test_infinities_and_nan_in_keys_that_only_some_rows_see(dtype, heads, sq):
    """Drafted tokens: the last slots are hidden from the first rows, whose results must not notice what is in them."""
    from splitd_flash_attn import split_flash_attn_paged_func

    lens = [70, 33, sq, 200]
    k, v, table, seqlens, _ = make_cache(lens, 16, heads[1], dtype, 13)
    q = make_q(4, sq, heads[0], dtype, 13)
    for mask in ({"causal": True}, {"window_size": (20, 0)}):
        clean, clean_lse = split_flash_attn_paged_func(q, k, v, table, seqlens, return_lse=True, **mask)
        k2, v2 = k.clone(), v.clone()
        for b, n in enumerate(lens):
            last = table[b, (n - 1) // 16].long(), (n - 1) % 16
            k2[last], v2[last] = float("nan"), float("nan")
        out, lse = split_flash_attn_paged_func(q, k2, v2, table, seqlens, return_lse=True, **mask)
        assert torch.equal(lse[:, :, :-1], clean_lse[:, :, :-1]) and torch.isnan(lse[:, :, -1]).all()
        # a tile with such a value is summed one key at a time: other roundings of the same sum of 32 terms
        seen = torch.isfinite(clean_lse).transpose(1, 2)[:, :-1, :, None]
        diff = (out[:, :-1].double() - clean[:, :-1].double()).abs()
        assert torch.isfinite(out[:, :-1]).all() and torch.isnan(out[:, -1]).all()
        bound = torch.finfo(dtype).eps * clean[:, :-1].double().abs() + 64 * 2.0**-23 * v.abs().nan_to_num(0).amax().double()
        assert (diff <= bound * seen + 0.0).all()
        v2 = v.clone()
        for b, n in enumerate(lens):
            v2[table[b, (n - 1) // 16].long(), (n - 1) % 16, :, 5] = float("inf")
        out = split_flash_attn_paged_func(q, k, v2, table, seqlens, **mask)
        assert torch.isfinite(out[:, :-1]).all() and (out[:, -1, :, 5] == float("inf")).all()
        rest = torch.ones(D, dtype=torch.bool, device="cuda")
        rest[5] = False
        assert torch.isfinite(out[:, -1][..., rest]).all()
    assert_status_ok()


def test_strided_caches_and_queries():
    """Keys and values interleaved in one allocation, heads before rows, a slice of a larger q."""
    from splitd_flash_attn import split_flash_attn_paged_func

    lens = [130, 9]
    k, v, table, seqlens, _ = make_cache(lens, 16, 2, torch.bfloat16, 6)
    big = torch.randn(2, 1, 24, D, device="cuda").to(torch.bfloat16)
    q = big[:, :, 8:16]
    want = split_flash_attn_paged_func(q.contiguous(), k, v, table, seqlens)
    kv = torch.stack((k, v), 1)
    assert torch.equal(split_flash_attn_paged_func(q, kv[:, 0], kv[:, 1], table, seqlens), want)
    kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    assert torch.equal(split_flash_attn_paged_func(q, kt, vt, table, seqlens), want)
    wide = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2][:, : table.shape[1]] = table
    assert torch.equal(split_flash_attn_paged_func(q, k, v, wide[:, ::2], seqlens), want)
    odd = torch.randn(2, 1, 8, D + 1, device="cuda").to(torch.bfloat16)[..., 1:]  # copied: rows at odd addresses
    assert torch.equal(
        split_flash_attn_paged_func(odd, k, v, table, seqlens), split_flash_attn_paged_func(odd.contiguous(), k, v, table, seqlens)
    )


def test_pages_shared_between_sequences():
    from splitd_flash_attn import split_flash_attn_paged_func

    k, v, table, _, _ = make_cache([160], 16, 2, torch.bfloat16, 7)
    q = make_q(1, 1, 8, torch.bfloat16, 7).expand(3, -1, -1, -1)
    lens = [160, 160, 50]
    out = split_flash_attn_paged_func(q, k, v, table.expand(3, -1), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert torch.equal(out[0], out[1])
    ref, _, _, otol, _, _ = attention_ref(q, k, v, table.expand(3, -1), lens)
    assert_within(out, ref, otol, "out")


def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements; the pages in use are its last ones."""
    from splitd_flash_attn import split_flash_attn_paged_func

    lens = [70, 33]
    k, v, table, seqlens, _ = make_cache(lens, 16, 2, torch.bfloat16, 8, spare=0)
    q = make_q(2, 1, 8, torch.bfloat16, 8)
    want = split_flash_attn_paged_func(q, k, v, table, seqlens)
    pages = 2**31 // (16 * 2 * D) + 100
    big = torch.empty(pages, 16, 2, D, dtype=torch.bfloat16, device="cuda")
    big[-k.shape[0] :] = k
    got = split_flash_attn_paged_func(q, big, _at_end(v, pages), torch.where(table >= 0, table + pages - k.shape[0], table), seqlens)
    assert torch.equal(got, want)
    assert_status_ok()


def _at_end(t, pages):
    big = torch.empty(pages, *t.shape[1:], dtype=t.dtype, device=t.device)
    big[-t.shape[0] :] = t
    return big


def test_same_bits_every_time_and_in_a_graph():
    """No atomics on results: the same bits on every call, from a captured graph too, with lengths that grow between
    replays, and with two graphs that share nothing but the cache on two streams."""
    from splitd_flash_attn import split_flash_attn_paged_func

    lens = [3000, 17, 900]
    k, v, table, seqlens, _ = make_cache(lens, 32, 2, torch.bfloat16, 10, fill=0.5)
    q = make_q(3, 1, 8, torch.bfloat16, 10)

    def run(w, lengths):
        return split_flash_attn_paged_func(q, k, v, table, lengths, key_weights=w, return_lse=True)

    w1, w2 = torch.zeros(3, 3000, device="cuda"), torch.zeros(3, 3000, device="cuda")
    a, b = run(w1, seqlens), run(w2, seqlens)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(w1, w2)
    graphs, outs, ws, lengths = [], [], [], []
    for i in range(2):
        ws.append(torch.zeros(3, 3000, device="cuda"))
        lengths.append(seqlens.clone())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(ws[i], lengths[i])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(ws[i], lengths[i]))
        graphs.append(graph)
    lengths[1] -= 5
    ws[0].zero_(), ws[1].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in range(2):
        w = torch.zeros(3, 3000, device="cuda")
        for _ in range(3):
            want = run(w, lengths[i])
        assert torch.equal(outs[i][0], want[0]) and torch.equal(outs[i][1], want[1]) and torch.equal(ws[i], w)
    assert_status_ok()


def test_bad_pages_and_lengths_are_reported_and_not_followed():
    from splitd_flash_attn import split_flash_attn_paged_func
    from splitd_flash_attn.interface import kernel_status, reset_kernel_status

    lens = [100, 60]
    k, v, table, seqlens, _ = make_cache(lens, 16, 2, torch.bfloat16, 11)
    q = make_q(2, 1, 8, torch.bfloat16, 11)
    want = split_flash_attn_paged_func(q, k, v, table, seqlens)
    for bad in (-1, k.shape[0], 2**31 - 1, -(2**31)):
        t = table.clone()
        t[0, 2] = bad
        try:
            out = split_flash_attn_paged_func(q, k, v, t, seqlens)
            assert kernel_status() == 107
            assert torch.equal(out[1], want[1]) and torch.isfinite(out).all()
        finally:
            reset_kernel_status()
    # a length beyond the table's row is cut to it; a negative one counts as 0
    cut = table[:, :3].contiguous()
    try:
        out = split_flash_attn_paged_func(q, k, v, cut, seqlens)
        assert kernel_status() == 108
        assert torch.equal(out, split_flash_attn_paged_func(q, k, v, cut, torch.tensor([48, 48], dtype=torch.int32, device="cuda")))
    finally:
        reset_kernel_status()
    out, lse = split_flash_attn_paged_func(
        q, k, v, table, torch.tensor([-3, -(2**31)], dtype=torch.int32, device="cuda"), return_lse=True
    )
    assert (out == 0).all() and (lse == -math.inf).all()
    w = torch.zeros(2, 50, device="cuda")
    try:
        out = split_flash_attn_paged_func(q, k, v, table, seqlens, key_weights=w)
        assert kernel_status() == 108 and torch.equal(out, want)
        full = torch.zeros(2, 100, device="cuda")
        split_flash_attn_paged_func(q, k, v, table, seqlens, key_weights=full)
        assert torch.equal(w, full[:, :50])
    finally:
        reset_kernel_status()
    assert_status_ok()


def test_empty_calls():
    from splitd_flash_attn import split_flash_attn_paged_func

    k, v, table, seqlens, _ = make_cache([20], 16, 2, torch.bfloat16, 12)
    q = make_q(1, 1, 8, torch.bfloat16, 12)
    assert split_flash_attn_paged_func(q[:0], k, v, table[:0], seqlens[:0]).shape == (0, 1, 8, D)
    assert split_flash_attn_paged_func(q[:, :0], k, v, table, seqlens).shape == (1, 0, 8, D)
    zero = torch.zeros_like(seqlens)
    for kk, tt in ((k[:0], table), (k, table[:, :0])):
        out, lse = split_flash_attn_paged_func(q, kk, kk, tt, zero, return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    w = torch.zeros(1, 0, device="cuda")
    assert torch.isfinite(split_flash_attn_paged_func(q, k, v, table, seqlens, key_weights=w)).all()
    assert_status_ok()
