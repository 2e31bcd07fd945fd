"""GPU: eviction next to what goes on around it: weights that change meanwhile, and decoding before and after."""
import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import D, assert_within, attention_ref, evict_ref, make_cache, rows_of
from test_gpu_paged_cache import freq, some_weights, tokens

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


@pytest.mark.parametrize("lens,keep,width", [([100, 30, 0, 51], 50, 50), ([100, 30, 0, 51], 50, 77), ([20000, 40000], 9000, 20001), ([5], 3, 4000)])
def test_width_of_the_new_weights(lens, keep, width):
    from splitd_flash_attn import split_paged_evict_func

    need = -(-keep // 16)
    k, v, table, seqlens, free = make_cache(lens, 16, 1, torch.bfloat16, 61, spare=need * len(lens), fill=7.0)
    new = free.view(len(lens), need)
    w = some_weights(lens, "plain", 3)
    n, kept, nw = split_paged_evict_func(k, v, table, seqlens, w, new, keep, 1, 2)
    full = torch.full((len(lens), width), float("nan"), device="cuda")
    del full  # the result gets this memory
    n2, kept2, wide = split_paged_evict_func(k, v, table, seqlens, w, new, keep, 1, 2, weights_len=width)
    assert wide.shape == (len(lens), width) and wide.is_contiguous()
    assert torch.equal(n, n2) and torch.equal(kept, kept2) and torch.equal(wide[:, :keep], nw) and (wide[:, keep:] == 0).all()
    assert_status_ok()


@pytest.mark.parametrize("compiled", [False, True])
def test_decode_evict_decode_evict(compiled):
    """The loop of a server: weights are collected, the cache is cut when it has outgrown its budget, and again. Every step
    against attention in 64 bits on what the cache holds, the weights against their sums, every cut against the plain
    selection; the recent slots survive both."""
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func

    hq, hkv, page, dtype = 8, 2, 16, torch.bfloat16
    keep, first, recent, width = 20, 2, 6, 48
    k, v, table, _, free = make_cache([width, width], page, hkv, dtype, 63, spare=6, fill=0.0)
    k.zero_(), v.zero_()
    other = free.view(2, 3).clone()
    f = freq(512)
    seqlens = torch.zeros(2, dtype=torch.int32, device="cuda")
    position = torch.zeros(2, dtype=torch.int64, device="cuda")
    w = torch.zeros(2, width, device="cuda")

    def decode(q, kk, vv, k, v, table, seqlens, position, w):
        qr = split_paged_append_func(q, kk, vv, k, v, table, seqlens, inv_freq=f, positions=position[:, None] - 1)
        return qr, split_flash_attn_paged_func(qr, k, v, table, seqlens, causal=True, key_weights=w)

    def cut(k, v, table, seqlens, w, other):
        return split_paged_evict_func(k, v, table, seqlens, w, other, keep, first, recent, weights_len=w.shape[1])

    if compiled:
        decode, cut = torch.compile(decode, fullgraph=True), torch.compile(cut, fullgraph=True)
    held = [[], []]  # the position of each slot's token, of each sequence
    want_w = torch.zeros(2, width, dtype=torch.float64, device="cuda")
    tol_w = torch.zeros_like(want_w)
    step = 0
    for turn, count in enumerate((30, 25, 9)):
        for _ in range(count):
            q, kk, vv = (tokens((2, 1), h, dtype, 7 * step + i) for i, h in enumerate((hq, hkv, hkv)))
            seqlens, position, step = seqlens + 1, position + 1, step + 1
            qr, out = decode(q, kk, vv, k, v, table, seqlens, position, w)
            for b in range(2):
                held[b].append(step - 1)
            now = seqlens.tolist()
            assert now == [len(h) for h in held]
            ref, _, wr, otol, _, wtol = attention_ref(qr, k, v, table, now, causal=True)
            assert_within(out, ref, otol, f"step {step}")
            want_w[:, : wr.shape[1]] += wr
            tol_w[:, : wr.shape[1]] += wtol + 2.0**-22 * (1 + want_w[:, : wr.shape[1]])
            assert_within(w, want_w, tol_w, "weights")
        if turn == 2:
            break
        n, kept, new_w = cut(k, v, table, seqlens, w, other)
        want = evict_ref(w, now, keep, first, recent)
        for b in range(2):
            assert kept[b].tolist() == want[b] and want[b][-recent:] == list(range(now[b] - recent, now[b]))
            old = rows_of(k, table, b, now[b])[kept[b].long()], rows_of(v, table, b, now[b])[kept[b].long()]
            assert torch.equal(rows_of(k, other, b, keep), old[0]) and torch.equal(rows_of(v, other, b, keep), old[1])
            held[b] = [held[b][j] for j in want[b]]
            assert held[b][-recent:] == list(range(step - recent, step))  # the newest tokens
            for t in (want_w, tol_w):
                t[b] = torch.cat((t[b, kept[b].long()], t.new_zeros(width - keep)))
        seqlens, w = n, new_w
        table, other = other, table
        assert torch.equal(w[:, keep:], torch.zeros_like(w[:, keep:]))
    assert_status_ok()
