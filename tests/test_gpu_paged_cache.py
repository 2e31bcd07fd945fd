"""GPU: append to and eviction from a paged cache, and a decoder's steps with all of its operators together."""
import math

import pytest
import torch

from gpu_utils import assert_status_ok
from paged_utils import D, assert_within, attention_ref, evict_ref, make_cache, rotate_ref, rows_of

pytestmark = pytest.mark.gpu


def freq(r, base=10000.0):
    return torch.pow(torch.tensor(base, dtype=torch.float64, device="cuda"), -torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / max(r, 1))


def tokens(lead, heads, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*lead, heads, D, device="cuda", generator=g).to(dtype)


def check_append(new, held, hq, hkv, page, dtype, packed, r=512, interleaved=False, positions=None, with_q=True, seed=0):
    """new, held: new tokens and old length of each sequence."""
    from splitd_flash_attn import split_paged_append_func

    lens = [a + b for a, b in zip(new, held)]
    k_pages, v_pages, table, seqlens, _ = make_cache(lens, page, hkv, dtype, seed, fill=7.0)
    k0, v0 = k_pages.clone(), v_pages.clone()
    B = len(new)
    lead = (sum(new),) if packed else (B, new[0])
    q, k, v = (tokens(lead, h, dtype, seed + i) for i, h in enumerate((hq, hkv, hkv)))
    cu = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    f = freq(r) if r else None
    pos = None
    if positions:
        pos = torch.randint(0, 100000, lead, device="cuda")
    got = split_paged_append_func(
        q if with_q else None, k, v, k_pages, v_pages, table, seqlens, inv_freq=f, positions=pos,
        cu_seqlens_q=cu if packed else None, interleaved=interleaved, factor=1.5 if r else 1.0,
    )
    assert (got is not None) == with_q
    flat = [t if packed else t.flatten(0, 1) for t in (q, k, v)]
    fgot = got if packed or not with_q else got.flatten(0, 1)
    fpos = None if pos is None else pos.flatten()
    for b in range(B):
        here = slice(sum(new[:b]), sum(new[: b + 1]))
        n = lens[b]
        slots = torch.arange(held[b], n, device="cuda")
        at = (table[b].long()[slots // page], slots % page)
        p = slots if fpos is None else fpos[here]
        for name, x, y in (("q", flat[0][here], fgot[here] if with_q else None), ("k", flat[1][here], k_pages[at])):
            if y is None:
                continue
            ref, tol = rotate_ref(x, p, f if r else freq(0), interleaved, 1.5 if r else 1.0)
            assert_within(y, ref, tol, name)
        assert torch.equal(v_pages[at], flat[2][here])
        k0[at], v0[at] = k_pages[at], v_pages[at]
    assert torch.equal(k_pages, k0) and torch.equal(v_pages, v0)  # everything else is as it was
    assert_status_ok()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(8, 1), (32, 4), (6, 6), (6, 3)])
@pytest.mark.parametrize("page", [16, 48, 1])
def test_append_one_token_per_sequence(dtype, heads, page):
    check_append([1] * 5, [0, 3, 15, 16, 47], *heads, page, dtype, False, seed=heads[0])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("r", [512, 256, 100, 34, 0])
@pytest.mark.parametrize("packed", [False, True])
def test_append_prompts(interleaved, r, packed):
    new = [33, 1, 0, 70, 16] if packed else [19] * 4
    held = [0, 40, 9, 100, 3][: len(new)]
    check_append(new, held, 8, 2, 16, torch.bfloat16, packed, r, interleaved)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("with_q", [False, True])
def test_append_with_positions_and_without_q(packed, with_q):
    check_append([5, 5], [2, 30], 8, 2, 16, torch.float16, packed, positions=True, with_q=with_q)


def test_append_many_sequences():
    check_append([b % 3 for b in range(100)], [b % 7 for b in range(100)], 8, 2, 16, torch.bfloat16, True)


def test_append_long_prompt():
    check_append([3000, 1, 2000], [10, 0, 77], 32, 4, 64, torch.bfloat16, True, 256, True)


def test_append_leaves_padding_rows_alone_and_reports_bad_pages():
    from splitd_flash_attn import split_paged_append_func
    from splitd_flash_attn.interface import cu_seqlens_validation, kernel_status, reset_kernel_status

    lens = [20, 33]
    k_pages, v_pages, table, seqlens, _ = make_cache(lens, 16, 2, torch.bfloat16, 1, fill=7.0)
    k0, v0 = k_pages.clone(), v_pages.clone()
    q, k, v = (tokens((2, 2), h, torch.bfloat16, h) for h in (8, 2, 2))
    # lengths 0 and 1 for two new tokens: both rows of the first and the first row of the second are not stored
    short = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    out = split_paged_append_func(q, k, v, k_pages, v_pages, table, short, inv_freq=freq(512))
    assert torch.isfinite(out).all()
    row = (table[1, 0].long(), 0)
    assert torch.equal(k_pages[row], k[1, 1]) and torch.equal(v_pages[row], v[1, 1])
    k_pages[row], v_pages[row] = k0[row], v0[row]
    assert torch.equal(k_pages, k0) and torch.equal(v_pages, v0)
    assert kernel_status() == 0
    for bad, code in ((-1, 107), (k_pages.shape[0], 107)):
        t = table.clone()
        t[0, 1] = bad
        try:
            split_paged_append_func(q, k, v, k_pages, v_pages, t, seqlens)
            assert kernel_status() == code
        finally:
            reset_kernel_status()
        assert torch.equal(k_pages[table[0, 1].long()], k0[table[0, 1].long()])
        at = (table[1].long()[torch.tensor([1, 2], device="cuda")], torch.tensor([15, 0], device="cuda"))
        assert torch.equal(k_pages[at], k[1])
    try:
        split_paged_append_func(q, k, v, k_pages, v_pages, table[:, :1], seqlens)
        assert kernel_status() == 108
    finally:
        reset_kernel_status()
    # packed tokens behind the last sequence are not stored (value checks off: they would refuse the call)
    k_pages.copy_(k0), v_pages.copy_(v0)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    with cu_seqlens_validation(False):
        split_paged_append_func(None, k.flatten(0, 1), v.flatten(0, 1), k_pages, v_pages, table, seqlens, cu_seqlens_q=cu)
    last = [(table[b, (lens[b] - 1) // 16].long(), (lens[b] - 1) % 16) for b in range(2)]
    for b in range(2):
        assert torch.equal(k_pages[last[b]], k.flatten(0, 1)[b])
        k_pages[last[b]], v_pages[last[b]] = k0[last[b]], v0[last[b]]
    assert torch.equal(k_pages, k0) and torch.equal(v_pages, v0)
    assert_status_ok()


def test_append_strided_tokens_and_caches():
    from splitd_flash_attn import split_paged_append_func

    lens = [20, 33]
    k_pages, v_pages, table, seqlens, _ = make_cache(lens, 16, 2, torch.bfloat16, 1, fill=7.0)
    qkv = tokens((2, 3), 12, torch.bfloat16, 2)
    q, k, v = qkv[:, :, :8], qkv[:, :, 8:10], qkv[:, :, 10:]
    kv = torch.stack((k_pages, v_pages), 1)
    a = split_paged_append_func(q, k, v, kv[:, 0], kv[:, 1], table, seqlens, inv_freq=freq(512))
    b = split_paged_append_func(q.contiguous(), k.contiguous(), v.contiguous(), k_pages, v_pages, table, seqlens, inv_freq=freq(512))
    assert torch.equal(a, b) and torch.equal(kv[:, 0], k_pages) and torch.equal(kv[:, 1], v_pages)


def test_append_refuses_one_memory_for_keys_and_values_and_misaligned_caches():
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func

    k_pages, v_pages, table, seqlens, _ = make_cache([20], 16, 2, torch.bfloat16, 1, fill=7.0)
    k = tokens((1, 1), 2, torch.bfloat16, 2)
    with pytest.raises(ValueError, match="same memory"):
        split_paged_append_func(None, k, k, k_pages, k_pages, table, seqlens)
    odd = torch.zeros(k_pages.numel() + 4, dtype=torch.bfloat16, device="cuda")[4:].view(k_pages.shape)
    with pytest.raises(ValueError, match="16-byte"):
        split_paged_append_func(None, k, k, odd, v_pages, table, seqlens)
    with pytest.raises(ValueError, match="16-byte"):
        split_flash_attn_paged_func(k, k_pages, odd, table, seqlens)
    # reading keys and values from one memory is fine, as in the dense attention
    a = split_flash_attn_paged_func(k, k_pages, k_pages, table, seqlens)
    assert torch.equal(a, split_flash_attn_paged_func(k, k_pages, k_pages.clone(), table, seqlens))


def test_misaligned_contiguous_tokens_are_copied():
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_rotary_func

    k_pages, v_pages, table, seqlens, _ = make_cache([20, 5], 16, 2, torch.bfloat16, 1, fill=7.0)
    q, k = tokens((2, 1), 8, torch.bfloat16, 2), tokens((2, 1), 2, torch.bfloat16, 3)

    def shifted(t):
        s = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        s.copy_(t)
        assert s.is_contiguous() and s.data_ptr() % 16
        return s

    caches = [(k_pages.clone(), v_pages.clone()) for _ in range(2)]
    a = split_paged_append_func(q, k, k, *caches[0], table, seqlens, inv_freq=freq(512))
    b = split_paged_append_func(shifted(q), shifted(k), shifted(k), *caches[1], table, seqlens, inv_freq=freq(512))
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(*caches))
    assert torch.equal(split_flash_attn_paged_func(q, *caches[0], table, seqlens), split_flash_attn_paged_func(shifted(q), *caches[0], table, seqlens))
    pos = torch.arange(1, device="cuda")
    assert torch.equal(split_rotary_func(q, k, pos, freq(512))[1], split_rotary_func(q, shifted(k), pos, freq(512))[1])


def test_under_inference_mode_and_after_it():
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func
    from splitd_flash_attn import interface
    from splitd_flash_attn.interface import kernel_status, reset_kernel_status

    k_pages, v_pages, table, seqlens, _ = make_cache([21, 5], 16, 1, torch.bfloat16, 1, fill=7.0)
    q, k = tokens((2, 1), 5, torch.bfloat16, 2), tokens((2, 1), 1, torch.bfloat16, 3)
    saved = interface._status_flags.copy()
    interface._status_flags.clear()
    try:
        with torch.inference_mode():
            qr = split_paged_append_func(q, k, k, k_pages, v_pages, table, seqlens, inv_freq=freq(512))
            a = split_flash_attn_paged_func(qr, k_pages, v_pages, table, seqlens)
        qr = split_paged_append_func(q, k, k, k_pages, v_pages, table, seqlens, inv_freq=freq(512))
        b = split_flash_attn_paged_func(qr, k_pages, v_pages, table, seqlens)
        assert torch.equal(a, b) and not b.is_inference()
        reset_kernel_status()
        assert kernel_status() == 0
    finally:
        interface._status_flags.update(saved)


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------


def check_evict(lens, keep, first, recent, hkv, page, dtype, weights, seed=0):
    from splitd_flash_attn import split_paged_evict_func

    need = -(-keep // page)
    k_pages, v_pages, table, seqlens, free = make_cache(lens, page, hkv, dtype, seed, spare=need * len(lens) + 1, fill=7.0)
    new_table = free[: need * len(lens)].view(len(lens), need)
    k0, v0 = k_pages.clone(), v_pages.clone()
    n_out, kept, w_out = split_paged_evict_func(k_pages, v_pages, table, seqlens, weights, new_table, keep, first, recent)
    want = evict_ref(weights, lens, keep, first, recent)
    for b, slots in enumerate(want):
        m = len(slots)
        assert int(n_out[b]) == m
        assert kept[b].tolist() == slots + [-1] * (keep - m)
        s = torch.tensor(slots, device="cuda", dtype=torch.long)
        assert torch.equal(torch.nan_to_num(w_out[b, :m]), torch.nan_to_num(weights[b, s])) and (w_out[b, m:] == 0).all()
        i = torch.arange(m, device="cuda")
        to, frm = (new_table[b].long()[i // page], i % page), (table[b].long()[s // page], s % page)
        assert torch.equal(k_pages[to], k0[frm]) and torch.equal(v_pages[to], v0[frm])
        k_pages[to], v_pages[to] = k0[to], v0[to]
    assert torch.equal(k_pages, k0) and torch.equal(v_pages, v0)  # nothing else was written
    assert_status_ok()


def some_weights(lens, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.rand(len(lens), max(max(lens), 1) + 5, device="cuda", generator=g)
    if kind == "ties":
        w = (w * 4).floor()
    elif kind == "zeros":
        w = torch.zeros_like(w)
    elif kind == "signs":
        w = (w - 0.5) * 1e3
        w[:, ::3] = -0.0
        w[:, 1::3] = 0.0
    elif kind == "special":
        w[:, ::5] = float("nan")
        w[:, 1::7] = float("inf")
        w[:, 2::7] = -float("inf")
        w[:, 3::4] = 1e-42
    return w


@pytest.mark.parametrize("kind", ["plain", "ties", "zeros", "signs", "special"])
@pytest.mark.parametrize("lens,keep,first,recent", [
    ([100], 50, 0, 0), ([100], 50, 4, 16), ([100, 30, 51, 50, 49, 0, 1], 50, 4, 46), ([64], 1, 0, 0), ([64], 1, 1, 0), ([64], 1, 0, 1),
    ([5000, 700, 4100], 1000, 3, 100), ([9], 9, 4, 5), ([3, 2], 9, 4, 5),
])
def test_evict(kind, lens, keep, first, recent):
    check_evict(lens, keep, first, recent, 2, 16, torch.bfloat16, some_weights(lens, kind, keep))


@pytest.mark.parametrize("hkv,page,dtype", [(1, 1, torch.float16), (4, 48, torch.bfloat16), (6, 100, torch.float16), (9, 64, torch.bfloat16)])
def test_evict_layouts(hkv, page, dtype):
    check_evict([333, 90], 77, 2, 9, hkv, page, dtype, some_weights([333, 90], "ties"))


def test_evict_long():
    lens = [70000, 20]
    check_evict(lens, 4001, 16, 300, 1, 64, torch.bfloat16, some_weights(lens, "plain"))


@pytest.mark.parametrize("kind", ["plain", "ties"])
def test_evict_longer_than_the_keys_in_shared_memory(kind):
    """More than 8 x 49152 slots; page table entries all name the same few pages (reading shared pages is fine)."""
    from splitd_flash_attn import split_paged_evict_func

    n, keep = 800001, 1003
    k = torch.randn(10, 1000, 1, D, device="cuda").to(torch.bfloat16)
    v = torch.randn(10, 1000, 1, D, device="cuda").to(torch.bfloat16)
    table = (torch.arange(801, device="cuda", dtype=torch.int32) % 8)[None]
    new = torch.tensor([[8, 9]], device="cuda", dtype=torch.int32)
    w = some_weights([n], kind, 5)
    m, kept, nw = split_paged_evict_func(k, v, table, torch.tensor([n], device="cuda", dtype=torch.int32), w, new, keep, 1, 2)
    s = torch.tensor(evict_ref(w, [n], keep, 1, 2)[0], device="cuda")
    assert int(m) == keep and torch.equal(kept[0].long(), s) and torch.equal(nw[0], w[0, s])
    flat = k.view(-1, D)
    assert torch.equal(flat[8000 : 8000 + keep], flat[s // 1000 % 8 * 1000 + s % 1000])
    assert_status_ok()


def test_evict_bad_pages_and_lengths():
    from splitd_flash_attn import split_paged_evict_func
    from splitd_flash_attn.interface import kernel_status, reset_kernel_status

    lens = [60, 40]
    k, v, table, seqlens, free = make_cache(lens, 16, 2, torch.bfloat16, 3, spare=6, fill=7.0)
    new = free[:4].view(2, 2)
    w = some_weights(lens, "plain")
    k0 = k.clone()
    for which in (0, 1):
        t, nt = table.clone(), new.clone()
        (t if which == 0 else nt)[0, 0] = k.shape[0]
        try:
            split_paged_evict_func(k, v, t, seqlens, w, nt, 30, 4, 4)
            assert kernel_status() == 107
        finally:
            reset_kernel_status()
    k.copy_(k0)
    try:  # weights for 50 slots only: a longer sequence is cut to them
        n, kept, _ = split_paged_evict_func(k, v, table, seqlens, w[:, :50], new, 30, 4, 4)
        assert kernel_status() == 108 and n.tolist() == [30, 30]
        assert kept.tolist() == evict_ref(w, [50, 40], 30, 4, 4)
    finally:
        reset_kernel_status()
    n, kept, nw = split_paged_evict_func(k, v, table, torch.tensor([-5, 0], dtype=torch.int32, device="cuda"), w, new, 30, 4, 4)
    assert n.tolist() == [0, 0] and (kept == -1).all() and (nw == 0).all()
    n, kept, nw = split_paged_evict_func(k, v, table[:0], seqlens[:0], w[:0], new[:0], 30)
    assert n.shape == (0,) and kept.shape == (0, 30) and nw.shape == (0, 30)
    assert_status_ok()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


def _decode(steps, k_pages, v_pages, table, seqlens, f, qs, ks, vs, w, capture=False):
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func

    q, k, v = qs[0].clone(), ks[0].clone(), vs[0].clone()

    def step():
        seqlens.add_(1)
        qr = split_paged_append_func(q, k, v, k_pages, v_pages, table, seqlens, inv_freq=f)
        return split_flash_attn_paged_func(qr, k_pages, v_pages, table, seqlens, causal=True, key_weights=w)

    outs = []
    if capture:
        state = [t.clone() for t in (k_pages, v_pages, seqlens, w)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for t, s in zip((k_pages, v_pages, seqlens, w), state):
            t.copy_(s)
    for i in range(steps):
        q.copy_(qs[i]), k.copy_(ks[i]), v.copy_(vs[i])
        if capture:
            graph.replay()
            outs.append(out.clone())
        else:
            outs.append(step())
    return outs


def test_prompt_decode_evict_decode():
    """A prompt goes in, tokens are decoded one by one, the cache is cut, decoding goes on: against attention in 64 bits on
    what the cache should hold; and the decode loop captured as a graph gives the same bits."""
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func

    hq, hkv, page, dtype, steps = 8, 2, 16, torch.bfloat16, 6
    prompt = [37, 5, 80]
    total = [n + steps for n in prompt]
    k_pages, v_pages, table, _, free = make_cache(total, page, hkv, dtype, 20, spare=12)
    k_pages.fill_(float("nan")), v_pages.fill_(float("nan"))
    f = freq(512)
    q0, k0, v0 = (tokens((sum(prompt),), h, dtype, 40 + i) for i, h in enumerate((hq, hkv, hkv)))
    cu = torch.tensor([0] + prompt, device="cuda").cumsum(0).to(torch.int32)
    seqlens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    split_paged_append_func(q0, k0, v0, k_pages, v_pages, table, seqlens, inv_freq=f, cu_seqlens_q=cu)
    qs, ks, vs = (tokens((steps, 3, 1), h, dtype, 50 + i) for i, h in enumerate((hq, hkv, hkv)))
    w = torch.zeros(3, max(total), device="cuda")
    state = [t.clone() for t in (k_pages, v_pages, seqlens, w)]
    outs = _decode(steps, k_pages, v_pages, table, seqlens, f, qs, ks, vs, w)
    again = [t.clone() for t in state]
    outs_g = _decode(steps, again[0], again[1], table, again[2], f, qs, ks, vs, again[3], capture=True)
    assert all(torch.equal(a, b) for a, b in zip(outs, outs_g)) and torch.equal(w, again[3])
    assert seqlens.tolist() == total
    want_w, wtol_sum = torch.zeros_like(w, dtype=torch.float64), torch.zeros_like(w, dtype=torch.float64)
    for i in range(steps):
        lens = [n + i + 1 for n in prompt]
        pos = torch.tensor(lens, device="cuda")[:, None] - 1
        # the rotated query as the append rounds it: its own test holds it to the 64-bit rotation
        from splitd_flash_attn import split_rotary_func

        qr, _ = split_rotary_func(qs[i], None, pos, f)
        ref, _, wr, otol, _, wtol = attention_ref(qr, k_pages, v_pages, table, lens, causal=True)
        assert_within(outs[i], ref, otol, f"step {i}")
        want_w[:, : wr.shape[1]] += wr
        wtol_sum[:, : wr.shape[1]] += wtol + 2.0**-22
    assert_within(w, want_w, wtol_sum, "weights")
    # cut to 20 slots and go on
    new_table = free[:6].view(3, 2)
    n, kept, nw = split_paged_evict_func(k_pages, v_pages, table, seqlens, w, new_table, 20, 2, 4)
    assert n.tolist() == [min(20, x) for x in total]
    assert kept[0].tolist() == evict_ref(w, total, 20, 2, 4)[0]
    table2 = torch.cat((new_table, free[6:9].view(3, 1)), 1)
    n2 = n + 1
    pos = torch.tensor(total, device="cuda")[:, None]
    qr = split_paged_append_func(qs[0], ks[0], vs[0], k_pages, v_pages, table2, n2, inv_freq=f, positions=pos)
    w2 = torch.zeros(3, 21, device="cuda")
    w2[:, :20] = nw
    out = split_flash_attn_paged_func(qr, k_pages, v_pages, table2, n2, causal=True, key_weights=w2)
    ref, _, wr, otol, _, wtol = attention_ref(qr, k_pages, v_pages, table2, n2.tolist(), causal=True)
    assert_within(out, ref, otol, "after eviction")
    for b in range(3):
        m = int(n[b])
        old = rows_of(k_pages, table, b, total[b])[kept[b, :m].long()]
        assert torch.equal(rows_of(k_pages, table2, b, m), old)
    assert_status_ok()


def test_decode_step_compiles_without_a_break():
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func

    lens = [40, 21]
    k, v, table, seqlens, free = make_cache(lens, 16, 2, torch.bfloat16, 21, spare=4, fill=0.0)
    q1, k1, v1 = (tokens((2, 1), h, torch.bfloat16, 60 + h) for h in (8, 2, 2))
    f = freq(512)
    new_table = free[:4].view(2, 2)

    def step(q, kk, vv, kp, vp, w):
        qr = split_paged_append_func(q, kk, vv, kp, vp, table, seqlens, inv_freq=f)
        out, lse = split_flash_attn_paged_func(qr, kp, vp, table, seqlens, causal=True, key_weights=w, return_lse=True)
        return (out * 1.0, lse) + split_paged_evict_func(kp, vp, table, seqlens, w, new_table, 24, 2, 2)

    res = []
    for fn in (step, torch.compile(step, fullgraph=True)):
        kp, vp, w = k.clone(), v.clone(), torch.zeros(2, 40, device="cuda")
        res.append((*fn(q1, k1, v1, kp, vp, w), kp, vp, w))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    assert_status_ok()


def test_on_a_stream_of_its_own():
    from splitd_flash_attn import split_flash_attn_paged_func, split_paged_append_func, split_paged_evict_func

    lens = [3000, 21]
    k, v, table, seqlens, free = make_cache(lens, 16, 2, torch.bfloat16, 22, spare=80, fill=0.0)
    q1, k1, v1 = (tokens((2, 1), h, torch.bfloat16, 60 + h) for h in (8, 2, 2))
    f = freq(512)
    new_table = free[:74].view(2, 37)

    def step(kp, vp, w):
        qr = split_paged_append_func(q1, k1, v1, kp, vp, table, seqlens, inv_freq=f)
        out = split_flash_attn_paged_func(qr, kp, vp, table, seqlens, key_weights=w)
        return (out, kp, vp, w) + split_paged_evict_func(kp, vp, table, seqlens, w, new_table, 590)

    want = step(k.clone(), v.clone(), torch.zeros(2, 3000, device="cuda"))
    args = [(k.clone(), v.clone(), torch.zeros(2, 3000, device="cuda")) for _ in range(3)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for s, a in zip(streams, args):
        with torch.cuda.stream(s):
            got.append(step(*a))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(want, g))
    assert_status_ok()


def test_custom_ops_keep_their_schemas():
    """What torch checks of a custom op: aliasing and mutation as declared, fake kernels, autograd, dynamic shapes."""
    ops = torch.ops.splitd_flash_attn
    k, v, table, seqlens, free = make_cache([40, 21], 16, 2, torch.bfloat16, 23, spare=4, fill=0.0)
    q, kk = tokens((2, 1), 8, torch.bfloat16, 1), tokens((2, 1), 2, torch.bfloat16, 2)
    w, f, none, pos = torch.rand(2, 40, device="cuda"), freq(512), -(2**31), torch.arange(1, device="cuda")
    for op, args in (
        (ops.paged_attn, (q, k, v, table, seqlens, w, 0.05, True, none, none, 0.0)),
        (ops.paged_attn, (q, k, v, table, seqlens, None, 0.05, False, 5, 0, 20.0)),
        (ops.paged_append, (q, kk, kk, k, v, table, seqlens, f, None, None, False, 1.0)),
        (ops.paged_append, (None, kk, kk, k, v, table, seqlens, None, None, None, False, 1.0)),
        (ops.paged_evict, (k, v, table, seqlens, w, free[:4].view(2, 2), 20, 2, 2)),
        (ops.rotary, (q.clone().requires_grad_(), kk.clone().requires_grad_(), pos, f, False, 1.0, False)),
        (ops.rotary, (None, kk, pos, f, True, 1.0, True)),
    ):
        torch.library.opcheck(op.default, args)
    assert_status_ok()
