"""The operators around a cache of head_dim-512 keys and values, as they are measured: rotary positions (forward and
backward), the append of new tokens to a paged cache, attention of a few new tokens over the paged cache, and the
eviction of keys by their accumulated attention weight.

``run`` computes a case in its plain form (elementary torch operations in 32 bits or more) or, where ``own`` is
true, through the package's public functions. Layouts: tokens (batch, tokens, heads, 512) or packed
(tokens, heads, 512); cache pages (pages, page_size, kv_heads, 512); page_table (batch, pages per sequence) int32.
"""
import math
import os
import sys

import torch

own = False

D = 512
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

# Head layouts of this repository's tests and benchmark: 32:4 of the layer it is benchmarked on, 8:1 (one KV head),
# 8:2, 6:3 and the ungrouped ones.
HEADS = ((32, 4), (8, 1), (8, 2), (6, 3), (6, 6), (4, 4))


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemm4-attention-kernels_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import splitd_flash_attn

    return splitd_flash_attn


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def _attention(name, batch, sq, length, hq, hkv, page, dtype="bf16", ragged=True, window=-1, softcap=0.0, weights=False):
    return {"name": name, "op": "attention", "batch": batch, "sq": sq, "length": length, "hq": hq, "hkv": hkv, "page": page,
            "dtype": dtype, "ragged": ragged, "window": window, "softcap": softcap, "weights": weights}


def _append(name, batch, tokens, length, hq, hkv, page, dtype="bf16", packed=False, rotary=D, interleaved=False):
    return {"name": name, "op": "append", "batch": batch, "tokens": tokens, "length": length, "hq": hq, "hkv": hkv, "page": page,
            "dtype": dtype, "packed": packed, "rotary": rotary, "interleaved": interleaved}


def _rotary(name, batch, seqlen, hq, hkv, dtype="bf16", rotary=D, interleaved=False, start=0, stretch=1.0):
    return {"name": name, "op": "rotary", "batch": batch, "seqlen": seqlen, "hq": hq, "hkv": hkv, "dtype": dtype, "rotary": rotary,
            "interleaved": interleaved, "start": start, "stretch": stretch}


def _evict(name, batch, length, keep, first, recent, hkv, page, dtype="bf16", ragged=True):
    return {"name": name, "op": "evict", "batch": batch, "length": length, "keep": keep, "first": first, "recent": recent, "hkv": hkv,
            "page": page, "dtype": dtype, "ragged": ragged}


def listed():
    return [
        # one chat turn at its beginning: one sequence, a short cache, one KV head; latency is what counts
        _attention("attention 1 x 1000", 1, 1, 1000, 8, 1, 16, ragged=False),
        # one user far into a long document: the split over the cache's length is all the parallelism there is
        _attention("attention 1 x 131072", 1, 1, 131072, 32, 4, 64, ragged=False),
        # a server's ordinary decode step, sequences of every age
        _attention("attention 32 x 8192", 32, 1, 8192, 32, 4, 64),
        # four drafted tokens verified at once, capped scores in a sliding window, pages that no tile divides
        _attention("attention draft of 4, window", 8, 4, 20011, 32, 4, 48, "fp16", window=8191, softcap=30.0),
        # a decode step that also keeps score of which keys are looked at, for the eviction below
        _attention("attention with weights", 8, 1, 16384, 32, 4, 64, weights=True),
        # a decode step's new tokens go into the cache: 64 sequences, a token each
        _append("append 64 x 1", 64, 1, 5000, 32, 4, 64),
        # prompts of different lengths, packed, behind what their sequences hold already; half the head rotated in pairs
        _append("append packed prompts", 6, 4096, 4500, 32, 4, 48, packed=True, rotary=256, interleaved=True),
        # a short odd prompt, a quarter of the head rotated
        _rotary("rotary 2 x 113", 2, 113, 6, 3, "fp16", rotary=128, interleaved=True),
        # the layer's training step of 16384 tokens, positions of a stretched long context
        _rotary("rotary 2 x 8192", 2, 8192, 32, 4, start=1000000, stretch=8.0),
        # a short cache is halved
        _evict("evict 1 x 1000", 1, 1000, 500, 4, 64, 1, 16, ragged=False),
        # sequences that outgrew their budget, all at once
        _evict("evict 8 x 16384", 8, 16384, 4096, 4, 512, 4, 64),
        # one long document cut to an odd budget
        _evict("evict 1 x 131072", 1, 131072, 20000, 16, 1000, 4, 100, ragged=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "append", "rotary", "evict"))
    hq, hkv = rng.choice(HEADS)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    page = rng.choice((16, 32, 48, 64, 100, 128, 256))
    rotary = rng.choice((D, D, 256, 128, 64, 2 * rng.randint(1, 255)))
    interleaved = rng.random() < 0.5
    if op == "attention":
        batch, sq, length = _log(rng, 1, 64), _log(rng, 1, 8), _log(rng, 1, 131072)
        length = min(length, 32 * 8192 * 2 // (batch * hkv))
        window = rng.choice((-1, -1, _log(rng, 1, 16384)))
        c = _attention("", batch, sq, length, hq, hkv, page, dtype, True, window, rng.choice((0.0, 0.0, 15.0, 50.0)), rng.random() < 0.3)
    elif op == "append":
        batch, tokens = _log(rng, 1, 64), _log(rng, 1, 4096)
        tokens = min(tokens, max(1, 16384 // batch))
        c = _append("", batch, tokens, tokens + _log(rng, 1, 4096), hq, hkv, page, dtype, rng.random() < 0.5, rotary, interleaved)
    elif op == "rotary":
        batch, seqlen = _log(rng, 1, 8), _log(rng, 1, 16384)
        seqlen = min(seqlen, 16384 // batch)
        c = _rotary("", batch, seqlen, hq, hkv, dtype, rotary, interleaved, _log(rng, 1, 1000000), rng.choice((1.0, 4.0, 8.0)))
    else:
        batch, length = _log(rng, 1, 16), _log(rng, 64, 131072)
        length = min(length, 131072 * 4 // (batch * hkv))
        keep = max(8, int(length * rng.uniform(0.05, 0.9)))
        c = _evict("", batch, length, keep, rng.randint(0, 4), rng.randint(0, keep // 4), hkv, page, dtype, True)
    del c["name"]
    return c


def _lengths(n, longest, ragged):
    """Lengths between a quarter of the longest and the longest, the first the longest."""
    if not ragged:
        return [longest] * n
    return [max(1, longest - (longest * 3 // 4) * (b * 617 % 1000) // 1000) for b in range(n)]


def _tokens(case):
    """New tokens of each sequence of an append."""
    return _lengths(case["batch"], case["tokens"], case["packed"])


def work(case):
    h = D * 2
    if case["op"] == "attention":
        lengths = _lengths(case["batch"], case["length"], case["ragged"])
        seen = [n if case["window"] < 0 else min(n, case["window"] + case["sq"]) for n in lengths]
        rows = case["sq"] * case["hq"]
        q = case["batch"] * rows * (2 * h + 4)
        extra = 8 * sum(seen) if case["weights"] else 0
        return {"bytes": sum(seen) * case["hkv"] * 2 * h + q + extra, "flops": 4 * D * rows * sum(seen)}
    if case["op"] == "append":
        t = sum(_tokens(case))
        return {"bytes": t * (2 * case["hq"] + 4 * case["hkv"]) * h, "flops": 3 * t * case["rotary"] * (case["hq"] + case["hkv"])}
    if case["op"] == "rotary":
        n = case["batch"] * case["seqlen"] * (case["hq"] + case["hkv"])
        return {"bytes": 4 * n * h, "flops": 6 * n * case["rotary"]}
    lengths = _lengths(case["batch"], case["length"], case["ragged"])
    kept = sum(min(n, case["keep"]) for n in lengths)
    return {"bytes": kept * case["hkv"] * 4 * h + sum(lengths) * 4 + kept * 8, "flops": sum(lengths)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _cache(g, lengths, page, hkv, dtype, spare=0):
    """Pages in the order in which a server's allocator gives them out after a while: any. Unused entries are 0."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    k = torch.randn(pages, page, hkv, D, device="cuda", dtype=dtype, generator=g)
    v = torch.randn(pages, page, hkv, D, device="cuda", dtype=dtype, generator=g)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    width = max(need)
    first = torch.tensor([0] + need[:-1], device="cuda").cumsum(0)
    at = first[:, None] + torch.arange(width, device="cuda")[None]
    inside = torch.arange(width, device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(inside, order[at.clamp(max=pages - 1)], torch.zeros((), dtype=torch.int32, device="cuda"))
    return k, v, table.contiguous(), order[sum(need):]


def _frequencies(rotary, stretch=1.0):
    i = torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda")
    return torch.pow(torch.tensor(1000000.0, dtype=torch.float64, device="cuda"), -i / rotary) / stretch


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=g).mul_(scale).to(dtype)

    s = {"case": case}
    if case["op"] == "attention":
        lengths = _lengths(case["batch"], case["length"], case["ragged"])
        s["k_pages"], s["v_pages"], s["table"], _ = _cache(g, lengths, case["page"], case["hkv"], dtype, spare=3)
        s["seqlens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        # scores of a standard deviation of 2: a few keys carry most of a row
        s["q"] = normal(case["batch"], case["sq"], case["hq"], D, scale=2.0)
        if case["weights"]:
            s["weights"] = torch.rand(case["batch"], max(lengths), device="cuda", generator=g)
    elif case["op"] == "append":
        new = _tokens(case)
        held = _lengths(case["batch"], case["length"] - case["tokens"], True)
        lengths = [a + b for a, b in zip(new, held)]
        s["k_pages"], s["v_pages"], s["table"], _ = _cache(g, lengths, case["page"], case["hkv"], dtype)
        s["seqlens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        lead = (sum(new),) if case["packed"] else (case["batch"], case["tokens"])
        s["q"], s["k"], s["v"] = normal(*lead, case["hq"], D), normal(*lead, case["hkv"], D), normal(*lead, case["hkv"], D)
        s["inv_freq"] = _frequencies(case["rotary"])
        s["cu"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    elif case["op"] == "rotary":
        lead = (case["batch"], case["seqlen"])
        s["q"], s["k"] = normal(*lead, case["hq"], D).requires_grad_(), normal(*lead, case["hkv"], D).requires_grad_()
        s["dq"], s["dk"] = normal(*lead, case["hq"], D, scale=0.01), normal(*lead, case["hkv"], D, scale=0.01)
        s["inv_freq"] = _frequencies(case["rotary"], case["stretch"])
        begin = torch.randint(case["start"], case["start"] + 1000, (case["batch"], 1), device="cuda", generator=g)
        s["positions"] = (begin + torch.arange(case["seqlen"], device="cuda")).to(torch.int32)
    else:
        lengths = _lengths(case["batch"], case["length"], case["ragged"])
        kept = [min(n, case["keep"]) for n in lengths]
        need = -(-max(kept) // case["page"])
        k, v, table, free = _cache(g, lengths, case["page"], case["hkv"], dtype, spare=need * len(lengths))
        s["k_pages"], s["v_pages"], s["table"], s["new_table"] = k, v, table, free.view(len(lengths), need).contiguous()
        s["seqlens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        # sums of softmax weights: most small, a few large, and keys that no row has looked at
        w = torch.rand(case["batch"], max(lengths), device="cuda", generator=g).pow_(4).mul_(16.0)
        s["weights"] = torch.where(w < 0.1, torch.zeros_like(w), w)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _slots(table, page, count):
    """Row of the flattened cache (pages * page_size) that holds each of the first `count` keys of a sequence."""
    j = torch.arange(count, device=table.device)
    return table.long()[:, j // page] * page + j % page


def _rotate(x, positions, inv_freq, interleaved, backward=False):
    """positions: the leading dimensions of x without its heads."""
    r = 2 * inv_freq.numel()
    angle = positions.double()[..., None, None] * inv_freq
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if backward:
        sin = -sin
    head, rest = x.detach()[..., :r].float(), x.detach()[..., r:].float()
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., : r // 2], head[..., r // 2 :])
    y1, y2 = a * cos - b * sin, a * sin + b * cos
    head = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((head, rest), -1).to(x.dtype)


def _plain_attention(s):
    case, q = s["case"], s["q"]
    b, sq, hq, hkv = case["batch"], case["sq"], case["hq"], case["hkv"]
    n = s["table"].shape[1] * case["page"]
    rows = _slots(s["table"], case["page"], n)
    k = s["k_pages"].view(-1, hkv, D)[rows].float().transpose(1, 2)
    v = s["v_pages"].view(-1, hkv, D)[rows].float().transpose(1, 2)
    qg = q.float().view(b, sq, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, D)
    scores = (qg @ k.transpose(-1, -2)).view(b, hkv, hq // hkv, sq, n) * D**-0.5
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    j = torch.arange(n, device=q.device)
    last = (s["seqlens"][:, None] - sq + torch.arange(sq, device=q.device))[:, None, None, :, None]
    seen = j <= last
    if case["window"] >= 0:
        seen = seen & (j >= last - case["window"])
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    out = (p.view(b, hkv, -1, n) @ v).view(b, hkv, hq // hkv, sq, D).permute(0, 3, 1, 2, 4).reshape(b, sq, hq, D).to(q.dtype)
    lse = (top + torch.log(total)).view(b, hq, sq)
    if not case["weights"]:
        return out, lse
    w = s["weights"]
    w += p.sum((1, 2, 3))[:, : w.shape[1]]
    return out, lse, w


def _plain_append(s):
    case, hkv, q = s["case"], s["case"]["hkv"], s["q"]
    cu = s["cu"].long()
    t = torch.arange(s["k"].shape[0] if case["packed"] else case["batch"] * case["tokens"], device=q.device)
    seq = torch.searchsorted(cu, t, right=True) - 1
    slot = s["seqlens"].long()[seq] - cu[seq + 1] + t
    row = s["table"].long()[seq, slot // case["page"]] * case["page"] + slot % case["page"]
    slot = slot if case["packed"] else slot.view(case["batch"], case["tokens"])
    out = _rotate(q, slot, s["inv_freq"], case["interleaved"])
    s["k_pages"].view(-1, hkv, D)[row] = _rotate(s["k"], slot, s["inv_freq"], case["interleaved"]).view(-1, hkv, D)
    s["v_pages"].view(-1, hkv, D)[row] = s["v"].view(-1, hkv, D)
    return out, s["k_pages"], s["v_pages"]


def _plain_rotary(s):
    f, i, p = s["inv_freq"], s["case"]["interleaved"], s["positions"]
    return (_rotate(s["q"], p, f, i), _rotate(s["k"], p, f, i), _rotate(s["dq"], p, f, i, True), _rotate(s["dk"], p, f, i, True))


def _plain_evict(s):
    case, w, n = s["case"], s["weights"], s["seqlens"][:, None]
    j = torch.arange(w.shape[1], device=w.device)
    score = torch.where((j < case["first"]) | (j >= n - case["recent"]), math.inf, w)
    score = torch.where(j < n, score, -math.inf)
    width = case["keep"]
    best = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :width]
    if best.shape[1] < width:
        best = torch.cat((best, best.new_full((best.shape[0], width - best.shape[1]), w.shape[1])), 1)
    count = n.clamp(max=case["keep"])
    i = torch.arange(width, device=w.device)
    kept = torch.sort(torch.where(i < count, best, w.shape[1]), dim=1).values
    inside = i < count
    new_weights = torch.where(inside, w.gather(1, kept.clamp(max=w.shape[1] - 1)), 0.0)
    at = torch.where(inside, kept, kept[:, :1])
    to = torch.where(inside, i, 0)
    page = case["page"]
    src = (s["table"].long().gather(1, at // page) * page + at % page).flatten()
    dst = (s["new_table"].long().gather(1, to // page) * page + to % page).flatten()
    for pages in (s["k_pages"], s["v_pages"]):
        flat = pages.view(-1, case["hkv"], D)
        flat[dst] = flat[src]
    kept = torch.where(inside, kept, -1).to(torch.int32)
    return count[:, 0].to(torch.int32), kept, new_weights, s["k_pages"], s["v_pages"]


def run(s):
    case = s["case"]
    if not own:
        return {"attention": _plain_attention, "append": _plain_append, "rotary": _plain_rotary, "evict": _plain_evict}[case["op"]](s)
    f = _package()
    if case["op"] == "attention":
        out, lse = f.split_flash_attn_paged_func(
            s["q"], s["k_pages"], s["v_pages"], s["table"], s["seqlens"], causal=case["window"] < 0,
            window_size=(None, None) if case["window"] < 0 else (case["window"], 0), softcap=case["softcap"],
            key_weights=s.get("weights"), return_lse=True,
        )
        return (out, lse, s["weights"]) if case["weights"] else (out, lse)
    if case["op"] == "append":
        with f.interface.cu_seqlens_validation(False):
            out = f.split_paged_append_func(
                s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["seqlens"], inv_freq=s["inv_freq"],
                cu_seqlens_q=s["cu"] if case["packed"] else None, interleaved=case["interleaved"],
            )
        return out, s["k_pages"], s["v_pages"]
    if case["op"] == "rotary":
        q, k = f.split_rotary_func(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=case["interleaved"])
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return q.detach(), k.detach(), dq, dk
    lens, kept, w = f.split_paged_evict_func(
        s["k_pages"], s["v_pages"], s["table"], s["seqlens"], s["weights"], s["new_table"], case["keep"],
        keep_first=case["first"], keep_recent=case["recent"],
    )
    return lens, kept, w, s["k_pages"], s["v_pages"]


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _turn(x, positions, inv_freq, interleaved, sign=1.0):
    """Complex numbers x1 + i x2 times e^(i angle). x: (..., heads, 512), positions like its leading dimensions."""
    r = 2 * inv_freq.numel()
    x = x.detach().double()
    pairs = x[..., :r].unflatten(-1, (-1, 2)) if interleaved else x[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
    turned = torch.view_as_complex(pairs.contiguous()) * torch.polar(
        torch.ones_like(inv_freq), sign * positions.double()[..., None, None] * inv_freq)
    pairs = torch.view_as_real(turned)
    y = x.clone()
    y[..., :r] = pairs.flatten(-2) if interleaved else pairs.transpose(-1, -2).flatten(-2)
    return y


def exact(case, seed):
    if case["op"] == "evict":
        return None  # nothing is computed: whole numbers, and copies
    s = prepare(case, seed)
    if case["op"] == "rotary":
        f, i, p = s["inv_freq"], case["interleaved"], s["positions"]
        return [_turn(s["q"], p, f, i), _turn(s["k"], p, f, i), _turn(s["dq"], p, f, i, -1.0), _turn(s["dk"], p, f, i, -1.0)]
    lengths, page = s["seqlens"].tolist(), case["page"]
    if case["op"] == "append":
        cu, f, i = s["cu"].tolist(), s["inv_freq"], case["interleaved"]
        packed = [x if case["packed"] else x.flatten(0, 1) for x in (s["q"], s["k"], s["v"])]
        out, kp, vp = torch.empty(packed[0].shape, dtype=torch.float64, device="cuda"), s["k_pages"].double(), s["v_pages"].double()
        for b, n in enumerate(lengths):
            here = slice(cu[b], cu[b + 1])
            at = torch.arange(n - (cu[b + 1] - cu[b]), n, device="cuda")
            out[here] = _turn(packed[0][here], at, f, i)
            where = s["table"][b].long()[at // page], at % page
            kp[where], vp[where] = _turn(packed[1][here], at, f, i), packed[2][here].double()
        return [out.view(s["q"].shape), kp, vp]
    hq, hkv, sq = case["hq"], case["hkv"], case["sq"]
    group = hq // hkv
    out = torch.zeros(case["batch"], sq, hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], hq, sq), -math.inf, dtype=torch.float64, device="cuda")
    w = s["weights"].double() if case["weights"] else None
    for b, n in enumerate(lengths):
        j = torch.arange(n, device="cuda")
        at = s["table"][b].long()[j // page], j % page
        for h in range(hkv):
            k, v = s["k_pages"][at[0], at[1], h].double(), s["v_pages"][at[0], at[1], h].double()
            for i in range(sq):
                end = n - sq + i + 1
                begin = 0 if case["window"] < 0 else max(0, end - 1 - case["window"])
                if end <= begin:
                    continue
                x = s["q"][b, i, h * group : (h + 1) * group].double() @ k[begin:end].T / math.sqrt(D)
                x = case["softcap"] * torch.tanh(x / case["softcap"]) if case["softcap"] else x
                total = torch.logsumexp(x, 1)
                p = torch.exp(x - total[:, None])
                lse[b, h * group : (h + 1) * group, i] = total
                out[b, i, h * group : (h + 1) * group] = p @ v[begin:end]
                if w is not None:
                    w[b, begin:end] += p.sum(0)
    return [out, lse] if w is None else [out, lse, w]
