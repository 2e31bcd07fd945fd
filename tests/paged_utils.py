"""Plain 64-bit forms of the operators on a paged cache and of rotary positions, and the error bounds of the kernels.

Bounds (u = 2^-24, one rounding in 32 bits; eps / 2 = one rounding to the 16-bit output):
  score    a dot product of 512 exact products is summed in chains of 8 matrix instructions (16 terms each, the tensor
           core may cut instead of round: 2 u each) and three additions: |error| <= 32 * 2 u * sum |q_d k_d| * scale =: delta
  p        2^(x - m) and m carry delta each and one 2-ulp exp2: relative 2 delta + 8 u; kept as two 16-bit numbers, the
           first cut below p (remainder < 2^-7 p in bf16), the second rounded (2^-9 of the remainder): 2^-16
  sums     over n keys: (n + 64) u relative to the sum of absolute values; joining adds a few u
  out      eps / 2 * |out| + (2 delta + 2^-16 + 8 u + (n + 64) u) * sum p |v|, doubled for numerator and denominator
"""
import math

import torch

D = 512
U = 2.0**-24


def make_cache(lens, page, hkv, dtype, seed, spare=2, fill=float("nan"), width=None, device="cuda"):
    """Pages in random order; every slot that no sequence uses holds `fill`. Unused table entries name no page."""
    g = torch.Generator(device=device).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    k = torch.randn(pages, page, hkv, D, device=device, generator=g).to(dtype)
    v = torch.randn(pages, page, hkv, D, device=device, generator=g).to(dtype)
    order = torch.randperm(pages, device=device, generator=g).to(torch.int32)
    width = max(max(need), 1) if width is None else width
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=device)
    used = torch.zeros(pages, page, dtype=torch.bool, device=device)
    at = 0
    for b, n in enumerate(lens):
        table[b, : need[b]] = order[at : at + need[b]]
        j = torch.arange(n, device=device)
        used[table[b].long()[j // page], j % page] = True
        at += need[b]
    k[~used] = fill
    v[~used] = fill
    return k, v, table, torch.tensor(lens, dtype=torch.int32, device=device), order[at:]


def rows_of(pages, table, b, n):
    page = pages.shape[1]
    j = torch.arange(n, device=pages.device)
    return pages[table[b].long()[j // page], j % page]


def attention_ref(q, k_pages, v_pages, table, lens, scale=None, causal=False, window=(None, None), softcap=0.0):
    """out, lse, weights (B, max length), and the bounds of the kernel's errors of the three."""
    B, sq, hq, _ = q.shape
    hkv = k_pages.shape[2]
    group = hq // hkv
    scale = D**-0.5 if scale is None else scale
    eps = torch.finfo(q.dtype).eps / 2
    left, right = window
    if causal:
        left, right = None, 0
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((B, hq, sq), -math.inf, dtype=torch.float64, device=q.device)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    w = torch.zeros(B, max(max(lens), 1), dtype=torch.float64, device=q.device)
    w_tol = torch.zeros_like(w)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        k, v = rows_of(k_pages, table, b, n).double(), rows_of(v_pages, table, b, n).double()
        j = torch.arange(n, device=q.device)
        for i in range(sq):
            at = n - sq + i
            seen = torch.ones(n, dtype=torch.bool, device=q.device)
            if left is not None and left >= 0:
                seen &= j >= at - left
            if right is not None and right >= 0:
                seen &= j <= at + right
            if not seen.any():
                continue
            js = j[seen]
            for h in range(hkv):
                hs = slice(h * group, (h + 1) * group)
                kk, vv, qq = k[js, h], v[js, h], q[b, i, hs].double()
                x = qq @ kk.T * scale
                delta = 64 * U * ((qq.abs() @ kk.abs().T) * scale).amax(1, keepdim=True)
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                    delta = delta + 8 * U * softcap
                total = torch.logsumexp(x, 1, keepdim=True)
                p = torch.exp(x - total)
                rel = 2 * (2 * delta + 2.0**-16 + (8 + 64 + len(js)) * U)
                out[b, i, hs] = p @ vv
                out_tol[b, i, hs] = eps * 1.01 * (p @ vv).abs() + rel * (p @ vv.abs()) + torch.finfo(q.dtype).smallest_normal * eps
                lse[b, hs, i] = total[:, 0]
                lse_tol[b, hs, i] = (delta + (len(js) + 80) * U + 4 * U * total.abs())[:, 0]
                w[b].index_add_(0, js, p.sum(0))
                w_tol[b].index_add_(0, js, (rel * p).sum(0))
    return out, lse, w, out_tol, lse_tol, w_tol


def rotate_ref(x, positions, inv_freq, interleaved=False, factor=1.0, sign=1.0):
    """positions: the leading dimensions of x without its heads. Returns the result and the bound of the kernel's error."""
    r = 2 * inv_freq.numel()
    eps = torch.finfo(x.dtype).eps / 2
    xd = x.detach().double()
    angle = sign * positions.double()[..., None, None] * inv_freq
    cos, sin = factor * torch.cos(angle), factor * torch.sin(angle)
    head = xd[..., :r]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., : r // 2], head[..., r // 2 :])
    y1, y2 = a * cos - b * sin, a * sin + b * cos
    # cos and sin to 2 ulp, their product with the factor, two products and a sum: 8 u of the absolute values
    t = 8 * U * abs(factor) * (a.abs() + b.abs())
    y, tol = xd.clone(), torch.zeros_like(xd)
    join = (lambda p, q: torch.stack((p, q), -1).flatten(-2)) if interleaved else (lambda p, q: torch.cat((p, q), -1))
    y[..., :r] = join(y1, y2)
    tol[..., :r] = join(t, t) + eps * 1.01 * y[..., :r].abs() + torch.finfo(x.dtype).smallest_normal * eps
    return y, tol


def evict_ref(weights, lens, keep, first, recent):
    """Kept slots of each sequence, ascending."""
    out = []
    for b, n in enumerate(lens):
        m = min(n, keep)
        if n <= keep:
            out.append(list(range(n)))
            continue
        w = weights[b].tolist()
        sure = set(range(first)) | set(range(n - recent, n))
        # largest first, NaN before everything, equal ones by slot
        rank = sorted((j for j in range(n) if j not in sure), key=lambda j: (0 if w[j] != w[j] else 1, -w[j] if w[j] == w[j] else 0.0, j))
        out.append(sorted(list(sure) + rank[: m - len(sure)]))
    return out


def assert_within(got, ref, tol, what):
    got = got.double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(got[~fine], ref[~fine]), f"{what}: other non-finite values"
    err = (got - ref).abs()[fine]
    over = err - tol[fine]
    if over.numel():
        at = int(over.argmax())
        assert float(over.max()) <= 0, f"{what}: error {float(err[at]):.3e}, bound {float(tol[fine][at]):.3e}"
        print(f"    {what}: largest error / bound {float((err / tol[fine].clamp(min=1e-300)).max()):.2f}")
