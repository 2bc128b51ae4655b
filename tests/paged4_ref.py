"""Plain restatements of the smaller paged caches' operators for their tests: rows in 4
bits by the definition of their codes, attention over what they stand for, the keys'
weights and the choice of an eviction in float64 or whole numbers, and the bounds that
fp32 and the results' rounding allow. No counterpart in the reference."""
import math

import torch

import paged_ref

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TOP = {torch.float16: 13, torch.bfloat16: 125}  # exponents of the largest scales


def quantise(x):
    """(codes, scales), uint8 (..., D / 2) and (..., D / 32), of 16-bit rows (..., D)."""
    y = x.double().unflatten(-1, (-1, 32))
    top = y.abs().amax(-1)
    bad = ~torch.isfinite(y).all(-1)
    top = torch.where(bad, torch.ones_like(top), top)
    mantissa, e = torch.frexp(top)  # top = mantissa 2^e, mantissa in [1/2, 1) or 0
    e = e - 3 + (mantissa > 0.875).to(e.dtype)  # (7/8 2^e = 7 2^(e - 3))
    e = torch.where(top == 0, torch.full_like(e, -126), e).clamp(-126, TOP[x.dtype])
    y = torch.where(bad[..., None], torch.zeros_like(y), y / torch.exp2(e.double())[..., None])
    a = y.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    a = torch.round(a / step) * step  # (torch.round: ties to even)
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    code = torch.searchsorted(levels, a.contiguous())
    assert bool((levels[code] == a).all())
    negative = torch.signbit(x.float()).unflatten(-1, (-1, 32)) & ~bad[..., None]
    code = (code + 8 * negative).flatten(-2).to(torch.uint8)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, scale


def values(codes, scales):
    """What rows stand for, float64."""
    x = codes.long()
    half = torch.stack([x % 16, x // 16], -1).flatten(-2)
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64, device=codes.device)
    size = torch.exp2(scales.double() - 127)
    size = torch.where(scales == 255, torch.full_like(size, math.nan), size)
    return (levels[half].unflatten(-1, (-1, 32)) * size[..., None]).flatten(-2)


def attention(q, k, v, table, kv_len, **kw):
    """paged_ref.attention over float64 caches (what 4-bit ones stand for), with bounds of
    paged4's own rounding:
      * o is rounded once, to q's format (u |o|);
      * the probabilities are two bf16 numbers, each half a step (2^-8) off at most, so off
        by 2^-16 of themselves;
      * a score is a sum of D exact products in fp32 (2 D with fp16 q as two numbers),
        whose rounding is at most (2 D + 4) 2^-24 sum |q k| scale, plus 2^-22 of the
        score's and the bias's magnitude;
      * the rest as there: 2 E and 2^-18 of A = sum p |v|, E + 2^-18 (1 + |lse|) for lse.
      * weights below 2^-126 of a row's largest are subnormal in fp32 and may be dropped:
        2^-126 |v| for each key (a code of 0 is exact, so o can be as small as that where
        the heavy keys' values are 0).
    paged_ref's score bound counts D products: twice it covers 2 D."""
    o, lse, o_tol, lse_tol = paged_ref.attention(q, k, v, table, kv_len, **kw)
    a, _, a_tol, _ = paged_ref.attention(q, k, v.abs(), table, kv_len, **kw)
    u = torch.finfo(q.dtype).eps / 2
    # paged_ref: o_tol = u (|o| + A) + (2 E + 2^-18) A, and for |v|, o = A itself.
    scores = a_tol - 2 * u * a
    dropped = 2.0 ** -126 * table.size(1) * k.size(2) * v.abs().nan_to_num(nan=0.0).max()
    return o, lse, u * o.abs() + 2.0 ** -16 * a + 2 * scores + dropped, 2 * lse_tol


def weights(q, k, table, kv_len, lse, before, causal=True, window=None, alibi=None, scale=None,
            restart=False):
    """(weights after, their bound) of paged_weights, k a float64 cache. A row's weight exp(z)
    of z = score - lse is off by E + 2^-21 (|z| + 1) of itself (E as in attention(); z, z
    log2(e) and exp2 are rounded once each, 2^-23 of their size), a sum of n by n 2^-24 of
    it, and each weight by 2^-126 where it is subnormal."""
    B, Hq, N, D = q.shape
    P, Hkv, page, _ = k.shape
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out, tol = before.double().clone(), torch.zeros_like(before, dtype=torch.float64)
    for b in range(B):
        length = min(max(int(kv_len[b]), 0), table.size(1) * page)
        tokens = torch.arange(length, device=q.device)
        pages = table[b].to(q.device).long()[tokens // page]
        there = (pages >= 0) & (pages < P)
        tokens, pages = tokens[there], pages[there]
        if tokens.numel() == 0:
            continue
        at = (length - N + torch.arange(N, device=q.device))[:, None]
        seen = torch.ones(N, tokens.numel(), dtype=torch.bool, device=q.device)
        if causal:
            seen &= tokens[None] <= at
        if window:
            seen &= tokens[None] > at - window
        for g in range(Hkv):
            kk = k[pages, g, tokens % page]
            got, off = torch.zeros_like(tokens, dtype=torch.float64), torch.zeros_like(tokens, dtype=torch.float64)
            for h in range(g * G, (g + 1) * G):
                x = q[b, h].double()
                s = x @ kk.t().contiguous() * scale
                size = x.abs() @ kk.abs().t().contiguous() * scale
                bias = torch.zeros_like(s)
                if alibi is not None:
                    bias = float(alibi[h]) * (at - tokens[None]).abs().double()
                e = (2 * D + 4) * 2.0 ** -24 * size + 2.0 ** -22 * (s.abs() + bias)
                z = s - bias - lse[b, h].double()[:, None]
                w = torch.where(seen, torch.exp(z), torch.zeros_like(z))
                # (a weight of 0 or far below any other has no error to speak of)
                rel = torch.where(w > 0, e + 2.0 ** -21 * (z.abs() + 1), torch.zeros_like(z))
                got += w.sum(0)
                off += (w * rel).sum(0)
            n = G * N
            off += n * 2.0 ** -24 * got + n * 2.0 ** -126
            at_w = (pages, g, tokens % page)
            fresh = (tokens >= length - N) | restart
            # (without restart, keys that no row sees are not touched, or 0 is added)
            old = torch.where(fresh, torch.zeros_like(got), before[at_w].double())
            out[at_w] = old + got
            tol[at_w] = off + 2.0 ** -24 * (old + got).abs()
    return out, tol


def order(w):
    """Weights as whole numbers in their order: NaN above all, both zeros alike."""
    u = w.contiguous().view(torch.int32).long() & 0xffffffff
    u = torch.where(u == 0x80000000, torch.zeros_like(u), u)
    key = torch.where(u >= 0x80000000, 0xffffffff - u, u + 0x80000000)
    return torch.where(torch.isnan(w), torch.full_like(key, 0xffffffff), key)


def evict(arrays, weights, table, kv_len, max_len, recent):
    """new_len of paged_evict; `arrays` ((pages, Hkv, page, ...) each) and weights in place,
    on the CPU, a request and kv head at a time."""
    P, Hkv, page = weights.shape
    new = []
    for b in range(table.size(0)):
        n = min(max(int(kv_len[b]), 0), table.size(1) * page)
        keep = min(n, max(int(max_len[b]), 0))
        new.append(keep)
        if keep == n:
            continue
        newest = min(recent, keep)
        old = n - newest
        tokens = torch.arange(n)
        pages, rows = table[b].long()[tokens // page], tokens % page
        there = (pages >= 0) & (pages < P)
        for g in range(Hkv):
            key = torch.where(there, order(weights[pages.clamp(0, P - 1), g, rows]), torch.zeros_like(pages))
            ranked = torch.sort(key[:old], descending=True, stable=True).indices[:keep - newest]
            kept = torch.cat([ranked.sort().values, tokens[old:]])
            move = there[kept] & there[:keep]  # (from and to places that exist)
            to, kept = tokens[:keep][move], kept[move]
            for a in arrays + [weights]:
                a[pages[to], g, rows[to]] = a[pages[kept], g, rows[kept]].clone()
    return torch.tensor(new, dtype=torch.int32)
