"""Plain restatements of the paged cache's operators for their tests: the tables by
a loop over requests and pages, attention in float64 from rows gathered token by
token, and the bounds its rounding allows. No counterpart in the reference."""
import math

import torch


def tables(table, old_len, new_len, free, ring, page, max_new=None, tokens=None):
    """(table, free, slots, kv_len, ring) after fa_p100.paged_tables; lists and CPU
    tensors, the inputs left alone."""
    table, free = table.clone(), free.clone()
    B, M = table.shape
    C, cap = free.numel(), table.size(1) * page
    head, count = int(ring[0]) % C, min(max(int(ring[1]), 0), C)
    taken = gone = 0
    kv_len, packed = [], []
    slots = None if max_new is None else torch.full((B, max_new), -1, dtype=torch.int32)
    before = table.clone()
    for b in range(B):
        old = min(max(int(old_len[b]), 0), cap)
        n = max(int(new_len[b]), 0)
        want_len = min(n, cap)
        have, want = -(-old // page), -(-want_len // page)
        got = have
        while got < want and taken < count:
            table[b, got] = free[(head + taken) % C]
            taken, got = taken + 1, got + 1
        for p in range(want, have):
            if gone < C - count:
                free[(head + count + gone) % C] = before[b, p]
                gone += 1
        length = min(want_len, got * page) if want_len > old else want_len
        kv_len.append(length)
        for i, j in enumerate(range(old, max(n, old))):
            at = int(table[b, j // page]) if j < length else -1
            slot = at * page + j % page if 0 <= at * page <= 2 ** 31 - 1 - j % page else -1
            packed.append(slot)
            if slots is not None and i < max_new:
                slots[b, i] = slot
    if tokens is not None:
        slots = torch.tensor((packed + [-1] * tokens)[:tokens], dtype=torch.int32)
    ring = torch.tensor([(head + taken) % C, count - taken + gone], dtype=torch.int32)
    return table, free, slots, torch.tensor(kv_len, dtype=torch.int32), ring


def attention(q, k_cache, v_cache, table, kv_len, causal=True, window=None, alibi=None,
              scale=None):
    """(o, lse, o_tol, lse_tol) in float64 on q's device, from the tokens' rows
    one request at a time. Keys in pages outside the pool are hidden.

    The tolerances are the rounding's: with u half a step of q's format, A = sum_j
    p_j |v_j| and E the error of a score,
      * o is rounded once (u |o|) and the probabilities once, as operands of the
        second product (u A);
      * a score is a sum of D products in fp32, whose rounding is at most (D + 2)
        2^-24 sum |q k| scale, plus the scale's and the bias's in fp32 (2^-22 of
        the score's magnitude and the bias's), and moves p and thereby o by
        2 E A at most and lse by E;
      * sums over keys, the exponentials and the joins in fp32: 2^-18 A (64 units
        of 2^-24: partial sums, up to log2 of the keys' count, and exp2's and the
        reciprocal's few), and 2^-18 (1 + |lse|) for lse.
    """
    B, Hq, N, D = q.shape
    P, Hkv, page, _ = k_cache.shape
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    dev = q.device
    o = torch.zeros(B, Hq, N, D, dtype=torch.float64, device=dev)
    lse = torch.full((B, Hq, N), math.inf, dtype=torch.float64, device=dev)
    o_tol, lse_tol = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(B):
        length = min(max(int(kv_len[b]), 0), table.size(1) * page)
        tokens = torch.arange(length, device=dev)
        pages = table[b].to(dev).long()[tokens // page]
        there = (pages >= 0) & (pages < P)
        tokens, pages = tokens[there], pages[there]
        if tokens.numel() == 0:
            continue
        k = k_cache[pages, :, tokens % page].double().transpose(0, 1)  # (Hkv, keys, D)
        v = v_cache[pages, :, tokens % page].double().transpose(0, 1)
        at = (length - N + torch.arange(N, device=dev))[:, None]
        seen = torch.ones(N, tokens.numel(), dtype=torch.bool, device=dev)
        if causal:
            seen &= tokens[None] <= at
        if window:
            seen &= tokens[None] > at - window
        for h in range(Hq):
            x = q[b, h].double()
            kk, vv = k[h // G], v[h // G]
            vv = torch.where(seen.any(0)[:, None], vv, torch.zeros_like(vv))
            s = x @ kk.t().contiguous() * scale
            size = x.abs() @ kk.abs().t().contiguous() * scale
            bias = torch.zeros_like(s)
            if alibi is not None:
                bias = float(alibi[h]) * (at - tokens[None]).abs().double()
            e = (D + 2) * 2.0 ** -24 * size + 2.0 ** -22 * (s.abs() + bias)
            e = torch.where(seen, e, torch.zeros_like(e)).amax(-1)
            s = (s - bias).masked_fill(~seen, -math.inf)
            some = seen.any(-1)
            p = torch.softmax(s, -1).masked_fill(~seen, 0.0)
            o[b, h] = p @ vv
            a = p @ vv.abs()
            o_tol[b, h] = u * (o[b, h].abs() + a) + (2 * e[:, None] + 2.0 ** -18) * a
            row = torch.logsumexp(s, -1)
            lse[b, h] = torch.where(some, row, torch.full_like(row, math.inf))
            lse_tol[b, h] = torch.where(some, e + 2.0 ** -18 * (1 + row.abs()), torch.zeros_like(e))
    return o, lse, o_tol, lse_tol


def check(got_o, got_lse, ref):
    """got against attention()'s (o, lse, tolerances)."""
    o, lse, o_tol, lse_tol = ref
    err = (got_o.double() - o).abs()
    assert bool(torch.isfinite(got_o).all())
    # (a value that rounds to a subnormal is off by half its fixed step)
    tiny = torch.finfo(got_o.dtype).smallest_normal * torch.finfo(got_o.dtype).eps
    over = err - o_tol - tiny
    assert bool((over <= 0).all()), f"o off by {err.max().item():.3e}, {over.max().item():.3e} over"
    if got_lse is not None:
        empty = torch.isinf(lse)
        assert torch.equal(torch.isinf(got_lse) & (got_lse > 0), empty)
        err = torch.where(empty, torch.zeros_like(lse), got_lse.double() - lse).abs()
        assert bool((err <= lse_tol).all()), f"lse off by {err.max().item():.3e}"
