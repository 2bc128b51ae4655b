"""Performance cases of the paged key/value cache: the block tables, the writes, the attention.

Each case is a plain dict of sizes and options; `prepare` makes what a serving
program holds before the call, `run` makes one pass through one operator (its
plain torch form, or fa_p100's call where `own` is true), `work` counts the
bytes and FLOPs that the pass cannot do without, `exact` computes attention's
outputs in float64, sequence by sequence.

A case's `op` is the operator:
  tables   fa_p100.paged_tables: pages and slots for the lengths of this step
  append   fa_p100.paged_append: the new tokens' keys and values into their slots
  attn     fa_p100.paged_attn: the newest tokens of each sequence over its cache
A cache holds P pages of `page` rows per kv head, (P, Hkv, page, D) with
layout "bhnd", or (P, page, Hkv, D) handed over as a transposed view with
"bnhd"; sequence b's token j is row j % page of page block_table[b, j // page].
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _fa():
    path = os.path.abspath("flash-attention-p100_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fa_p100
    return fa_p100


# ------------------------------------------------------------------ the cases

def _tables(name, B, page, top, prompts, leaving, packed):
    """B requests of up to `top` tokens: `prompts` of them enter with their whole
    prompt, `leaving` of them end, the others grow by one token. The slots come
    packed (one run of tokens) or as (B, the most new tokens)."""
    case = dict(op="tables", B=B, page=page, top=top, prompts=prompts, leaving=leaving,
                packed=packed)
    return dict(case, name=name) if name else case


def _append(name, T, Hkv, D, page, dtype, layout, spare):
    """T new tokens' rows, the last `spare` of them padding (slot -1)."""
    case = dict(op="append", T=T, Hkv=Hkv, D=D, page=page, dtype=dtype, layout=layout, spare=spare)
    return dict(case, name=name) if name else case


def _attn(name, B, Hq, Hkv, N, D, dtype, top, page, low=1.0, layout="bhnd", window=0, alibi=False,
          idle=0, lse=False):
    """B sequences of low * top to top cached tokens, the newest N of them queries;
    the last `idle` entries of the batch hold no request (length 0)."""
    case = dict(op="attn", B=B, Hq=Hq, Hkv=Hkv, N=N, D=D, dtype=dtype, top=top, page=page, low=low,
                layout=layout, window=window, alibi=alibi, idle=idle, lse=lse)
    return dict(case, name=name) if name else case


def listed():
    return [
        # A decoding step of a serving batch: one more token each, a page now
        # and then (the smallest call: latency).
        _tables("tables_step", 64, 16, 4000, 0, 0, False),
        # Admission: prompts of all lengths enter while others end, their
        # tokens packed as one run.
        _tables("tables_prompts", 96, 16, 16384, 40, 24, True),
        # The decoding step's new keys and values.
        _append("append_step", 64, 8, 128, 16, "bf16", "bhnd", 0),
        # The packed prompts' keys and values after the prefill's projections,
        # padded to a round number of tokens.
        _append("append_prompts", 65536, 8, 128, 32, "fp16", "bnhd", 1001),
        # One user's chat turn: one token over a short cache, the heads of a
        # 0.6B decoder.
        _attn("attn_one", 1, 16, 8, 1, 128, "bf16", 1021, 16),
        # A serving batch of ragged contexts, grouped heads 32/8, one slot of
        # the batch unused.
        _attn("attn_batch", 16, 32, 8, 1, 128, "fp16", 8192, 16, low=0.1, idle=1),
        # Many short requests at once, with ALiBi.
        _attn("attn_many", 250, 32, 4, 1, 128, "fp16", 600, 16, low=0.05, alibi=True),
        # Five drafted tokens per sequence checked at once, rows stored as the
        # projections leave them, with the row sums for a later join.
        _attn("attn_draft", 8, 16, 4, 5, 64, "bf16", 4003, 32, low=0.3, layout="bnhd", lse=True),
        # A sliding-window layer: only the last 1024 tokens are read.
        _attn("attn_window", 24, 12, 12, 1, 64, "bf16", 9000, 64, low=0.1, window=1024),
        # Wide heads, few kv heads, small pages.
        _attn("attn_wide", 4, 16, 2, 1, 256, "bf16", 8000, 8, low=0.5),
        # A long document: two sequences, one kv head shared by eight.
        _attn("attn_long", 2, 64, 8, 1, 128, "bf16", 131072, 128, low=0.9),
        # A full serving batch of long contexts (the largest call).
        _attn("attn_serving", 64, 32, 8, 1, 128, "bf16", 16384, 32, low=0.2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the ranges above: sizes spread over their logarithm, ragged ones among them."""
    while True:
        op = rng.choice(["tables", "append", "attn", "attn", "attn"])
        page = 2 ** rng.randint(3, 8)
        if op == "tables":
            B = _log_int(rng, 1, 1000)
            prompts = rng.randint(0, B) if rng.random() < 0.6 else 0
            case = _tables("", B, page, _log_int(rng, 64, 32768), prompts,
                           rng.randint(0, B - prompts), bool(rng.random() < 0.5 or prompts))
            if _pool(case) > 400000 or _new_tokens(case) > 600000:
                continue
            return case
        Hkv = rng.choice([1, 2, 4, 8, 12])
        D = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        dtype, layout = rng.choice(["fp16", "bf16"]), rng.choice(["bhnd", "bnhd"])
        if op == "append":
            T = _log_int(rng, 1, 65536)
            case = _append("", T, Hkv, D, page, dtype, layout, rng.choice([0, 0, T // 7]))
            if work(case)["bytes"] > 5.4e8:
                continue
            return case
        Hq = Hkv * rng.choice([1, 2, 4, 8])
        if Hq > 64:
            continue
        B = _log_int(rng, 1, 256)
        case = _attn("", B, Hq, Hkv, rng.choice([1, 1, 1, 1, 2, 4, 7]), D, dtype,
                     _log_int(rng, 50, 131072), page, low=rng.choice([0.05, 0.3, 1.0]),
                     layout=layout, window=rng.choice([0, 0, 0, 1024]), alibi=rng.random() < 0.2,
                     idle=rng.choice([0, 0, B // 6]))
        if case["top"] < case["N"]:
            continue
        w, rows = work(case), B * Hkv * case["top"] * D
        if w["bytes"] <= 2.6e9 and rows <= 1.1e9 and \
                (case["window"] == 0 or case["top"] * B <= 400000):
            return case


# ---------------------------------------------------------- lengths and pages

def _fractions(n):
    """n numbers spread evenly over [0, 1), in no order."""
    return [(0.5 + 0.6180339887498949 * i) % 1.0 for i in range(n)]


def _attn_lengths(case):
    live = case["B"] - case["idle"]
    lens = [max(case["N"], int(round(case["top"] * (case["low"] + (1.0 - case["low"]) * f))))
            for f in _fractions(live)]
    if lens:
        lens[0] = max(case["N"], case["top"])
    return lens + [0] * case["idle"]


def _tables_lengths(case):
    """(old, new) lengths of the requests."""
    pairs = []
    for i, f in enumerate(_fractions(case["B"])):
        n = max(1, int(round(case["top"] * f)))
        if i < case["prompts"]:
            pairs.append((0, n))
        elif i < case["prompts"] + case["leaving"]:
            pairs.append((n, 0))
        else:
            pairs.append((n, n + 1))
    return pairs


def _pages(n, page):
    return (n + page - 1) // page


def _width(top, page):
    """Table entries per sequence: room for a quarter more than the longest."""
    return _pages(top + top // 4 + 1, page)


def _pool(case):
    used = sum(max(_pages(o, case["page"]), _pages(n, case["page"])) for o, n in _tables_lengths(case))
    return used + used // 8 + 1


def _new_tokens(case):
    return sum(max(n - o, 0) for o, n in _tables_lengths(case))


# ------------------------------------------------------------------ the inputs

def _cache(case, P, gen):
    Hkv, page, D = case["Hkv"], case["page"], case["D"]
    shape = (P, page, Hkv, D) if case["layout"] == "bnhd" else (P, Hkv, page, D)
    out = []
    for _ in range(2):
        t = torch.empty(shape, device="cuda", dtype=_DTYPES[case["dtype"]])
        for part in t.split(max(1, P // 8)):
            part.copy_(torch.randn(part.shape, device="cuda", generator=gen))
        out.append(t.transpose(1, 2) if case["layout"] == "bnhd" else t)
    return out


def _prepare_tables(case, seed):
    rng = torch.Generator().manual_seed(int(seed))
    B, page = case["B"], case["page"]
    order = torch.randperm(B, generator=rng)
    old, new = (torch.tensor(x, dtype=torch.int32)[order] for x in zip(*_tables_lengths(case)))
    pool, width = _pool(case), _width(case["top"], page)
    perm = torch.randperm(pool, generator=rng).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    have, used = (old + page - 1) // page, 0
    for b, n in enumerate(have.tolist()):
        table[b, :n] = perm[used:used + n]
        used += n
    # The free pages lie in a ring of `pool` entries, anywhere in it.
    head = int(torch.randint(0, pool, (), generator=rng))
    free = torch.full((pool,), -1, dtype=torch.int32)
    free[(head + torch.arange(pool - used)) % pool] = perm[used:]
    tokens = _new_tokens(case)
    return dict(table=table.cuda(), old=old.cuda(), new=new.cuda(), free=free.cuda(),
                ring=torch.tensor([head, pool - used], dtype=torch.int32).cuda(), page=page,
                max_new=None if case["packed"] else 1,
                tokens=tokens + tokens // 16 + 1 if case["packed"] else None)


def _prepare_append(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    T, page = case["T"], case["page"]
    P = _pages(T, page) + T // (8 * page) + 2
    k_cache, v_cache = _cache(case, P, gen)
    # Tokens of one sequence follow each other within a page; the pages are anywhere.
    pages = torch.randperm(P, device="cuda", generator=gen)
    t = torch.arange(T, device="cuda") + int(seed) % page
    slots = (pages[t // page] * page + t % page).to(torch.int32)
    if case["spare"]:
        slots[T - case["spare"]:] = -1
    k, v = (torch.randn((T, case["Hkv"], case["D"]), device="cuda", generator=gen)
            .to(_DTYPES[case["dtype"]]) for _ in range(2))
    return dict(k=k, v=v, k_cache=k_cache, v_cache=v_cache, slots=slots)


def _prepare_attn(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    rng = torch.Generator().manual_seed(int(seed))
    B, Hq, N, D, page = (case[x] for x in ("B", "Hq", "N", "D", "page"))
    live = B - case["idle"]
    lens = torch.tensor(_attn_lengths(case), dtype=torch.int32)
    lens[:live] = lens[:live][torch.randperm(live, generator=rng)]
    need = (lens + page - 1) // page
    used = int(need.sum())
    P = used + used // 8 + 1
    perm = torch.randperm(P, generator=rng).to(torch.int32)
    table = torch.full((B, _width(case["top"], page)), -1, dtype=torch.int32)
    first = 0
    for b, n in enumerate(need.tolist()):
        table[b, :n] = perm[first:first + n]
        first += n
    k_cache, v_cache = _cache(case, P, gen)
    shape = (B, N, Hq, D) if case["layout"] == "bnhd" else (B, Hq, N, D)
    q = torch.randn(shape, device="cuda", generator=gen).to(_DTYPES[case["dtype"]])
    if case["layout"] == "bnhd":
        q = q.transpose(1, 2)
    slopes = None
    if case["alibi"]:
        slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)]).cuda()
    return dict(q=q, k_cache=k_cache, v_cache=v_cache, table=table.cuda(), lens=lens.cuda(),
                top=max(1, int(lens.max())), window=case["window"], slopes=slopes, lse=case["lse"])


_PREPARE = {"tables": _prepare_tables, "append": _prepare_append, "attn": _prepare_attn}


def prepare(case, seed):
    return dict(_PREPARE[case["op"]](case, seed), op=case["op"])


# ------------------------------------------------------------- the plain forms

def _tables_plain(s):
    table, free, page = s["table"], s["free"], s["page"]
    B, M = table.shape
    C, dev = free.numel(), table.device
    old = s["old"].long().clamp(0, M * page)
    new = s["new"].long().clamp(min=0)
    want_len = new.clamp(max=M * page)
    have, want = (old + page - 1) // page, (want_len + page - 1) // page
    need, gone = (want - have).clamp(min=0), (have - want).clamp(min=0)
    first, first_gone = need.cumsum(0) - need, gone.cumsum(0) - gone
    head, count = s["ring"].long().unbind()
    given = torch.minimum((count - first).clamp(min=0), need)
    kv_len = torch.where(want_len > old, torch.minimum(want_len, (have + given) * page), want_len)
    i = torch.arange(M, device=dev)[None, :]
    # Pages that go back to the ring, written past its last free page.
    back = (i >= want[:, None]) & (i < have[:, None])
    dst = (head + count + first_gone[:, None] + i - want[:, None]) % C
    wider = torch.cat([free, free.new_zeros(1)])
    wider[torch.where(back, dst, torch.full_like(dst, C)).flatten()] = table.flatten()
    src = (head + first[:, None] + i - have[:, None]) % C
    fresh = (i >= have[:, None]) & (i < (have + given)[:, None])
    table.copy_(torch.where(fresh, free[src], table))
    free.copy_(wider[:C])
    ring = torch.stack([(head + given.sum()) % C, count - given.sum() + gone.sum()])
    # The slot of every new token.
    if s["tokens"] is None:
        pos = old[:, None] + torch.arange(s["max_new"], device=dev)[None, :]
        row = torch.arange(B, device=dev)[:, None].expand_as(pos)
        known = torch.ones_like(pos, dtype=torch.bool)
    else:
        grown = (new - old).clamp(min=0)
        ends = grown.cumsum(0)
        t = torch.arange(s["tokens"], device=dev)
        row = torch.searchsorted(ends, t, right=True)
        known = row < B
        row = row.clamp(max=B - 1)
        pos = old[row] + t - (ends - grown)[row]
    known = known & (pos < kv_len[row])
    page_of = table[row, (pos // page).clamp(max=M - 1)].long()
    slots = torch.where(known, page_of * page + pos % page, torch.full_like(pos, -1))
    return table, slots.to(torch.int32), kv_len.to(torch.int32), free, ring.to(torch.int32)


def _append_plain(s):
    page = s["k_cache"].size(2)
    live = s["slots"] >= 0
    slots = s["slots"][live].long()
    s["k_cache"][slots // page, :, slots % page] = s["k"][live]
    s["v_cache"][slots // page, :, slots % page] = s["v"][live]
    return s["k_cache"], s["v_cache"]


def _attn_plain(s):
    q, lens, dev = s["q"], s["lens"].long(), s["q"].device
    B, Hq, N, D = q.shape
    P, Hkv, page, _ = s["k_cache"].shape
    pages = _pages(s["top"], page)
    ids = s["table"][:, :pages].long().clamp(min=0)

    def rows(cache):  # (B, Hkv, pages * page, D), in 32 bits
        x = cache[ids].float()
        return x.transpose(1, 2).reshape(B, Hkv, pages * page, D)

    k, v = rows(s["k_cache"]), rows(s["v_cache"])
    G, K = Hq // Hkv, pages * page
    x = q.float().reshape(B, Hkv, G * N, D)
    scores = torch.matmul(x, k.transpose(-1, -2)).reshape(B, Hq, N, K) / math.sqrt(D)
    i = (lens[:, None] - N + torch.arange(N, device=dev)[None, :])[:, None, :, None]
    j = torch.arange(K, device=dev)[None, None, None, :]
    if s["slopes"] is not None:
        scores = scores - s["slopes"][None, :, None, None] * (i - j).abs()
    seen = j <= i
    if s["window"]:
        seen = seen & (j > i - s["window"])
    scores = scores.masked_fill(~seen, -math.inf)
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(scores - m)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(B, Hkv, G * N, K), v).reshape(B, Hq, N, D)
    o = (o / torch.where(total == 0, torch.ones_like(total), total)).to(q.dtype)
    if not s["lse"]:
        return o
    lse = (m + torch.log(total)).squeeze(-1)
    return o, torch.where(total.squeeze(-1) == 0, torch.full_like(lse, math.inf), lse)


_PLAIN = {"tables": _tables_plain, "append": _append_plain, "attn": _attn_plain}


# --------------------------------------------------------- the framework's calls

def _tables_own(s):
    slots, kv_len, ring = _fa().paged_tables(s["table"], s["old"], s["new"], s["free"], s["ring"],
                                             s["page"], max_new=s["max_new"], tokens=s["tokens"])
    return s["table"], slots, kv_len, s["free"], ring


def _append_own(s):
    _fa().paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
    return s["k_cache"], s["v_cache"]


def _attn_own(s):
    return _fa().paged_attn(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], causal=True,
                            sliding_window=s["window"] or None, alibi_slopes=s["slopes"],
                            return_lse=s["lse"])


_OWN = {"tables": _tables_own, "append": _append_own, "attn": _attn_own}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ------------------------------------------------------- what the path needs

def work(case):
    if case["op"] == "tables":
        page, moved = case["page"], 0
        for old, new in _tables_lengths(case):
            moved += abs(_pages(new, page) - _pages(old, page))
        # lengths in and out, a page read and written for each that moves, the
        # page of the token a request grows from, the slots
        slots = _new_tokens(case) if case["packed"] else case["B"]
        grows = sum(1 for old, new in _tables_lengths(case) if new > old and old % page)
        return {"bytes": 12 * case["B"] + 8 * moved + 4 * grows + 4 * slots, "flops": 0}
    if case["op"] == "append":
        rows = case["T"] - case["spare"]
        return {"bytes": 2 * 2 * 2 * rows * case["Hkv"] * case["D"] + 4 * case["T"], "flops": 0}
    B, Hq, Hkv, N, D, page = (case[x] for x in ("B", "Hq", "Hkv", "N", "D", "page"))
    keys = pairs = pages = 0
    for n in _attn_lengths(case):
        if n == 0:
            continue
        low = max(0, n - N + 1 - case["window"]) if case["window"] else 0
        keys += n - low
        pages += _pages(n, page) - low // page
        pairs += sum(min(n - N + 1 + i, case["window"] or n) for i in range(N))
    return {"bytes": 2 * 2 * B * Hq * N * D + 2 * 2 * Hkv * D * keys + 4 * pages + 4 * B,
            "flops": 4 * D * Hq * pairs}


# ------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """Attention from its definition, one sequence and kv head at a time, and the
    written caches as a list of rows; the tables are whole numbers."""
    if case["op"] == "tables":
        return None
    if case["op"] == "append":
        return _exact_append(_prepare_append(case, seed))
    s = _prepare_attn(case, seed)
    q, page = s["q"], case["page"]
    B, Hq, N, D = q.shape
    G = Hq // case["Hkv"]
    out = torch.zeros((B, Hq, N, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, N), math.inf, dtype=torch.float64, device="cuda")
    lens = s["lens"].tolist()
    for b, length in enumerate(lens):
        if length == 0:
            continue
        start = max(0, length - N + 1 - case["window"]) if case["window"] else 0
        tokens = torch.arange(start, length, device="cuda")
        where = s["table"][b].long()[tokens // page]
        for g in range(case["Hkv"]):
            keys = s["k_cache"][where, g, tokens % page].double()
            values = s["v_cache"][where, g, tokens % page].double()
            for n in range(N):
                at = length - N + n
                if at < 0:
                    continue
                heads = slice(g * G, (g + 1) * G)
                z = q[b, heads, n].double() @ keys.t().contiguous() * D ** -0.5
                if case["alibi"]:
                    z = z - s["slopes"][heads].double()[:, None] * (at - tokens).abs()
                hidden = tokens > at
                if case["window"]:
                    hidden = hidden | (tokens <= at - case["window"])
                z = z.masked_fill(hidden, -math.inf)
                lse[b, heads, n] = torch.logsumexp(z, -1)
                out[b, heads, n] = torch.softmax(z, -1) @ values
    return (out, lse) if case["lse"] else out


def _exact_append(s):
    """The caches as rows in slot order, token t's row put at slots[t]."""
    written = []
    for cache, new in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        P, Hkv, page, D = cache.shape
        rows = cache.double().permute(0, 2, 1, 3).reshape(P * page, Hkv, D)
        live = (s["slots"] >= 0).nonzero().squeeze(-1)
        rows.index_copy_(0, s["slots"][live].long(), new[live].double())
        written.append(rows.reshape(P, page, Hkv, D).permute(0, 2, 1, 3))
    return tuple(written)
