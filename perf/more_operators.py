"""Performance cases of a smaller key/value cache: rows held in 4 bits, and the rows that matter.

Each case is a plain dict of sizes and options; `prepare` makes what a serving
program holds before the call, `run` makes one pass through one operator (its
plain torch form, or fa_p100's call where `own` is true), `work` counts the
bytes and FLOPs that the pass cannot do without, `exact` computes the outputs in
float64.

A case's `op` is the operator:
  append   fa_p100.paged_append into a 4-bit cache: new tokens' rows quantised into
           their slots; what they stand for is read back with paged_gather
  gather   fa_p100.paged_gather: rows of a cache by their slots, dense
  attn     fa_p100.paged_attn over a 4-bit cache: the newest tokens of each request
  weights  fa_p100.paged_weights: the attention weight that each cached key gets from
           the newest rows, added to what it got before
  evict    fa_p100.paged_evict: each kv head keeps the newest and the heaviest keys

A cache holds P pages of `page` rows per kv head, (P, Hkv, page, row) with layout
"bhnd", or (P, page, Hkv, row) handed over as a transposed view with "bnhd". With
`bits` 16 a row is D values of `dtype`. With 4 it is D / 2 bytes, value d in the low
(d even) or high half of byte d // 2, and D / 32 bytes of scales: a half is a sign
and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, a scale byte x stands for 2^(x - 127) and
is that of 32 values. The scale of a block is the least power of two of which its
largest value is 7 times or less; values are rounded to the nearest, ties to the
even code. Token j of request b is row j % page of page table[b, j // page].
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# The largest scales: six times these is within the format that the values came in.
_TOP_SCALE = {"fp16": 127 + 13, "bf16": 127 + 125}


def _fa():
    path = os.path.abspath("flash-attention-p100_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fa_p100
    return fa_p100


# ------------------------------------------------------------------ the cases

def _append(name, T, Hkv, D, page, dtype, layout):
    """T new tokens' rows into a 4-bit cache."""
    case = dict(op="append", bits=4, T=T, Hkv=Hkv, D=D, page=page, dtype=dtype, layout=layout)
    return dict(case, name=name) if name else case


def _gather(name, bits, T, Hkv, D, page, dtype, layout, spare):
    """T rows, the last `spare` of them padding (slot -1, zeros)."""
    case = dict(op="gather", bits=bits, T=T, Hkv=Hkv, D=D, page=page, dtype=dtype, layout=layout,
                spare=spare)
    return dict(case, name=name) if name else case


def _attn(name, B, Hq, Hkv, N, D, dtype, top, page, low=1.0, layout="bhnd", window=0, alibi=False,
          idle=0, lse=False):
    """B requests of low * top to top tokens in 4 bits, the newest N of them queries;
    the last `idle` entries of the batch hold no request (length 0)."""
    case = dict(op="attn", bits=4, B=B, Hq=Hq, Hkv=Hkv, N=N, D=D, dtype=dtype, top=top, page=page,
                low=low, layout=layout, window=window, alibi=alibi, idle=idle, lse=lse)
    return dict(case, name=name) if name else case


def _weights(name, bits, B, Hq, Hkv, N, D, dtype, top, page, low=1.0, layout="bhnd", idle=0,
             restart=False):
    """The weights that N newest rows of each request give its keys; with `restart`
    nothing was added before."""
    case = dict(op="weights", bits=bits, B=B, Hq=Hq, Hkv=Hkv, N=N, D=D, dtype=dtype, top=top,
                page=page, low=low, layout=layout, idle=idle, restart=restart)
    return dict(case, name=name) if name else case


def _evict(name, B, Hkv, D, dtype, top, page, keep, recent, low=1.0, layout="bhnd"):
    """B requests of low * top to top tokens; those over `keep` are cut to it."""
    case = dict(op="evict", bits=16, B=B, Hkv=Hkv, D=D, dtype=dtype, top=top, page=page, keep=keep,
                recent=recent, low=low, layout=layout)
    return dict(case, name=name) if name else case


def listed():
    return [
        # A decoding step's new keys and values (the smallest call: latency).
        _append("append_step", 64, 8, 128, 16, "bf16", "bhnd"),
        # The packed prompts' keys and values after the prefill's projections.
        _append("append_prompts", 65536, 8, 128, 32, "fp16", "bnhd"),
        # A prompt's cached beginning, wanted dense for the attention of its new part.
        _gather("gather_prefix", 4, 30011, 8, 128, 16, "bf16", "bhnd", 0),
        # Sequences moved out of a 16-bit cache to make room.
        _gather("gather_out", 16, 20000, 4, 80, 64, "fp16", "bnhd", 1333),
        # One user's chat turn: one token over a short cache, the heads of a 0.6B decoder.
        _attn("attn_one", 1, 16, 8, 1, 128, "bf16", 1021, 16),
        # A serving batch of ragged contexts, grouped heads 32/8, one slot unused.
        _attn("attn_batch", 16, 32, 8, 1, 128, "fp16", 8192, 16, low=0.1, idle=1),
        # Five drafted tokens per request checked at once, with the row sums that the
        # weights below need.
        _attn("attn_draft", 8, 16, 4, 5, 64, "bf16", 4003, 32, low=0.3, layout="bnhd", lse=True),
        # A full serving batch of long contexts.
        _attn("attn_serving", 64, 32, 8, 1, 128, "bf16", 16384, 32, low=0.2),
        # The weights of a decoding step of that batch's like.
        _weights("weights_step", 4, 16, 32, 8, 1, 128, "bf16", 8192, 16, low=0.1, idle=1),
        # A prompt judged by its last 32 rows, before it is cut.
        _weights("weights_window", 16, 2, 32, 8, 32, 128, "bf16", 16384, 32, restart=True),
        # A budget kept while decoding: 76 tokens over it, the newest 256 stay.
        _evict("evict_step", 32, 8, 128, "bf16", 1100, 16, 1024, 256),
        # Long prompts cut to an eighth.
        _evict("evict_prompts", 4, 8, 128, "fp16", 32768, 32, 4096, 64, low=0.5, layout="bnhd"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the ranges above: sizes spread over their logarithm, ragged ones among them."""
    while True:
        op = rng.choice(["append", "gather", "attn", "attn", "weights", "evict"])
        page = 2 ** rng.randint(3, 8)
        Hkv = rng.choice([1, 2, 4, 8, 12])
        dtype, layout = rng.choice(["fp16", "bf16"]), rng.choice(["bhnd", "bnhd"])
        bits = rng.choice([4, 16])
        narrow = [64, 80, 96, 128, 128, 128, 256]  # (4-bit rows: whole blocks of 32)
        D = rng.choice(narrow if op == "evict" or (bits == 16 and op in ("gather", "weights"))
                       else [64, 96, 128, 128, 128, 160, 256])
        if op in ("append", "gather"):
            T = _log_int(rng, 1, 65536)
            if op == "append":
                case = _append("", T, Hkv, D, page, dtype, layout)
            else:
                case = _gather("", bits, T, Hkv, D, page, dtype, layout, rng.choice([0, 0, T // 7]))
            if work(case)["bytes"] > 6.0e8:
                continue
            return case
        if op == "evict":
            top = _log_int(rng, 100, 65536)
            case = _evict("", _log_int(rng, 1, 128), Hkv, D, dtype, top, page,
                          max(1, int(top * rng.choice([0.1, 0.4, 0.9]))), rng.choice([0, 16, 256]),
                          low=rng.choice([0.1, 0.5, 1.0]), layout=layout)
            if case["B"] * top * Hkv * D > 1.4e8:
                continue
            return case
        Hq = Hkv * rng.choice([1, 2, 4, 8])
        if Hq > 64:
            continue
        B, top = _log_int(rng, 1, 256), _log_int(rng, 50, 131072)
        low, idle = rng.choice([0.05, 0.3, 1.0]), rng.choice([0, 0, B // 6])
        if op == "attn":
            case = _attn("", B, Hq, Hkv, rng.choice([1, 1, 1, 1, 2, 4, 7]), D, dtype, top, page,
                         low=low, layout=layout, window=rng.choice([0, 0, 0, 1024]),
                         alibi=rng.random() < 0.2, idle=idle, lse=rng.random() < 0.3)
        else:
            case = _weights("", bits, B, Hq, Hkv, rng.choice([1, 1, 1, 3, 16, 64]), D, dtype, top,
                            page, low=low, layout=layout, idle=idle, restart=rng.random() < 0.3)
        if top < case["N"]:
            continue
        if B * Hkv * top * D <= 1.1e9 and B * Hq * case["N"] * top <= 1.5e8 and \
                work(case)["flops"] <= 3e10 and work(case)["bytes"] <= 7e8:
            return case


# ---------------------------------------------------------- lengths and pages

def _fractions(n):
    """n numbers spread evenly over [0, 1), in no order."""
    return [(0.5 + 0.6180339887498949 * i) % 1.0 for i in range(n)]


def _lengths(case):
    live, least = case["B"] - case.get("idle", 0), case.get("N", 1)
    lens = [max(least, int(round(case["top"] * (case["low"] + (1.0 - case["low"]) * f))))
            for f in _fractions(live)]
    if lens:
        lens[0] = max(least, case["top"])
    return lens + [0] * (case["B"] - live)


def _pages(n, page):
    return (n + page - 1) // page


# ------------------------------------------------------------------ the inputs

def _empty_pool(case, P, width, dtype):
    Hkv, page = case["Hkv"], case["page"]
    if case["layout"] == "bnhd":
        return torch.zeros((P, page, Hkv, width), device="cuda", dtype=dtype).transpose(1, 2)
    return torch.zeros((P, Hkv, page, width), device="cuda", dtype=dtype)


def _pool(case, P, gen):
    """A pool of rows of random values: (rows, None), or (codes, scales) in 4 bits."""
    D, dtype = case["D"], _DTYPES[case["dtype"]]
    four = case["bits"] == 4
    rows = _empty_pool(case, P, D // 2 if four else D, torch.uint8 if four else dtype)
    scales = _empty_pool(case, P, D // 32, torch.uint8) if four else None
    step = max(1, (1 << 24) // (case["Hkv"] * case["page"] * D))
    for p in range(0, P, step):
        n = min(step, P - p)
        x = torch.randn((n, case["Hkv"], case["page"], D), device="cuda", generator=gen).to(dtype)
        if four:
            rows[p:p + n], scales[p:p + n] = _quantise(x, case["dtype"])
        else:
            rows[p:p + n] = x
    return rows, scales


def _requests(case, rng, spare=8):
    """(lens, table, pages of the pool): pages of each request anywhere in the pool."""
    B, page = case["B"], case["page"]
    live = B - case.get("idle", 0)
    lens = torch.tensor(_lengths(case), dtype=torch.int32)
    lens[:live] = lens[:live][torch.randperm(live, generator=rng)]
    need = (lens + page - 1) // page
    used = int(need.sum())
    P = used + used // spare + 1
    perm = torch.randperm(P, generator=rng).to(torch.int32)
    table = torch.full((B, _pages(case["top"] + case["top"] // 4 + 1, page)), -1, dtype=torch.int32)
    first = 0
    for b, n in enumerate(need.tolist()):
        table[b, :n] = perm[first:first + n]
        first += n
    return lens, table, P


def _slots(case, P, seed, gen):
    """Slots of T tokens: one sequence's follow each other within a page, the pages are anywhere."""
    T, page = case["T"], case["page"]
    pages = torch.randperm(P, device="cuda", generator=gen)
    t = torch.arange(T, device="cuda") + int(seed) % page
    return (pages[t // page] * page + t % page).to(torch.int32)


def _prepare_append(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    T, page, D = case["T"], case["page"], case["D"]
    P = _pages(T, page) + T // (8 * page) + 2
    state = dict(slots=_slots(case, P, seed, gen), dtype=case["dtype"])
    for name in ("k", "v"):
        # (channels of their own size, as projections have them)
        size = torch.exp(torch.randn((case["Hkv"], D), device="cuda", generator=gen))
        state[name] = (torch.randn((T, case["Hkv"], D), device="cuda", generator=gen) * size
                       ).to(_DTYPES[case["dtype"]])
        state[name + "_cache"] = _empty_pool(case, P, D // 2, torch.uint8)
        state[name + "_scale"] = _empty_pool(case, P, D // 32, torch.uint8)
    return state


def _prepare_gather(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    T, page = case["T"], case["page"]
    P = _pages(T, page) + T // (8 * page) + 2
    slots = _slots(case, P, seed, gen)
    if case["spare"]:
        slots[T - case["spare"]:] = -1
    k_cache, k_scale = _pool(case, P, gen)
    v_cache, v_scale = _pool(case, P, gen)
    return dict(slots=slots, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale,
                dtype=case["dtype"])


def _queries(case, gen):
    B, Hq, N, D = (case[x] for x in ("B", "Hq", "N", "D"))
    shape = (B, N, Hq, D) if case["layout"] == "bnhd" else (B, Hq, N, D)
    q = torch.randn(shape, device="cuda", generator=gen).to(_DTYPES[case["dtype"]])
    return q.transpose(1, 2) if case["layout"] == "bnhd" else q


def _prepare_attn(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    lens, table, P = _requests(case, torch.Generator().manual_seed(int(seed)))
    k_cache, k_scale = _pool(case, P, gen)
    v_cache, v_scale = _pool(case, P, gen)
    slopes = None
    if case["alibi"]:
        slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["Hq"]) for h in range(case["Hq"])]).cuda()
    return dict(q=_queries(case, gen), k_cache=k_cache, v_cache=v_cache, k_scale=k_scale,
                v_scale=v_scale, table=table.cuda(), lens=lens.cuda(), top=max(1, int(lens.max())),
                window=case["window"], slopes=slopes, lse=case["lse"])


def _prepare_weights(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    lens, table, P = _requests(case, torch.Generator().manual_seed(int(seed)))
    k_cache, k_scale = _pool(case, P, gen)
    state = dict(q=_queries(case, gen), k_cache=k_cache, k_scale=k_scale, table=table.cuda(),
                 lens=lens.cuda(), top=max(1, int(lens.max())), restart=case["restart"])
    # What the step's attention left: the rows' sums.
    scores = _scores(state).view(-1, case["N"], state["scores_width"])
    state["lse"] = torch.cat([torch.logsumexp(x.double(), -1).float()
                              for x in scores.split(max(1, (1 << 26) // scores[0].numel()))]
                             ).view(case["B"], case["Hq"], case["N"])
    state["lse"][state["lens"] == 0] = math.inf
    # What the keys got from the rows before: some ten rows' worth.
    shape = (P, case["Hkv"], case["page"])
    one = case["Hq"] / case["Hkv"] / case["top"]
    state["weights"] = one * torch.exp(2 * torch.randn(shape, device="cuda", generator=gen))
    return state


def _prepare_evict(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    lens, table, P = _requests(case, torch.Generator().manual_seed(int(seed)))
    k_cache, _ = _pool(case, P, gen)
    v_cache, _ = _pool(case, P, gen)
    # Few keys are heavy, and many of the light ones weigh the same: nothing.
    shape = (P, case["Hkv"], case["page"])
    weights = torch.exp(2 * torch.randn(shape, device="cuda", generator=gen))
    weights = torch.where(weights < 0.2, torch.zeros_like(weights), weights)
    return dict(k_cache=k_cache, v_cache=v_cache, weights=weights, table=table.cuda(),
                lens=lens.cuda(), top=int(lens.max()), recent=case["recent"], keep=case["keep"],
                max_len=torch.full((case["B"],), case["keep"], dtype=torch.int32, device="cuda"))


_PREPARE = {"append": _prepare_append, "gather": _prepare_gather, "attn": _prepare_attn,
            "weights": _prepare_weights, "evict": _prepare_evict}


def prepare(case, seed):
    return dict(_PREPARE[case["op"]](case, seed), op=case["op"])


# ------------------------------------------------------------- the plain forms

def _quantise(x, dtype):
    """(codes, scales) of rows of values: bytes of two codes, and a byte per 32 values."""
    x = x.float().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    # The exponent of the least power of two of which `top` is 7/4 or less, less 2.
    e = ((top.view(torch.int32) + 0x1FFFFF) >> 23) - 2
    e = e.clamp(1, _TOP_SCALE[dtype])
    y = x / (e << 23).view(torch.float32)[..., None]
    a = y.abs()
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    code = (code + 8 * (torch.signbit(x) & torch.isfinite(top)[..., None])).flatten(-2)
    e = torch.where(torch.isfinite(top), e, torch.full_like(e, 255))
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), e.to(torch.uint8)


def _values(codes, scales):
    """What codes and scales stand for, in 32 bits."""
    levels = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), device=codes.device)
    x = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    size = (scales.int() << 23).view(torch.float32)
    return (levels[x].unflatten(-1, (-1, 32)) * size[..., None]).flatten(-2)


def _rows_at(cache, scale, pages, rows):
    """Rows (..., Hkv, D) of a cache, in 32 bits."""
    x = cache[pages, :, rows]
    return x.float() if scale is None else _values(x, scale[pages, :, rows])


def _append_plain(s):
    page, slots = s["k_cache"].size(2), s["slots"].long()
    out = []
    for name in ("k", "v"):
        codes, scales = _quantise(s[name], s["dtype"])
        s[name + "_cache"][slots // page, :, slots % page] = codes
        s[name + "_scale"][slots // page, :, slots % page] = scales
        out.append(_rows_at(s[name + "_cache"], s[name + "_scale"], slots // page, slots % page)
                   .to(_DTYPES[s["dtype"]]))
    return tuple(out)


def _gather_plain(s):
    page, slots = s["k_cache"].size(2), s["slots"].long()
    live = (slots >= 0)[:, None, None]
    at = slots.clamp(min=0)
    out = []
    for name in ("k", "v"):
        x = _rows_at(s[name + "_cache"], s[name + "_scale"], at // page, at % page)
        out.append(torch.where(live, x, torch.zeros_like(x)).to(_DTYPES[s["dtype"]]))
    return tuple(out)


def _batch(cache, scale, ids):
    """The rows of the pages ids (B, pages): (B, Hkv, pages * page, D), in 32 bits."""
    x = cache[ids].float() if scale is None else _values(cache[ids], scale[ids])
    return x.transpose(1, 2).flatten(2, 3)


def _page_ids(s):
    page = s["k_cache"].size(2)
    return s["table"][:, :_pages(s["top"], page)].long().clamp(min=0)


def _places(s, K):
    """The token of each row (B, 1, N, 1), and of each key."""
    N, dev = s["q"].size(2), s["q"].device
    i = (s["lens"].long()[:, None] - N + torch.arange(N, device=dev)[None, :])[:, None, :, None]
    return i, torch.arange(K, device=dev)[None, None, None, :]


def _scores(s):
    """The scaled scores (B, Hq, N, keys) under causal masking, -inf where a key is hidden."""
    q, ids = s["q"], _page_ids(s)
    B, Hq, N, D = q.shape
    k = _batch(s["k_cache"], s["k_scale"], ids)
    Hkv, K = k.size(1), k.size(2)
    x = q.float().reshape(B, Hkv, Hq // Hkv * N, D)
    scores = torch.matmul(x, k.transpose(-1, -2)).reshape(B, Hq, N, K) / math.sqrt(D)
    i, j = _places(s, K)
    s["scores_width"] = K
    return scores.masked_fill(j > i, -math.inf)


def _attn_plain(s):
    scores = _scores(s)
    B, Hq, N, K = scores.shape
    i, j = _places(s, K)
    if s["slopes"] is not None:
        scores = scores - s["slopes"][None, :, None, None] * (i - j).abs()
    if s["window"]:
        scores = scores.masked_fill(j <= i - s["window"], -math.inf)
    m = scores.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(scores - m)
    total = p.sum(-1, keepdim=True)
    v = _batch(s["v_cache"], s["v_scale"], _page_ids(s))
    o = torch.matmul(p.reshape(B, v.size(1), -1, K), v).reshape(B, Hq, N, -1)
    o = (o / torch.where(total == 0, torch.ones_like(total), total)).to(s["q"].dtype)
    if not s["lse"]:
        return o
    lse = (m + torch.log(total)).squeeze(-1)
    return o, torch.where(total.squeeze(-1) == 0, torch.full_like(lse, math.inf), lse)


def _weights_plain(s):
    scores = _scores(s)
    B, Hq, N, K = scores.shape
    Hkv, page = s["weights"].size(1), s["weights"].size(2)
    got = torch.exp(scores - s["lse"][..., None]).reshape(B, Hkv, -1, K).sum(2)
    lens = s["lens"].long()
    b, j = (torch.arange(K, device=lens.device)[None, :] < lens[:, None]).nonzero(as_tuple=True)
    pages, rows = _page_ids(s)[b, j // page], j % page
    got = got.transpose(1, 2)[b, j]  # (tokens, Hkv)
    if not s["restart"]:  # (a row's own token has no weight from before)
        got = got + torch.where((j < lens[b] - N)[:, None], s["weights"][pages, :, rows], 0.0)
    s["weights"][pages, :, rows] = got
    return s["weights"]


def _evict_plain(s):
    w, lens = s["weights"], s["lens"].long()
    page, Hkv, dev = w.size(2), w.size(1), w.device
    new = torch.minimum(lens, s["max_len"].long())
    ids = _page_ids(s)
    weight = w[ids].transpose(1, 2).flatten(2, 3)  # (B, Hkv, keys)
    K = weight.size(2)
    j = torch.arange(K, device=dev)[None, None, :]
    newest = j >= (lens - new.clamp(max=s["recent"]))[:, None, None]
    weight = torch.where(newest, math.inf, weight)
    weight = torch.where(j >= lens[:, None, None], -math.inf, weight)
    most = min(K, s["keep"])
    order = torch.sort(weight, dim=-1, descending=True, stable=True).indices[..., :most]
    to = torch.arange(most, device=dev)[None, None, :]
    live = (to < new[:, None, None]).expand_as(order)
    src = torch.where(live, order, K).sort(-1).values
    b, h, to = live.nonzero(as_tuple=True)
    src = src[b, h, to]
    from_page, to_page = ids[b, src // page], ids[b, to // page]
    for name in ("k_cache", "v_cache", "weights"):
        s[name][to_page, h, to % page] = s[name][from_page, h, src % page]
    return s["k_cache"], s["v_cache"], w, new.to(torch.int32)


_PLAIN = {"append": _append_plain, "gather": _gather_plain, "attn": _attn_plain,
          "weights": _weights_plain, "evict": _evict_plain}


# --------------------------------------------------------- the framework's calls

def _append_own(s):
    fa = _fa()
    fa.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"],
                    v_scale=s["v_scale"])
    return fa.paged_gather(s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"],
                           v_scale=s["v_scale"], dtype=s["k"].dtype)


def _gather_own(s):
    return _fa().paged_gather(s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"],
                              v_scale=s["v_scale"], dtype=_DTYPES[s["dtype"]])


def _attn_own(s):
    return _fa().paged_attn(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], causal=True,
                            sliding_window=s["window"] or None, alibi_slopes=s["slopes"],
                            return_lse=s["lse"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _weights_own(s):
    _fa().paged_weights(s["q"], s["k_cache"], s["table"], s["lens"], s["lse"], s["weights"],
                        restart=s["restart"], k_scale=s["k_scale"])
    return s["weights"]


def _evict_own(s):
    new = _fa().paged_evict(s["k_cache"], s["v_cache"], s["weights"], s["table"], s["lens"],
                            s["max_len"], recent=s["recent"])
    return s["k_cache"], s["v_cache"], s["weights"], new


_OWN = {"append": _append_own, "gather": _gather_own, "attn": _attn_own, "weights": _weights_own,
        "evict": _evict_own}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ------------------------------------------------------- what the path needs

def _row_bytes(case):
    return case["D"] // 2 + case["D"] // 32 if case["bits"] == 4 else 2 * case["D"]


def work(case):
    op, Hkv, D, page = case["op"], case["Hkv"], case["D"], case["page"]
    if op == "append":  # rows in, cache rows out, what they stand for out
        return {"bytes": 2 * case["T"] * Hkv * (2 * 2 * D + _row_bytes(case)) + 4 * case["T"], "flops": 0}
    if op == "gather":
        rows = 2 * Hkv * (case["T"] - case["spare"])
        return {"bytes": rows * _row_bytes(case) + 2 * Hkv * case["T"] * 2 * D + 4 * case["T"], "flops": 0}
    if op == "evict":  # the weights; rows that move, read and written, and their weights
        over = [n for n in _lengths(case) if n > case["keep"]]
        moved = len(over) * Hkv * case["keep"]
        return {"bytes": 4 * Hkv * sum(over) + moved * (4 * _row_bytes(case) + 4) + 12 * case["B"], "flops": 0}
    B, Hq, N = case["B"], case["Hq"], case["N"]
    window = case.get("window", 0)
    keys = pairs = pages = tokens = 0
    for n in _lengths(case):
        if n == 0:
            continue
        low = max(0, n - N + 1 - window) if window else 0
        keys += n - low
        tokens += n
        pages += _pages(n, page) - low // page
        pairs += sum(min(n - N + 1 + i, window or n) for i in range(N))
    if op == "weights":
        passes = 1 if case["restart"] else 2
        return {"bytes": 2 * B * Hq * N * D + 4 * B * Hq * N + Hkv * keys * (_row_bytes(case) + 4 * passes)
                + 4 * pages + 4 * B, "flops": 2 * D * Hq * pairs}
    return {"bytes": 2 * 2 * B * Hq * N * D + 2 * Hkv * _row_bytes(case) * keys + 4 * pages + 4 * B
            + (4 * B * Hq * N if case["lse"] else 0), "flops": 4 * D * Hq * pairs}


# ------------------------------------------------------------- in 64 bits

def _exact_rows(cache, scale, pages, h, rows):
    """Rows (tokens, D) of one kv head, in 64 bits, from the bits of their codes."""
    x = cache[pages, h, rows]
    if scale is None:
        return x.double()
    x = x.long()
    half = torch.empty(x.size(0), 2 * x.size(1), dtype=torch.int64, device=x.device)
    half[:, 0::2], half[:, 1::2] = x % 16, x // 16
    e, m = half // 2 % 4, (half % 2).double()
    size = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2((e - 1).double()))
    power = torch.exp2(scale[pages, h, rows].double() - 127).repeat_interleave(32, -1)
    return torch.where(half >= 8, -size, size) * power


def _exact_append(s):
    """Rows rounded by the steps between the levels: 1/2 up to 2, 1 up to 4, 2 above."""
    out = []
    for name in ("k", "v"):
        x = s[name].double().unflatten(-1, (-1, 32))
        mantissa, exponent = torch.frexp(x.abs().amax(-1))  # mantissa in [1/2, 1)
        exponent = exponent - 3 + (mantissa > 0.875).int()
        exponent = exponent.clamp(-126, _TOP_SCALE[s["dtype"]] - 127).double()
        y = x / torch.exp2(exponent)[..., None]
        step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
        y = (torch.round(y / step) * step).clamp(-6, 6)
        out.append((y * torch.exp2(exponent)[..., None]).flatten(-2))
    return tuple(out)


def _exact_gather(s):
    page, Hkv = s["k_cache"].size(2), s["k_cache"].size(1)
    live = (s["slots"] >= 0).nonzero().squeeze(-1)
    slots = s["slots"][live].long()
    out = []
    for name in ("k", "v"):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        D = cache.size(3) * (1 if scale is None else 2)
        x = torch.zeros((s["slots"].numel(), Hkv, D), dtype=torch.float64, device="cuda")
        for h in range(Hkv):
            x[live, h] = _exact_rows(cache, scale, slots // page, h, slots % page)
        out.append(x)
    return tuple(out)


def _exact_scores(case, s, b, g, tokens, rows):
    """The scores (group, N, keys) of one request and kv head, in 64 bits, hidden ones -inf."""
    N, page, G = case["N"], case["page"], case["Hq"] // case["Hkv"]
    where = s["table"][b].long()[tokens // page]
    keys = _exact_rows(s["k_cache"], s["k_scale"], where, g, tokens % page)
    z = s["q"][b, g * G:(g + 1) * G].double() @ keys.t().contiguous() * case["D"] ** -0.5
    at = rows[None, :, None]
    if s.get("slopes") is not None:
        z = z - s["slopes"][g * G:(g + 1) * G].double()[:, None, None] * (at - tokens).abs()
    hidden = tokens > at
    if case.get("window"):
        hidden = hidden | (tokens <= at - case["window"])
    return z.masked_fill(hidden, -math.inf), where


def _exact_attn(case, s):
    B, Hq, N, D = s["q"].shape
    G, page = Hq // case["Hkv"], case["page"]
    out = torch.zeros((B, Hq, N, D), dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, N), math.inf, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lens"].tolist()):
        if length == 0:
            continue
        start = max(0, length - N + 1 - case["window"]) if case["window"] else 0
        tokens = torch.arange(start, length, device="cuda")
        rows = length - N + torch.arange(N, device="cuda")
        for g in range(case["Hkv"]):
            z, where = _exact_scores(case, s, b, g, tokens, rows)
            values = _exact_rows(s["v_cache"], s["v_scale"], where, g, tokens % page)
            lse[b, g * G:(g + 1) * G] = torch.logsumexp(z, -1)
            out[b, g * G:(g + 1) * G] = torch.softmax(z, -1) @ values
    return (out, lse) if case["lse"] else out


def _exact_weights(case, s):
    out, N, page = s["weights"].double(), case["N"], case["page"]
    G = case["Hq"] // case["Hkv"]
    for b, length in enumerate(s["lens"].tolist()):
        if length == 0:
            continue
        tokens = torch.arange(length, device="cuda")
        rows = length - N + torch.arange(N, device="cuda")
        for g in range(case["Hkv"]):
            z, where = _exact_scores(case, s, b, g, tokens, rows)
            got = torch.exp(z - s["lse"][b, g * G:(g + 1) * G].double()[..., None]).sum((0, 1))
            old = out[where, g, tokens % page]
            fresh = case["restart"] | (tokens >= length - N)
            out[where, g, tokens % page] = torch.where(fresh, got, old + got)
    return out


def _exact_evict(case, s):
    """A request and kv head at a time: the keys by weight and then by age, the newest apart."""
    caches = [s[name].double() for name in ("k_cache", "v_cache", "weights")]
    page, lens = case["page"], s["lens"].tolist()
    for b, length in enumerate(lens):
        if length <= case["keep"]:
            continue
        old = length - min(case["recent"], case["keep"])
        for g in range(case["Hkv"]):
            tokens = torch.arange(length, device="cuda")
            where, at = s["table"][b].long()[tokens // page], tokens % page
            weight = s["weights"][where[:old], g, at[:old]].double()
            heavy = torch.argsort(-weight, stable=True)[:case["keep"] - (length - old)]
            kept = torch.cat([heavy.sort().values, tokens[old:]])
            for c in caches:
                c[where[:case["keep"]], g, at[:case["keep"]]] = c[where[kept], g, at[kept]]
    new = torch.tensor([min(n, case["keep"]) for n in lens], dtype=torch.int32, device="cuda")
    return (*caches, new)


def exact(case, seed):
    """The outputs from the operators' definitions; None where that takes too long."""
    s = _PREPARE[case["op"]](case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "gather":
        return _exact_gather(s)
    return {"attn": _exact_attn, "weights": _exact_weights, "evict": _exact_evict}[case["op"]](case, s)
