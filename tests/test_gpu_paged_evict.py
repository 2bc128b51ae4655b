"""The keys' weights of a paged cache and the eviction by them, on the GPU: weights against
float64 with their bound, evictions bit for bit (paged4_ref.py), and all operators of the
smaller caches together as a serving loop runs them. No counterpart in the reference, which
has no cache."""
import ctypes
import math

import pytest
import torch

import paged4_ref
import paged_ref
from test_gpu_paged4 import DEV, DTYPES, cache_of, fa, hide_rest, pool, rows

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ weights

def cache16(B, Hkv, D, page, lens, seed, dtype, layout="bhnd"):
    """((k_cache, None), float64 k, table) of a 16-bit cache."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + 3
    perm = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((B, max(need + [1]) + 2), 2 ** 30, dtype=torch.int32)
    used = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[used:used + n]
        used += n
    kc = pool(P, Hkv, page, D, layout, 0, dtype)
    kc.copy_(rows(kc.shape, dtype, seed))
    return (kc, None), kc.double(), table.to(DEV)


def weight_cache(four, B, Hkv, D, page, lens, seed, dtype, layout="bhnd"):
    if not four:
        return cache16(B, Hkv, D, page, lens, seed, dtype, layout)
    caches, k, _, table = cache_of(B, Hkv, D, page, lens, seed, layout)
    hide_rest(caches, table, lens, page)
    return (caches[0], caches[2]), k, table


def row_sums(q, k, table, lens, **kw):
    """The rows' lse as fp32, from float64."""
    return paged_ref.attention(q, k, k, table, lens, **kw)[1].float()


def check_weights(q, cache, k, table, lens, restart=False, layout="bhnd", lse=None, **kw):
    kc, ks = cache
    lse = row_sums(q, k, table, lens, **kw) if lse is None else lse
    w = pool(kc.size(0), kc.size(1), kc.size(2), 1, layout, 0, torch.float32)[..., 0]
    w.copy_(rows(w.shape, torch.float32, 77).abs() * 0.01)
    before = w.clone()
    names = dict(causal="causal", window="sliding_window", alibi="alibi_slopes", scale="softmax_scale")
    out = fa().paged_weights(q, kc, table, torch.tensor(lens, dtype=torch.int32, device=DEV), lse, w,
                             restart=restart, k_scale=ks, **{names[x]: v for x, v in kw.items()})
    assert out is None
    want, tol = paged4_ref.weights(q, k, table, lens, lse, before, restart=restart, **kw)
    err = (w.double() - want).abs()
    assert bool(torch.isfinite(w).all()) and bool((err <= tol).all()), \
        f"off by {err.max().item():.3e}, {(err - tol).max().item():.3e} over"
    return w, before


LENGTHS = [1, 63, 64, 65, 0, 700, 129, 17]


@pytest.mark.parametrize("restart", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,N", [(4, 4, 1), (8, 1, 1), (6, 2, 5), (12, 1, 7), (6, 2, 1), (4, 2, 2),
                                      (32, 2, 1), (34, 2, 1)])
@pytest.mark.parametrize("four,D", [(True, 32), (True, 64), (True, 96), (True, 128), (True, 160), (True, 256),
                                    (False, 8), (False, 40), (False, 64), (False, 80), (False, 128), (False, 256)])
def test_weights_match_float64(four, D, Hq, Hkv, N, dtype, restart):
    page = {8: 1, 32: 1, 40: 2, 64: 16, 80: 8, 96: 8, 128: 32, 160: 4, 256: 64}[D]
    cache, k, table = weight_cache(four, len(LENGTHS), Hkv, D, page, LENGTHS, D + N, DTYPES[dtype])
    q = rows((len(LENGTHS), Hq, N, D), DTYPES[dtype], 9)
    check_weights(q, cache, k, table, LENGTHS, restart)


@pytest.mark.parametrize("restart", [False, True])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
@pytest.mark.parametrize("four,dtype", [(True, "bf16"), (True, "fp16"), (False, "bf16")])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=5), dict(window=64, alibi=True, scale=0.3),
                                dict(causal=False, alibi=True, scale=0.02), dict(window=1)])
def test_weights_options(kw, four, dtype, layout, restart):
    lens = [3, 64, 0, 257, 1000, 66]
    cache, k, table = weight_cache(four, 6, 2, 96, 16, lens, 5, DTYPES[dtype], layout)
    q = rows((6, 3, 10, 96), DTYPES[dtype], 9).transpose(1, 2)
    if kw.get("alibi"):
        kw = dict(kw, alibi=torch.linspace(-0.1, 0.5, 10, device=DEV))
    w, before = check_weights(q, cache, k, table, lens, restart, layout, **kw)
    if kw.get("window") and not restart:  # keys that no row sees keep their weight
        at = torch.arange(1000 - 3 + 1 - kw["window"], device=DEV)
        pages = table[4].long()[at // 16]
        assert torch.equal(w[pages, :, at % 16], before[pages, :, at % 16])


@pytest.mark.parametrize("B,Hq,Hkv,N,D,top,page", [(1, 8, 1, 1, 128, 20000, 16), (2, 32, 8, 32, 128, 3000, 32),
                                                   (70, 8, 2, 1, 64, 3000, 32), (200, 4, 1, 1, 128, 400, 16),
                                                   (1, 8, 1, 200, 64, 900, 8)])
@pytest.mark.parametrize("four", [True, False])
def test_weights_of_long_and_many_requests(B, Hq, Hkv, N, D, top, page, four):
    lens = [max(N, int(top * ((0.5 + 0.618034 * i) % 1.0))) for i in range(B)]
    cache, k, table = weight_cache(four, B, Hkv, D, page, lens, B, torch.bfloat16)
    q = rows((B, Hq, N, D), torch.bfloat16, 9)
    a, _ = check_weights(q, cache, k, table, lens)
    b, _ = check_weights(q, cache, k, table, lens)
    assert torch.equal(a, b)


def test_weights_add_up_to_the_rows():
    """With paged_attn's own lse a row's weights sum to 1: a kv head's to its rows' number."""
    lens = [500, 64, 30]
    caches, k, v, table = cache_of(3, 2, 128, 16, lens, 4)
    kc, vc, ks, vs = caches
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = rows((3, 8, 2, 128), torch.bfloat16, 9)
    _, lse = fa().paged_attn(q, kc, vc, table, n, return_lse=True, k_scale=ks, v_scale=vs)
    w = torch.full((kc.size(0), 2, 16), 7.0, device=DEV)
    fa().paged_weights(q, kc, table, n, lse, w, restart=True, k_scale=ks)
    for b, length in enumerate(lens):
        at = torch.arange(length, device=DEV)
        got = w[table[b].long()[at // 16], :, at % 16].double().sum(0)
        # (8 rows; scores and lse off by at most paged4_ref's bounds: some 1e-4 each here)
        assert float((got - 8).abs().max()) < 8e-3


def test_weights_of_hidden_pages_and_nan():
    lens = [100, 64]
    for four in (True, False):
        cache, k, table = weight_cache(four, 2, 2, 64, 16, lens, 6, torch.float16)
        table[0, 2], table[1, 0] = -1, cache[0].size(0)
        q = rows((2, 4, 2, 64), torch.float16, 9)
        check_weights(q, cache, k, table, lens)
        # rows without lse add nothing, NaN rows make their request's keys NaN and no others
        lse = row_sums(q, k, table, lens)
        lse[0, 1], lse[1, 3, 1] = math.inf, math.nan
        w = torch.zeros(cache[0].shape[:3], device=DEV)
        fa().paged_weights(q, cache[0], table, torch.tensor(lens, dtype=torch.int32, device=DEV), lse, w,
                           k_scale=cache[1])
        at = torch.arange(63, device=DEV)
        mine = w[table[1].long()[at[16:] // 16], :, at[16:] % 16]
        assert bool(torch.isnan(mine[:, 1]).all()) and bool(torch.isfinite(mine[:, 0]).all())
        assert int(torch.isnan(w).sum()) == 64 - 16


# ------------------------------------------------------------------ evict

def evict_case(four, B, Hkv, D, page, lens, seed, dtype=torch.bfloat16, layout="bhnd", ties=False):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + 2
    perm = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((B, max(need + [1]) + 1), 2 ** 30, dtype=torch.int32)
    used = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[used:used + n]
        used += n
    if four:
        arrays = [pool(P, Hkv, page, w, layout) for w in (D // 2, D // 2, D // 32, D // 32)]
        for a in arrays:
            a.copy_(torch.randint(0, 256, a.shape, generator=g).to(torch.uint8))
    else:
        arrays = [pool(P, Hkv, page, D, layout, 0, dtype) for _ in range(2)]
        for i, a in enumerate(arrays):
            a.copy_(rows(a.shape, dtype, seed + i))
    w = pool(P, Hkv, page, 1, layout, 0, torch.float32)[..., 0]
    x = torch.exp(2 * torch.randn(w.shape, generator=g))
    if ties:
        x = torch.round(x)
    w.copy_(x)
    return arrays, w, table


def check_evict(arrays, w, table, lens, max_len, recent):
    kw = dict(k_scale=arrays[2], v_scale=arrays[3]) if len(arrays) == 4 else {}
    n = torch.tensor(lens, dtype=torch.int32)
    want, want_w = [a.cpu().contiguous() for a in arrays], w.cpu().contiguous()
    budget = max_len if isinstance(max_len, list) else [max_len] * len(lens)
    new = paged4_ref.evict(want, want_w, table, n, budget, recent)
    versions = [t._version for t in (*arrays, w)]
    given = torch.tensor(max_len, dtype=torch.int32, device=DEV) if isinstance(max_len, list) else max_len
    got = fa().paged_evict(arrays[0], arrays[1], w, table.to(DEV), n.to(DEV), given, recent, **kw)
    assert torch.equal(got.cpu(), new)
    for a, b in zip((*arrays, w), (*want, want_w)):
        assert torch.equal(a.cpu().contiguous().view(torch.uint8), b.view(torch.uint8))
    assert all(t._version > v for t, v in zip((*arrays, w), versions))


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd", "inner"])
@pytest.mark.parametrize("four,D,page,Hkv", [(True, 32, 1, 1), (True, 64, 16, 3), (True, 96, 2, 2), (True, 128, 32, 8),
                                             (True, 224, 8, 1), (True, 256, 64, 2), (False, 8, 4, 2),
                                             (False, 72, 16, 3), (False, 128, 16, 8), (False, 256, 128, 1)])
def test_evict_keeps_the_newest_and_heaviest(four, D, page, Hkv, layout, ties):
    lens = [1, 2, 0, 65, 700, 129, 300, 17]
    arrays, w, table = evict_case(four, len(lens), Hkv, D, page, lens, D, layout=layout, ties=ties)
    # (of a longer table: in several launches)
    long_table = torch.nn.functional.pad(table, (0, 20000 // page), value=2 ** 30)
    kept = [t.clone() for t in (*arrays, w)]
    for t in (table, long_table):
        for x, y in zip((*arrays, w), kept):
            x.copy_(y)
        for max_len, recent in ((299, 16), ([0, 1, 5, 64, 100, 129, -4, 3], 2), (40, 1000), (7, 0)):
            check_evict(arrays, w, t, lens, max_len, recent)


@pytest.mark.parametrize("B,Hkv,top,keep,recent", [(1, 2, 60000, 5000, 64), (1, 1, 9000, 8999, 0), (1, 8, 4097, 4096, 4095),
                                                   (40, 2, 1500, 200, 100), (130, 1, 90, 30, 8), (2, 1, 20000, 17000, 7),
                                                   (140, 2, 2500, 900, 50)])
@pytest.mark.parametrize("four", [True, False])
def test_evict_long_and_many(B, Hkv, top, keep, recent, four):
    lens = [max(1, int(top * ((0.5 + 0.618034 * i) % 1.0))) for i in range(B)]
    lens[0] = top
    check_evict(*evict_case(four, B, Hkv, 64, 16, lens, B, ties=True), lens, keep, recent)


def test_evict_orders_every_kind_of_weight():
    """NaN above all, -inf, zeros of both signs and subnormals among equals."""
    special = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, -math.nan, 1e-45, -1e-45, 1.0, -1.0, 1.0, 3e38])
    lens = [600]
    for seed in range(4):
        arrays, w, table = evict_case(False, 1, 2, 64, 8, lens, seed)
        pick = torch.randint(0, len(special), w.shape, generator=torch.Generator().manual_seed(seed))
        w.copy_(special[pick])
        for keep in (550, 333, 150, 20):
            check_evict(arrays, w, table, lens, keep, 3)
    # all alike: the oldest stay
    arrays, w, table = evict_case(False, 1, 2, 64, 8, lens, 9)
    w.fill_(0.25)
    check_evict(arrays, w, table, lens, 100, 10)


@pytest.mark.parametrize("four", [True, False])
def test_evict_of_all_with_any_workspace(four):
    """Nothing is kept, and what the workspace held does not matter."""
    lens = [300, 40000, 1]
    case = evict_case(four, 3, 2, 64, 16, lens, 4)
    size = 3 * 2 * (case[2].size(1) * 16 + 2)
    for junk in (0, 2 ** 20, -2 ** 20):
        torch.full((size,), junk, dtype=torch.int32, device=DEV)  # (freed, and allocated again)
        check_evict(*case, lens, 0, 5)


def test_evict_with_pages_outside_the_pool():
    """Their tokens are the lightest, and nothing is read or written there."""
    lens = [200, 64]
    arrays, w, table = evict_case(True, 2, 2, 64, 16, lens, 3)
    table[0, 1], table[0, 7], table[1, 0], table[1, 3] = -1, w.size(0), 2 ** 31 - 1, -2 ** 31
    for keep in (150, 40, 20):
        check_evict(arrays, w, table, lens, keep, 30)


@pytest.mark.parametrize("four", [True, False])
def test_pages_past_32_bits(four):
    """Pools of more than 2^32 bytes: as in a small one, with the same pages near the end."""
    Hkv, page, D, n = 8, 256, 256, 700
    row = [D // 2, D // 2, D // 32, D // 32] if four else [D, D]
    dtype = torch.uint8 if four else torch.bfloat16
    P = (1 << 32) // (Hkv * page * D // (2 if four else 1)) + 9
    ends = torch.tensor([P - 1, P - 4, P - 2], device=DEV)
    if four:
        small = [torch.randint(1, 120, (3, Hkv, page, w), dtype=dtype, device=DEV) for w in row]
    else:
        small = [rows((3, Hkv, page, w), dtype, w) for w in row]
    w = rows((3, Hkv, page), torch.float32, 7).abs()
    q, lens = rows((1, 16, 3, D), torch.bfloat16, 5), torch.tensor([n], dtype=torch.int32, device=DEV)
    lse = torch.full((1, 16, 3), 6.0, device=DEV)

    def step(arrays, w, table):
        four_args = dict(k_scale=arrays[2], v_scale=arrays[3]) if four else {}
        fa().paged_weights(q, arrays[0], table, lens, lse, w, k_scale=arrays[2] if four else None)
        fa().paged_evict(arrays[0], arrays[1], w, table, lens, 300, recent=9, **four_args)

    large = [torch.empty(P, *x.shape[1:], dtype=x.dtype, device=DEV) for x in (*small, w)]
    for x, y in zip(large, (*small, w)):
        x[ends] = y
    step(large[:-1], large[-1], ends[None].to(torch.int32))
    step(small, w, torch.arange(3, dtype=torch.int32, device=DEV)[None])
    for x, y in zip(large, (*small, w)):
        assert torch.equal(x[ends].contiguous().view(torch.uint8), y.view(torch.uint8))


def test_evict_captured_and_on_another_stream():
    lens = [500, 80, 333]
    case = evict_case(True, 3, 2, 128, 16, lens, 5)
    arrays, w, table = case[0], case[1], case[2].to(DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    first = [t.clone() for t in (*arrays, w)]
    q, lse = rows((3, 4, 1, 128), torch.bfloat16, 1), torch.zeros(3, 4, 1, device=DEV)

    def step():
        fa().paged_weights(q, arrays[0], table, n, lse, w, k_scale=arrays[2])
        return fa().paged_evict(arrays[0], arrays[1], w, table, n, 100, 10, k_scale=arrays[2], v_scale=arrays[3])

    def reset(i):
        for t, x in zip((*arrays, w), first):
            t.copy_(x)
        arrays[2].fill_(120)
        w.copy_(torch.exp(torch.randn(w.shape, generator=torch.Generator().manual_seed(i))).to(DEV))
        n.copy_(torch.tensor([500 - i, 80, 101 + i], dtype=torch.int32))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        reset(0)
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        reset(i)
        graph.replay()
        got = [t.clone() for t in (out, *arrays, w)]
        reset(i)
        new = step()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, (new, *arrays, w))), i


def test_evict_refusals():
    lens = [20, 5]
    arrays, w, table = evict_case(True, 2, 2, 64, 16, lens, 2)
    kc, vc, ks, vs = arrays
    table, n = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    four = dict(k_scale=ks, v_scale=vs)
    f = fa().paged_evict
    for args, kw in (((kc, vc, w.double(), table, n, 4), four), ((kc, vc, w[:1], table, n, 4), four),
                     ((kc, vc, w.cpu(), table, n, 4), four), ((kc, vc, w, table, n.long(), 4), four),
                     ((kc, vc, w, table[:1], n, 4), four), ((kc, vc, w, table, n, n[:1]), four),
                     ((kc, vc, w, table, n, n.float()), four), ((kc, vc, w, table, n, 4, -1), four),
                     ((kc, vc, w, table, n, 4), {}), ((kc, kc, w, table, n, 4), four),
                     ((kc, vc, w[:1].expand(w.shape), table, n, 4), four),
                     ((kc, vc, w, table, n, 4), dict(k_scale=ks, v_scale=ks))):
        with pytest.raises(RuntimeError):
            f(*args, **kw)
    q, lse = rows((2, 4, 1, 64), torch.float16, 9), torch.zeros(2, 4, 1, device=DEV)
    g = fa().paged_weights
    for args, kw in (((q, kc, table, n, lse[:1], w), dict(k_scale=ks)), ((q, kc, table, n, lse.half(), w), dict(k_scale=ks)),
                     ((q, kc, table, n, lse, w[:1]), dict(k_scale=ks)), ((q, kc, table, n, lse, w), {}),
                     ((q[..., :32].contiguous(), kc, table, n, lse, w), dict(k_scale=ks)),
                     ((q, kc, table, n, lse, w[:1].expand(w.shape)), dict(k_scale=ks)),
                     ((q, kc, table, n[:1], lse, w), dict(k_scale=ks)),
                     ((q.bfloat16(), kc.half(), table, n, lse, w), {})):
        with pytest.raises(RuntimeError):
            g(*args, **kw)
    with pytest.raises(RuntimeError, match="no backward"):
        g(q, kc, table, n, lse, w.clone().requires_grad_(), k_scale=ks)


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("four", [True, False])
def test_a_serving_loop_with_a_budget(four, dtype):
    """Prompts enter, every step appends a token, attends, adds up the keys' weights, cuts
    what is over the budget and gives the pages back, all on the device; attention is
    checked against float64 over the rows that each kv head still has."""
    dt, page, Hq, Hkv, D, B, P = DTYPES[dtype], 8, 8, 2, 64, 5, 90
    budget, recent = 40, 8
    f = fa()
    if four:
        kc, vc, ks, vs = (torch.zeros(P, Hkv, page, w, dtype=torch.uint8, device=DEV) for w in (D // 2, D // 2, D // 32, D // 32))
        both, k_only = dict(k_scale=ks, v_scale=vs), dict(k_scale=ks)
    else:
        kc, vc = (torch.zeros(P, Hkv, page, D, dtype=dt, device=DEV) for _ in range(2))
        both, k_only = {}, {}
    i32 = dict(dtype=torch.int32, device=DEV)
    w = torch.full((P, Hkv, page), math.nan, device=DEV)
    table, lens = torch.zeros(B, 12, **i32), torch.zeros(B, **i32)
    free, ring = torch.arange(P, **i32), torch.tensor([0, P], **i32)
    prompts = torch.tensor([60, 1, 33, 90, 48], **i32)
    kept = [[[] for _ in range(Hkv)] for _ in range(B)]  # (k, v) rows that a head still has
    slots, kv_len, ring = f.paged_tables(table, lens, prompts, free, ring, page, max_new=90)
    assert torch.equal(kv_len, prompts)
    k, v = rows((B, Hkv, 90, D), dt, 1), rows((B, Hkv, 90, D), dt, 2)
    f.paged_append(k, v, kc, vc, slots, **both)
    x, y = f.paged_gather(kc, vc, slots, dtype=dt, **both)  # what the cache holds of them
    for b in range(B):
        for g in range(Hkv):
            kept[b][g] = [(x[b, g, i].double(), y[b, g, i].double()) for i in range(int(prompts[b]))]
    lens = kv_len
    for step in range(30):
        new = lens + 1
        slots, kv_len, ring = f.paged_tables(table, lens, new, free, ring, page, max_new=1)
        assert torch.equal(kv_len, new)
        k, v, q = (rows((B, h, 1, D), dt, 100 + 3 * step + i) for i, h in enumerate((Hkv, Hkv, Hq)))
        f.paged_append(k, v, kc, vc, slots, **both)
        x, y = f.paged_gather(kc, vc, slots, dtype=dt, **both)
        o, lse = f.paged_attn(q, kc, vc, table, kv_len, return_lse=True, **both)
        f.paged_weights(q, kc, table, kv_len, lse, w, restart=step == 0, **k_only)
        for b in range(B):
            for g in range(Hkv):
                kept[b][g].append((x[b, g, 0].double(), y[b, g, 0].double()))
                n = len(kept[b][g])
                assert n == int(kv_len[b])
                heads = slice(g * Hq // Hkv, (g + 1) * Hq // Hkv)
                kk, vv = (torch.stack([r[i] for r in kept[b][g]])[None, None] for i in (0, 1))
                one = torch.zeros(1, 1, dtype=torch.int32)
                pad = 1 << (n - 1).bit_length()
                kk, vv = (torch.nn.functional.pad(t, (0, 0, 0, pad - n)) for t in (kk, vv))
                ref = paged4_ref.attention(q[b:b + 1, heads], kk, vv, one, [n])
                paged_ref.check(o[b:b + 1, heads], lse[b:b + 1, heads], ref)
        # each head's choice, from its weights
        at = [torch.arange(int(n), device=DEV) for n in kv_len]
        weight = [w[table[b].long()[at[b] // page], :, at[b] % page].t() for b in range(B)]
        cut = f.paged_evict(kc, vc, w, table, kv_len, budget, recent, **both)
        for b in range(B):
            assert int(cut[b]) == min(int(kv_len[b]), budget)
            if int(kv_len[b]) <= budget:
                continue
            for g in range(Hkv):
                n = int(kv_len[b])
                assert bool(torch.isfinite(weight[b][g]).all())
                heavy = torch.sort(weight[b][g][:n - recent], descending=True, stable=True).indices[:budget - recent]
                index = heavy.sort().values.tolist() + list(range(n - recent, n))
                kept[b][g] = [kept[b][g][i] for i in index]
        _, lens, ring = f.paged_tables(table, kv_len, cut, free, ring, page, max_new=0)
        assert torch.equal(lens, cut)
    held = sum(-(-int(n) // page) for n in lens)
    assert int(ring[1]) == P - held


@pytest.mark.parametrize("width", [1, 4000])
def test_new_lengths_in_the_budgets_place(width):
    """By the C entry: in one launch and in three, with several kv heads to a request."""
    from test_paged4_cpu import capi4
    from test_paged_cpu import Cache
    lens, budget = [700, 3, 0, 650, 64, 900], [100, 40, 5, 64, -3, 899]
    B, Hkv, D, page = len(lens), 3, 64, 16
    arrays, w, table = evict_case(False, B, Hkv, D, page, lens, 21)
    table = torch.nn.functional.pad(table, (0, width), value=2 ** 30)
    want, want_w = [a.cpu() for a in arrays], w.cpu()
    new = paged4_ref.evict(want, want_w, table, lens, budget, 16)
    n, both = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, budget))
    t = table.to(DEV)
    lib = capi4()
    nbytes = lib.fa_paged_evict_workspace_bytes(B, Hkv, t.size(1), page)
    ws = torch.full((nbytes,), 0x7f, dtype=torch.uint8, device=DEV)
    cache = Cache(arrays[0].data_ptr(), arrays[1].data_ptr(), *arrays[0].stride()[:3], arrays[0].size(0), page,
                  t.data_ptr(), t.size(1), t.size(1), n.data_ptr())
    assert lib.fa_paged_evict(ctypes.byref(cache), None, w.data_ptr(), *w.stride(), both.data_ptr(), 16,
                              both.data_ptr(), ws.data_ptr(), nbytes, B, Hkv, D,
                              torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(both.cpu(), new)
    for a, b in zip((*arrays, w), (*want, want_w)):
        assert torch.equal(a.cpu(), b)
