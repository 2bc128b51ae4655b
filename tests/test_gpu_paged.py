"""Paged key/value caches on the GPU: tables and slots against a loop over requests,
cache writes bit for bit, attention against float64 with the bounds its rounding
allows (paged_ref.py), and the three together as a serving loop runs them. No
counterpart in the reference, which has no cache."""
import math

import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


def fa():
    import fa_p100
    return fa_p100


# ------------------------------------------------------------------ tables

def table_inputs(B, page, top, pool, seed, mix):
    """Requests with pages and new lengths; `mix` picks how they change."""
    g = torch.Generator().manual_seed(seed)
    M = -(-top // page) + 2
    old = torch.randint(0, top + 1, (B,), generator=g)
    if mix == "enter":
        old = torch.zeros_like(old)
    have = (old + page - 1) // page
    while int(have.sum()) > pool:  # fits the pool
        old //= 2
        have = (old + page - 1) // page
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((B, M), -7, dtype=torch.int32)
    used = 0
    for b, n in enumerate(have.tolist()):
        table[b, :n] = perm[used:used + n]
        used += n
    other = torch.randint(0, top + 1, (B,), generator=g)
    pick = torch.randint(0, 5, (B,), generator=g)
    new = {"step": old + 1, "enter": other, "same": old.clone(), "draft": old + pick,
           "mixed": torch.where(pick == 0, torch.zeros_like(old), torch.where(pick == 1, other, old + pick)),
           "past": old + (M + 1) * page, "negative": torch.full_like(old, -3)}[mix]
    C = pool + 3
    head = int(torch.randint(0, C, (), generator=g))
    free = torch.full((C,), -9, dtype=torch.int32)
    free[(head + torch.arange(pool - used)) % C] = perm[used:]
    return table, old.to(torch.int32), new.to(torch.int32), free, torch.tensor(
        [head, pool - used], dtype=torch.int32)


def check_tables(table, old, new, free, ring, page, **kw):
    want = paged_ref.tables(table, old, new, free, ring, page, **kw)
    wide = torch.full((table.size(0), table.size(1) + 5), -11, dtype=torch.int32, device=DEV)
    t = wide[:, 2:2 + table.size(1)]  # rows apart, entries around them
    t.copy_(table)
    f, r = free.to(DEV), ring.to(DEV)
    for _ in range(2):  # the same inputs again: the same results
        slots, kv_len, ring_out = fa().paged_tables(t, old.to(DEV), new.to(DEV), f, r, page, **kw)
        got = [x.cpu() for x in (t, f, slots, kv_len, ring_out)]
        for name, a, b in zip(("table", "free", "slots", "kv_len", "ring"), got, want):
            assert torch.equal(a, b), name
    assert torch.equal(r.cpu(), ring)
    assert bool((wide[:, :2] == -11).all()) and bool((wide[:, -3:] == -11).all())
    return want


@pytest.mark.parametrize("mix", ["step", "enter", "same", "draft", "mixed", "past", "negative"])
@pytest.mark.parametrize("B,page,top,pool", [(1, 16, 100, 40), (3, 1, 20, 80), (64, 16, 300, 900),
                                             (257, 8, 60, 2500), (1000, 4, 30, 9000)])
def test_tables_match_the_loop(B, page, top, pool, mix):
    inputs = table_inputs(B, page, top, pool, seed=B + len(mix), mix=mix)
    check_tables(*inputs, page, max_new=3)
    check_tables(*inputs, page, max_new=0)
    want = check_tables(*inputs, page, tokens=B * top // 2 + 7)
    if mix == "mixed" and B >= 64:
        assert bool((want[3] < inputs[2]).any()) or bool((want[2] >= 0).any())


@pytest.mark.parametrize("B,pool", [(40, 100), (300, 700)])
def test_tables_when_pages_run_out(B, pool):
    """Pages go to the first requests in order; the one in between gets a part."""
    inputs = table_inputs(B, 4, 64, pool, seed=B, mix="enter")
    for kw in (dict(max_new=70), dict(tokens=64 * B)):
        _, _, _, kv_len, ring = check_tables(*inputs, 4, **kw)
        assert int(ring[1]) == 0 and bool((kv_len < inputs[2]).any())


def test_tables_long_prompt_and_many_tokens():
    inputs = table_inputs(5, 16, 131072, 50000, seed=2, mix="enter")
    check_tables(*inputs, 16, tokens=400000)
    check_tables(*inputs, 16, max_new=131072)


def test_tables_with_a_ring_out_of_bounds():
    """A head past the ring is taken modulo, a count past it clamped; nothing is
    written outside the ring."""
    table, old, new, free, ring = table_inputs(9, 4, 40, 200, seed=8, mix="mixed")
    for head, count in ((-5, 60), (10 ** 9, 60), (3, 10 ** 9), (3, -4)):
        check_tables(table, old, new, free, torch.tensor([head, count], dtype=torch.int32), 4,
                     tokens=300)


def test_tables_refusals():
    t, old, new, free, ring = (x.to(DEV) for x in table_inputs(4, 16, 100, 60, seed=1, mix="step"))
    f = fa().paged_tables
    for kw in (dict(), dict(max_new=1, tokens=4), dict(max_new=-1), dict(tokens=-1)):
        with pytest.raises(RuntimeError):
            f(t, old, new, free, ring, 16, **kw)
    for bad in ((t.long(), old, new, free, ring, 16), (t, old[:3], new, free, ring, 16),
                (t, old.cpu(), new, free, ring, 16), (t, old, new, free[:0], ring, 16),
                (t, old, new, free, ring[:1], 16), (t, old, new, free, ring, 24),
                (t, old, new, free, ring, 0), (t[0], old, new, free, ring, 16),
                (t, old, new, free[::2], ring, 16), (t.t(), old, new, free, ring, 16),
                (t[:1].expand(4, -1), old, new, free, ring, 16),
                (t, old, new, free, ring, 1 << 30)):
        with pytest.raises(RuntimeError):
            f(*bad, max_new=1)
    for kw in (dict(page_size=1 << 62, max_new=1), dict(page_size=16, max_new=1 << 62),
               dict(page_size=16, tokens=1 << 62)):  # (products past 64 bits)
        with pytest.raises(RuntimeError, match="2\\^30|2\\^31"):
            f(t, old, new, free, ring, **kw)


# ------------------------------------------------------------------ append

def pool_of(P, Hkv, page, D, dtype, layout, fill=None, seed=0):
    """(k_cache, v_cache) as (P, Hkv, page, D) views: dense, rows before heads, or
    the halves of one pool."""
    g = torch.Generator().manual_seed(seed)

    def make(*shape):
        return (torch.full(shape, fill) if fill is not None else torch.randn(shape, generator=g)).to(dtype).to(DEV)

    if layout == "bnhd":
        return [make(P, page, Hkv, D).transpose(1, 2) for _ in range(2)]
    if layout == "halves":
        both = make(P, 2, Hkv, page, D)
        return [both[:, 0], both[:, 1]]
    if layout == "wide":  # rows and heads apart
        both = make(2, P, Hkv + 1, page, D + 16)
        return [x[:, 1:, :, 8:8 + D] for x in both]
    return [make(P, Hkv, page, D) for _ in range(2)]


@pytest.mark.parametrize("layout", ["bhnd", "bnhd", "halves", "wide"])
@pytest.mark.parametrize("T,Hkv,D,page,dtype", [
    (1, 1, 8, 1, torch.half), (37, 3, 80, 4, torch.bfloat16), (1, 8, 128, 16, torch.bfloat16),
    (300, 2, 256, 32, torch.half), (1000, 5, 40, 16, torch.half)])
def test_append_matches_indexing(T, Hkv, D, page, dtype, layout):
    g = torch.Generator().manual_seed(T)
    P = T // page * 2 + 3
    slots = torch.randperm(P * page, generator=g)[:T].to(torch.int32)
    slots[torch.rand(T, generator=g) < 0.2] = -1
    for i, bad in enumerate((P * page, -100, 2 ** 31 - 1)):
        if T > 30:
            slots[i * 7] = bad
    k, v = (torch.randn(T, Hkv, D, generator=g).to(dtype) for _ in range(2))
    for form in ("rows", "sliced", "batched", "odd"):
        kc, vc = pool_of(P, Hkv, page, D, dtype, layout, seed=T)
        want = [kc.clone(), vc.clone()]
        live = (slots >= 0) & (slots < P * page)
        at = slots[live].long().to(DEV)
        for c, x in zip(want, (k, v)):
            c[at // page, :, at % page] = x[live].to(DEV)
        a, b, s = k.to(DEV), v.to(DEV), slots.to(DEV)
        if form == "sliced":  # as the projections of one product: rows apart
            both = torch.cat([a.flatten(1), b.flatten(1)], 1)
            a, b = (x.unflatten(1, (Hkv, D)) for x in both.chunk(2, 1))
        elif form == "batched":
            if T % 20:
                continue
            a, b = (x.unflatten(0, (20, T // 20)).transpose(1, 2) for x in (a, b))
            s = s.view(20, T // 20)
        elif form == "odd":  # rows that no 16-byte load can take
            a = torch.cat([a[..., :1], a], -1)[..., 1:]
        fa().paged_append(a, b, kc, vc, s)
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]), form


@pytest.mark.parametrize("Hkv,D,dtype", [(8, 128, torch.bfloat16), (3, 200, torch.half)])
def test_append_of_many_tokens(Hkv, D, dtype):
    """Prompts of more rows than L2 holds, with padding behind them: every row of the
    pool either written or as it was."""
    T, page = 20011, 32
    g = torch.Generator(device=DEV).manual_seed(D)
    P = T // page + 60
    slots = torch.randperm(P * page, device=DEV, generator=g)[:T].to(torch.int32)
    slots[-77:] = -1
    kc, vc = (torch.randn(P, Hkv, page, D, device=DEV, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(T, Hkv, D, device=DEV, generator=g).to(dtype) for _ in range(2))
    want = [kc.clone(), vc.clone()]
    at = slots[:-77].long()
    for c, x in zip(want, (k, v)):
        c[at // page, :, at % page] = x[:-77]
    fa().paged_append(k, v, kc, vc, slots)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_append_of_nothing_and_refusals():
    f = fa().paged_append
    kc, vc = pool_of(4, 2, 16, 64, torch.half, "bhnd")
    before = kc.clone()
    k = torch.zeros(3, 2, 64, dtype=torch.half, device=DEV)
    s = torch.arange(3, dtype=torch.int32, device=DEV)
    f(k[:0], k[:0], kc, vc, s[:0])
    f(k, k, kc, vc, s - 3)
    assert torch.equal(kc, before)
    for bad in ((k.float(), k.float(), kc, vc, s), (k, k.bfloat16(), kc, vc, s), (k, k[:2], kc, vc, s),
                (k, k, kc.bfloat16(), vc, s), (k, k, kc, vc[:3], s), (k, k, kc, vc, s[:2]),
                (k, k, kc, vc, s.long()), (k, k, kc, vc, s.cpu()), (k[:, :1], k[:, :1], kc, vc, s),
                (k[..., :60], k[..., :60], kc[..., :60], vc[..., :60], s),
                (k, k, kc[:, :, :12], vc[:, :, :12], s), (k, k, kc.transpose(2, 3), vc, s),
                (k, k, kc, vc.transpose(1, 2).contiguous().transpose(1, 2), s),
                (k[None], k[None], kc, vc, s), (k.requires_grad_(), k, kc, vc, s)):
        with pytest.raises(RuntimeError):
            f(*bad)
    versions = kc._version, vc._version
    with torch.no_grad():
        f(k, k, kc, vc, s)  # (requires grad)
    assert kc._version > versions[0] and vc._version > versions[1]
    assert torch.equal(kc[0, :, :3].transpose(0, 1), k)


def test_append_refuses_caches_whose_rows_are_shared():
    k = torch.zeros(3, 2, 64, dtype=torch.half, device=DEV)
    s = torch.arange(3, dtype=torch.int32, device=DEV)
    one, whole = pool_of(1, 2, 16, 64, torch.half, "bhnd", fill=1.0)[0], pool_of(4, 1, 16, 64, torch.half, "bhnd")[0]
    for kc in (one.expand(4, -1, -1, -1), whole.expand(-1, 2, -1, -1), whole[:, :, :1].expand(-1, 2, 16, -1)):
        with pytest.raises(RuntimeError, match="single memory location"):
            fa().paged_append(k, k, kc, kc, s)
    assert bool((one == 1).all())


# --------------------------------------------------------------- attention

def attn_inputs(lens, Hq, Hkv, N, D, page, dtype, layout="bhnd", seed=0, spare=2, peaked=1.0):
    """q, caches, table, kv_len: pages anywhere in the pool, every row that no
    request owns NaN, table entries past a request's pages out of the pool."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    need = [-(-n // page) for n in lens]
    P = sum(need) + 3
    perm = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((B, max(need + [1]) + spare), 10 ** 9, dtype=torch.int32)
    used = 0
    kc, vc = pool_of(P, Hkv, page, D, dtype, layout, fill=float("nan"))
    for b, n in enumerate(lens):
        table[b, :need[b]] = perm[used:used + need[b]]
        used += need[b]
        if n == 0:
            continue
        j = torch.arange(n)
        at = table[b, j // page].long()
        for c in (kc, vc):
            c[at.to(DEV), :, (j % page).to(DEV)] = torch.randn(n, Hkv, D, generator=g).to(dtype).to(DEV)
    q = (torch.randn(B, Hq, N, D, generator=g) * peaked).to(dtype).to(DEV)
    if layout == "bnhd":
        q = q.transpose(1, 2).contiguous().transpose(1, 2)
    return q, kc, vc, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)


def check_attn(args, causal=True, window=None, alibi=None, scale=None):
    q = args[0]
    o, lse = fa().paged_attn(*args, causal=causal, sliding_window=window, alibi_slopes=alibi,
                             softmax_scale=scale, return_lse=True)
    assert o.dtype == q.dtype and o.shape == q.shape and o.stride() == q.stride()
    paged_ref.check(o, lse, paged_ref.attention(*args, causal, window, alibi, scale))
    alone = fa().paged_attn(*args, causal=causal, sliding_window=window, alibi_slopes=alibi,
                            softmax_scale=scale)
    assert torch.equal(alone, o)
    return o, lse


LENS = [1, 2, 31, 32, 33, 64, 100, 257, 1000]


@pytest.mark.parametrize("dtype", [torch.half, torch.bfloat16])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 80, 96, 128, 200, 256])
def test_attn_head_dims(D, dtype):
    check_attn(attn_inputs(LENS, 6, 2, 1, D, 16, dtype, seed=D))


@pytest.mark.parametrize("page", [1, 2, 8, 32, 64, 512])
@pytest.mark.parametrize("layout", ["bhnd", "bnhd", "halves", "wide"])
def test_attn_pages_and_layouts(page, layout):
    check_attn(attn_inputs([5, 700, 0, 64, 513], 4, 4, 2, 64, page, torch.half, layout, seed=page))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 1), (16, 8), (33, 1), (40, 1), (12, 12), (71, 1)])
@pytest.mark.parametrize("N", [1, 5, 17])
def test_attn_heads_and_rows(Hq, Hkv, N):
    """Row tiles that hold one head's rows, several heads' or a part of one's; entries
    shorter than N (their first rows see no key)."""
    for causal in (True, False):
        check_attn(attn_inputs([3, 40, 330, 1, 0], Hq, Hkv, N, 64, 16, torch.bfloat16, seed=N + Hq),
                   causal)


@pytest.mark.parametrize("N", [1, 4, 40])
@pytest.mark.parametrize("window", [1, 16, 33, 300, 10 ** 9])
def test_attn_windows_read_nothing_behind_them(N, window):
    """Pages wholly outside every row's window are out of the pool in the table."""
    lens, page = [7, 64, 900, 2000, 0], 16
    q, kc, vc, table, kv_len = attn_inputs(lens, 4, 2, N, 64, page, torch.half, seed=window % 97)
    for b, n in enumerate(lens):
        first = max(0, n - N + 1 - window) // page
        table[b, :first] = -1
    check_attn((q, kc, vc, table, kv_len), window=window)
    check_attn((q, kc, vc, table, kv_len), window=window,
               alibi=torch.tensor([0.3, 0.0, 0.05, 1.0], device=DEV))


def test_attn_alibi_scale_and_dense():
    args = attn_inputs([1, 50, 1500], 8, 2, 3, 128, 32, torch.bfloat16, seed=4)
    slopes = torch.tensor([2.0 ** -h for h in range(8)], device=DEV)
    for causal in (True, False):
        check_attn(args, causal, alibi=slopes)
        check_attn(args, causal, scale=0.3)
        check_attn(args, causal, alibi=slopes, scale=0.02)


def test_attn_peaked_scores():
    """Scores up to a few hundred: the running maximum moves by large steps."""
    check_attn(attn_inputs([3000, 77], 4, 2, 2, 128, 16, torch.half, seed=9, peaked=20.0))
    check_attn(attn_inputs([3000, 77], 4, 2, 2, 128, 16, torch.bfloat16, seed=9, peaked=20.0))


@pytest.mark.parametrize("lens", [[1], [60000], [9000, 3, 1, 20000, 0, 5], [2500] * 40,
                                  [17 * i % 701 for i in range(600)], [0, 0, 0]])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (4, 4)])
def test_attn_batches_split_and_joined(lens, Hq, Hkv):
    """One long request, ragged batches, more requests than workgroups, none."""
    check_attn(attn_inputs(lens, Hq, Hkv, 1, 64, 16, torch.half, seed=len(lens)))


@pytest.mark.parametrize("lens,Hq,Hkv,N,D", [
    ([9000, 3, 700], 32, 1, 1, 256),                     # 32 rows of 256: every part run of a join
    ([5000, 1, 40], 7, 1, 5, 256),                       # 35 rows: a tile of three
    ([13 * i % 400 for i in range(300)], 8, 1, 1, 128),  # more items than stretches' workgroups
    ([3 * i % 50 for i in range(4500)], 1, 1, 1, 32),    # requests past 64 runs of 64
    ([40000] * 3, 16, 2, 4, 64)])
def test_attn_wide_tiles_and_large_batches(lens, Hq, Hkv, N, D):
    check_attn(attn_inputs(lens, Hq, Hkv, N, D, 16, torch.bfloat16, seed=D))


@pytest.mark.parametrize("lens,Hkv,D", [
    # 256 workgroups of one to three blocks: few requests, whose workgroups' parts are
    # joined first, and many, whose blocks are
    ([8100], 1, 128), ([12000], 1, 64), ([20000], 1, 128), ([24500], 1, 32), ([30, 24000], 1, 96),
    ([8000], 2, 256), ([5000, 5100, 4900], 1, 256), ([2040] * 8, 1, 128), ([2060] * 8, 1, 128),
    ([600] * 8, 4, 64), ([1, 700, 0, 650, 33] * 4, 2, 128), ([31 * i for i in range(40)], 1, 64),
    # (the join's narrow runs: one item of few and of many parts, a tile of few columns)
    ([50000], 1, 128), ([90000, 0], 1, 64), ([300, 7000], 2, 32), ([100, 90], 1, 16), ([40000], 2, 256)])
def test_attn_short_stretches(lens, Hkv, D):
    for N in (1, 3):
        check_attn(attn_inputs(lens, 4 * Hkv, Hkv, N, D, 32, torch.half, seed=N))


@pytest.mark.parametrize("D", [32, 64, 80, 128, 256])
@pytest.mark.parametrize("lens,Hq,Hkv,N", [
    ([9000, 3, 700], 7, 1, 5),                  # two row tiles, the second of three rows
    ([5000], 33, 1, 2), ([50, 0, 1300], 48, 2, 3),  # three
    ([40, 2000, 333], 8, 1, 15), ([70000], 16, 1, 10),  # four, five
    ([3, 800, 90], 4, 2, 100),                  # seven, and requests shorter than N
    ([41 * i for i in range(24)], 16, 2, 5), ([300] * 100, 40, 1, 1)])
def test_attn_row_tiles_abreast(lens, Hq, Hkv, N, D):
    """Full tables past 16 MB: the row tiles of a kv head go side by side."""
    spare = (16 << 20) // (4 * Hkv * D * 16) // len(lens) + 2
    args = attn_inputs(lens, Hq, Hkv, N, D, 16, torch.bfloat16, seed=N, spare=spare)
    check_attn(args)
    if N > 1:
        check_attn(args, causal=False)
        check_attn(args, window=60, alibi=torch.rand(Hq, device=DEV))


@pytest.mark.parametrize("seed", range(48))
def test_attn_random_calls(seed):
    """Every option crossed at random, requests shorter than N and pages outside the
    pool among them."""
    import random
    r = random.Random(seed)
    Hkv = r.choice([1, 1, 2, 3, 8])
    Hq, N = Hkv * r.choice([1, 2, 5, 8]), r.choice([1, 1, 1, 2, 6, 33])
    D, page = r.choice([16, 32, 64, 72, 96, 128, 128, 256]), 2 ** r.randint(0, 7)
    top = r.choice([3, 90, 1200, 6000])
    lens = [r.randint(0, top) for _ in range(r.choice([1, 2, 5, 20]))]
    causal = r.random() < 0.7
    window = r.choice([None, None, 1, 30, 700]) if causal else None
    alibi = torch.tensor([r.random() for _ in range(Hq)], device=DEV) if r.random() < 0.3 else None
    print(seed, lens, Hq, Hkv, N, D, page, causal, window, flush=True)
    args = attn_inputs(lens, Hq, Hkv, N, D, page, r.choice([torch.half, torch.bfloat16]),
                       r.choice(["bhnd", "bnhd", "halves", "wide"]), seed, r.randint(0, 3),
                       r.choice([1.0, 1.0, 8.0]))
    if r.random() < 0.3:
        args[3][torch.rand(args[3].shape, generator=torch.Generator().manual_seed(seed)).to(DEV) < 0.1] = -1
    check_attn(args, causal, window, alibi, r.choice([None, 0.05]))


@pytest.mark.parametrize("seed", range(24))
def test_attn_random_row_tiles(seed):
    """Two to nine row tiles per kv head, in tables large enough to take them abreast."""
    import random
    r = random.Random(100 + seed)
    Hkv, group, N = r.choice([(1, 8, 5), (1, 3, 33), (2, 16, 4), (1, 64, 1), (3, 5, 17), (1, 16, 16), (2, 2, 65)])
    D, page = r.choice([16, 64, 72, 128, 128, 256]), 2 ** r.randint(0, 6)
    top = r.choice([20, 300, 3000, 12000])
    lens = [r.randint(0, top) for _ in range(r.choice([1, 3, 12, 90 if top < 1000 else 6]))]
    causal = r.random() < 0.7
    window = r.choice([None, None, 40, 900]) if causal else None
    print(seed, lens, Hkv, group, N, D, page, causal, window, flush=True)
    spare = (16 << 20) // (4 * Hkv * D * page) // len(lens) + 2
    args = attn_inputs(lens, Hkv * group, Hkv, N, D, page, r.choice([torch.half, torch.bfloat16]),
                       r.choice(["bhnd", "bnhd"]), seed, spare)
    check_attn(args, causal, window)


def test_attn_pages_outside_the_pool_hide_their_keys():
    q, kc, vc, table, kv_len = attn_inputs([640, 100, 33], 4, 2, 2, 64, 16, torch.half, seed=6)
    bad = table.clone()
    bad[0, 3], bad[0, 20], bad[0, 39] = -1, kc.size(0), -2 ** 31
    bad[1, :7] = 2 ** 31 - 1
    bad[2, 2] = -5  # the newest token's page
    check_attn((q, kc, vc, bad, kv_len))


def test_attn_lengths_past_the_table_are_clamped():
    q, kc, vc, table, kv_len = attn_inputs([64, 64], 4, 2, 1, 64, 16, torch.half, spare=0)
    full = fa().paged_attn(q, kc, vc, table, kv_len)
    for n in (65, 2 ** 31 - 1):
        assert torch.equal(fa().paged_attn(q, kc, vc, table, torch.full_like(kv_len, n)), full)
    assert bool((fa().paged_attn(q, kc, vc, table, torch.full_like(kv_len, -1)) == 0).all())


def test_attn_equals_flash_attn_on_the_gathered_cache():
    """The same request through flash_attn's dense cache: both within their rounding."""
    N, n, page = 3, 900, 16
    q, kc, vc, table, kv_len = attn_inputs([n], 8, 2, N, 128, page, torch.bfloat16, seed=1)
    j = torch.arange(n, device=DEV)
    k, v = (c[table[0].long()[j // page], :, j % page].transpose(0, 1)[None] for c in (kc, vc))
    dense = fa().flash_attn(q, k, v, causal=True)
    ref = paged_ref.attention(q, kc, vc, table, kv_len)
    got = fa().paged_attn(q, kc, vc, table, kv_len)
    paged_ref.check(got, None, ref)
    assert bool(((got.double() - dense.double()).abs() <= 2 * ref[2] + 1e-6).all())


@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
def test_offsets_past_32_bits(layout):
    """A pool of 5.4 GB per cache: pages at both ends, written and read."""
    page, Hkv, D = 64, 8, 128
    P = 41000
    shape = (P, Hkv, page, D) if layout == "bhnd" else (P, page, Hkv, D)
    kc, vc = (torch.empty(shape, dtype=torch.half, device=DEV) for _ in range(2))
    if layout == "bnhd":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    pages = torch.tensor([[P - 1, 0, P - 2, 1, P // 2]], dtype=torch.int32)
    n = 5 * page - 7
    j = torch.arange(n)
    slots = (pages[0].long()[j // page] * page + j % page).to(torch.int32).to(DEV)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(n, Hkv, D, generator=g).half().to(DEV) for _ in range(2))
    fa().paged_append(k, v, kc, vc, slots)
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c[(slots // page).long(), :, (slots % page).long()], x)
    q = torch.randn(1, 16, 1, D, generator=g).half().to(DEV)
    check_attn((q, kc, vc, pages.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV)))


def test_attn_refusals():
    f = fa().paged_attn
    q, kc, vc, table, lens = attn_inputs([40, 50], 4, 2, 1, 64, 16, torch.half)
    for bad in ((q.float(), kc, vc, table, lens), (q.bfloat16(), kc, vc, table, lens),
                (q[0], kc, vc, table, lens), (q[:, :3], kc, vc, table, lens),
                (q[..., :32], kc, vc, table, lens), (q, kc, vc[:2], table, lens),
                (q, kc, vc, table[:1], lens), (q, kc, vc, table.long(), lens),
                (q, kc, vc, table.t(), lens), (q, kc, vc, table, lens[:1]),
                (q, kc, vc, table, lens.long()), (q, kc, vc, table, lens.cpu()),
                (q, kc, vc, table.cpu(), lens), (q, kc.cpu(), vc, table, lens),
                (q, kc[:, :, :5], vc[:, :, :5], table, lens), (q[:0], kc, vc, table[:0], lens[:0]),
                (q.clone().requires_grad_(), kc, vc, table, lens)):
        with pytest.raises(RuntimeError):
            f(*bad)
    with pytest.raises(RuntimeError, match="alibi_slopes"):
        f(q, kc, vc, table, lens, alibi_slopes=torch.ones(4))
    with torch.no_grad():
        assert torch.equal(f(q.clone().requires_grad_(), kc, vc, table, lens), f(q, kc, vc, table, lens))


def test_compiled_calls_run_as_they_are():
    q, kc, vc, table, lens = attn_inputs([40, 50], 4, 2, 1, 64, 16, torch.half)
    step = torch.compile(lambda x: fa().paged_attn(x * 1, kc, vc, table, lens) + 0, backend="eager")
    for seed in range(2):
        x = torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).half().to(DEV)
        assert torch.equal(step(x), fa().paged_attn(x, kc, vc, table, lens))


def test_on_a_side_stream_and_in_two_threads():
    """Calls on streams of their own, at the same time, with workspaces of their own."""
    import threading
    a = attn_inputs([5000, 1200], 8, 2, 1, 128, 16, torch.half, seed=1)
    b = attn_inputs([100, 7000, 3], 8, 8, 2, 64, 32, torch.bfloat16, seed=2)
    want = [fa().paged_attn(*x) for x in (a, b)]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i, args):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            outs = [fa().paged_attn(*args) for _ in range(20)]
        s.synchronize()
        got[i] = outs

    threads = [threading.Thread(target=work, args=(i, x)) for i, x in enumerate((a, b))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


def test_two_captured_graphs_replayed_at_once():
    """Each captured call has a workspace of its own: replays overlap on two streams."""
    calls = [attn_inputs([6000, 900], 8, 2, 1, 128, 16, torch.half, seed=3),
             attn_inputs([200, 3000, 77], 16, 2, 3, 64, 32, torch.bfloat16, seed=4)]
    want = [fa().paged_attn(*c) for c in calls]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(fa().paged_attn(*c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for o in outs:
            o.fill_(float("nan"))
        fa().paged_attn(*calls[0])  # eager work between the replays
        torch.cuda.synchronize()
        for _ in range(4):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_capi_step_with_a_poisoned_workspace():
    """The three entries through the C ABI: a NaN-filled workspace of the size asked
    for, slots that are not 16-byte aligned, nothing written around either."""
    from test_paged_cpu import Cache, capi
    from helpers import fa_opts
    import ctypes
    lib, page, P, B, M, Hq, Hkv, D = capi(), 16, 4000, 6, 700, 8, 2, 128
    g = torch.Generator().manual_seed(11)
    i32 = dict(dtype=torch.int32, device=DEV)
    table, free = torch.full((B, M), -1, **i32), torch.randperm(P, generator=g).to(**i32)
    old, ring = torch.zeros(B, **i32), torch.tensor([P - 5, P], **i32)
    new = torch.tensor([9000, 0, 1, 700, 33, 5001], **i32)
    T = int(new.sum())
    slots = torch.full((T + 9,), -77, **i32)
    kv_len, ring_out = torch.empty(B, **i32), torch.empty(2, **i32)
    at = lambda t: t.data_ptr()
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.fa_paged_tables(at(table), M, M, at(old), at(new), at(free), P, at(ring), page, B, 0,
                               T + 3, at(slots) + 4, at(kv_len), at(ring_out), stream) == 0
    assert torch.equal(kv_len, new) and slots[0] == -77 and slots[T + 4:].tolist() == [-77] * 5
    assert slots[T + 1:T + 4].tolist() == [-1] * 3
    want = paged_ref.tables(*(x.cpu() for x in (torch.full_like(table, -1), old, new, free, ring)),
                            page, tokens=T)
    assert torch.equal(table.cpu(), want[0]) and torch.equal(slots[1:T + 1].cpu(), want[2])
    k, v = (torch.randn(T, Hkv, D, generator=g).half().to(DEV) for _ in range(2))
    kc, vc = (torch.full((P, Hkv, page, D), float("nan"), dtype=torch.half, device=DEV) for _ in range(2))
    c = ctypes.pointer(Cache(at(kc), at(vc), kc.stride(0), kc.stride(1), kc.stride(2), P, page,
                             at(table), M, M, at(kv_len)))
    row = Hkv * D
    assert lib.fa_paged_append(at(k), at(v), row, 0, D, row, 0, D, at(slots) + 4, c, T, 1, Hkv, D,
                               stream) == 0
    q = torch.randn(B, Hq, 1, D, generator=g).half().to(DEV)
    o, lse = torch.full_like(q, float("nan")), torch.full((B, Hq, 1), float("nan"), device=DEV)
    size = lib.fa_paged_attn_workspace_bytes(B, Hq, Hkv, 1, D)
    ws = torch.full((size // 4 + 64,), float("nan"), device=DEV)
    assert lib.fa_paged_attn(at(q), at(o), at(lse), c, at(ws), size, B, Hq, Hkv, 1, D, 1, fa_opts(),
                             stream) == 0
    torch.cuda.synchronize()
    assert bool(torch.isnan(ws[size // 4:]).all())
    paged_ref.check(o, lse, paged_ref.attention(q, kc, vc, table, kv_len))
    assert torch.equal(fa().paged_attn(q, kc, vc, table, kv_len), o)


# ------------------------------------------------------- the three together

class Serving:
    """Requests over one pool, and beside it every request's tokens kept densely."""

    def __init__(self, B, Hq, Hkv, D, page, P, M, dtype, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.shape = (B, Hq, Hkv, D)
        self.page, self.dtype = page, dtype
        self.kc, self.vc = pool_of(P, Hkv, page, D, dtype, "bhnd", fill=float("nan"))
        self.table = torch.full((B, M), -1, dtype=torch.int32, device=DEV)
        self.free = torch.arange(P, dtype=torch.int32, device=DEV)
        self.ring = torch.tensor([0, P], dtype=torch.int32, device=DEV)
        self.lens = torch.zeros(B, dtype=torch.int32, device=DEV)
        self.tokens = [[] for _ in range(B)]  # (k, v) rows (Hkv, D)

    def rows(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype)

    def check(self, o, q, lens):
        """o of q against float64 attention over the tokens kept beside the cache."""
        B, Hq, Hkv, D = self.shape
        top = max(lens + [1])
        kc, vc = (torch.zeros(B, Hkv, top, D, dtype=self.dtype, device=DEV) for _ in range(2))
        for b, n in enumerate(lens):
            assert n == len(self.tokens[b])
            for i, c in enumerate((kc, vc)):
                if n:
                    c[b, :, :n] = torch.stack([t[i] for t in self.tokens[b]], 1).to(DEV)
        own = torch.arange(B, dtype=torch.int32, device=DEV)[:, None]  # a page per request
        paged_ref.check(o, None, paged_ref.attention(q, kc, vc, own, lens))


@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("pool", [260, 96])
def test_serving_loop(page, pool):
    """Prompts enter packed, decode one token a step, draft three and take some back,
    end, and others take their pages; every step's attention against the tokens."""
    f = fa()
    B, Hq, Hkv, D = 5, 8, 2, 64
    s = Serving(B, Hq, Hkv, D, page, pool // page, 320 // page, torch.half, seed=page)
    full = 0
    for step in range(30):
        lens = s.lens.tolist()
        kind = ("prompt", "decode", "draft", "decode", "end")[step % 5]
        new = list(lens)
        for b in range(B):
            if kind == "prompt" and lens[b] == 0:
                new[b] = int(torch.randint(1, 60, (), generator=s.g))
            elif kind == "decode" and lens[b]:
                new[b] += 1
            elif kind == "draft" and lens[b]:
                new[b] += 3
            elif kind == "end" and (b + step) % 3 == 0:
                new[b] = 0
        new_t = torch.tensor(new, dtype=torch.int32, device=DEV)
        grown = [max(n - o, 0) for n, o in zip(new, lens)]
        N = {"decode": 1, "draft": 3}.get(kind)
        if N:
            slots, kv_len, ring = f.paged_tables(s.table, s.lens, new_t, s.free, s.ring, page, max_new=N)
            k, v = s.rows(B, Hkv, N, D), s.rows(B, Hkv, N, D)
            f.paged_append(k.to(DEV), v.to(DEV), s.kc, s.vc, slots)
        else:
            total = sum(grown)
            slots, kv_len, ring = f.paged_tables(s.table, s.lens, new_t, s.free, s.ring, page,
                                                 tokens=total + 3)
            k, v = s.rows(total + 3, Hkv, D), s.rows(total + 3, Hkv, D)
            f.paged_append(k.to(DEV), v.to(DEV), s.kc, s.vc, slots)
        got, first = kv_len.tolist(), 0
        full += got != new
        for b in range(B):
            if got[b] <= lens[b]:
                s.tokens[b] = s.tokens[b][:got[b]]
            for i in range(got[b] - lens[b]):
                s.tokens[b].append((k[b, :, i], v[b, :, i]) if N else (k[first + i], v[first + i]))
            first += grown[b]
        q = s.rows(B, Hq, N or 1, D).to(DEV)
        s.check(f.paged_attn(q, s.kc, s.vc, s.table, kv_len), q, got)
        s.lens, s.ring = kv_len, ring
        if kind == "draft":  # two of the three are taken back
            back = torch.tensor([max(n - 2, 0) if g else n for n, g in zip(got, grown)],
                                dtype=torch.int32, device=DEV)
            _, s.lens, s.ring = f.paged_tables(s.table, s.lens, back, s.free, s.ring, page, max_new=0)
            s.tokens = [t[:n] for t, n in zip(s.tokens, s.lens.tolist())]
    assert full or pool > 200  # (the small pool does not hold all prompts)


def test_captured_decoding_steps():
    """One captured step (lengths, tables, append, attention) replayed with eager work
    in between: each replay's attention against the tokens so far."""
    f = fa()
    B, Hq, Hkv, D, page = 4, 8, 2, 128, 16
    s = Serving(B, Hq, Hkv, D, page, 60, 12, torch.bfloat16, seed=1)
    k, v = (torch.zeros(B, Hkv, 1, D, dtype=s.dtype, device=DEV) for _ in range(2))
    q = torch.zeros(B, Hq, 1, D, dtype=s.dtype, device=DEV)
    live = torch.tensor([1, 1, 0, 1], dtype=torch.int32, device=DEV)  # (an unused entry)

    def step():
        slots, kv_len, ring = f.paged_tables(s.table, s.lens, s.lens + live, s.free, s.ring, page,
                                             max_new=1)
        f.paged_append(k, v, s.kc, s.vc, slots)
        o = f.paged_attn(q, s.kc, s.vc, s.table, kv_len)
        s.lens.copy_(kv_len)
        s.ring.copy_(ring)
        return o

    state = [x.clone() for x in (s.lens, s.ring, s.table, s.free)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    for x, y in zip((s.lens, s.ring, s.table, s.free), state):
        x.copy_(y)
    other = attn_inputs([400, 30], 4, 2, 1, 64, 16, torch.half)
    for n in range(40):
        nk, nv, nq = s.rows(B, Hkv, 1, D), s.rows(B, Hkv, 1, D), s.rows(B, Hq, 1, D)
        for t, x in ((k, nk), (v, nv), (q, nq)):
            t.copy_(x)
        o.fill_(float("nan"))
        f.paged_attn(*other)  # eager work between the replays
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            if int(live[b]):
                s.tokens[b].append((nk[b, :, 0], nv[b, :, 0]))
        s.check(o, q, [(n + 1) * int(x) for x in live])
        assert s.lens.tolist() == [(n + 1) * int(x) for x in live]
