"""Paged caches in 4 bits on the GPU: codes and scales bit for bit, rows read back exactly,
attention against float64 with the bounds of its rounding (paged4_ref.py). No counterpart
in the reference, which has no cache."""
import math

import pytest
import torch

import paged4_ref
import paged_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def fa():
    import fa_p100
    return fa_p100


def pool(P, Hkv, page, width, layout="bhnd", fill=0x3a, dtype=torch.uint8):
    """A pool (P, Hkv, page, width) of bytes `fill`, its storage in the order of `layout`."""
    if layout == "bnhd":
        return torch.full((P, page, Hkv, width), fill, dtype=dtype, device=DEV).transpose(1, 2)
    if layout == "inner":  # a part of wider rows' pages
        return torch.full((P, 2, Hkv, page, width), fill, dtype=dtype, device=DEV)[:, 1]
    return torch.full((P, Hkv, page, width), fill, dtype=dtype, device=DEV)


def pools(P, Hkv, page, D, layout="bhnd"):
    """k_cache, v_cache, k_scale, v_scale of a 4-bit cache."""
    return (*(pool(P, Hkv, page, D // 2, layout) for _ in range(2)),
            *(pool(P, Hkv, page, D // 32, layout) for _ in range(2)))


def rows(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape, generator=g))
    return x.to(dtype).to(DEV)


# ------------------------------------------------------------------ append, gather

@pytest.mark.parametrize("layout", ["bhnd", "bnhd", "inner"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,page,Hkv,T", [(32, 1, 1, 1), (64, 16, 2, 5), (96, 8, 3, 33), (128, 16, 8, 200),
                                          (160, 4, 1, 17), (224, 32, 5, 64), (256, 64, 4, 300)])
def test_append_writes_the_definition(D, page, Hkv, T, dtype, layout):
    P = T // page + 3
    g = torch.Generator().manual_seed(T)
    slots = torch.randperm(P * page, generator=g)[:T].to(torch.int32)
    slots[::7] = torch.tensor([-1, P * page, 2 ** 31 - 1, -2 ** 31])[torch.arange(len(slots[::7])) % 4]
    k, v = rows((T, Hkv, D), DTYPES[dtype], 1), rows((T, Hkv, D), DTYPES[dtype], 2, 3.0)
    kc, vc, ks, vs = pools(P, Hkv, page, D, layout)
    want = [t.clone() for t in (kc, vc, ks, vs)]
    live = (slots >= 0) & (slots < P * page)
    at = slots[live].long().to(DEV)
    for x, codes, scales in ((k, want[0], want[2]), (v, want[1], want[3])):
        codes[at // page, :, at % page], scales[at // page, :, at % page] = paged4_ref.quantise(x[live.to(DEV)])
    versions = [t._version for t in (kc, vc, ks, vs)]
    fa().paged_append(k, v, kc, vc, slots.to(DEV), k_scale=ks, v_scale=vs)
    for name, a, b in zip(("k", "v", "k_scale", "v_scale"), (kc, vc, ks, vs), want):
        assert torch.equal(a, b), name
    assert all(t._version > n for t, n in zip((kc, vc, ks, vs), versions))
    for out in (torch.bfloat16, torch.float16):
        back = fa().paged_gather(kc, vc, slots.to(DEV), k_scale=ks, v_scale=vs, dtype=out)
        for got, codes, scales in zip(back, want[:2], want[2:]):
            exact = torch.zeros(T, Hkv, D, dtype=torch.float64, device=DEV)
            exact[live.to(DEV)] = paged4_ref.values(codes[at // page, :, at % page], scales[at // page, :, at % page])
            assert got.dtype == out and got.is_contiguous()
            assert torch.equal(got.isnan(), exact.isnan())
            assert torch.equal(got.nan_to_num(nan=0.0), exact.to(out).nan_to_num(nan=0.0))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_every_value_beside_every_scale(dtype):
    """All 65536 bit patterns, each in a block whose largest value fixes the scale (ties of
    every size among them), and each alone in its block; infinities and NaN too."""
    dt = DTYPES[dtype]
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt)
    tops = torch.tensor([0.0, 1.0, 1.75, 1.7578125, 6.0, 7.0, 2.0 ** -14, 2.0 ** -20, 1000.0, 57344.0, 65504.0]).to(dt)
    x = torch.zeros(65536, len(tops) + 1, 32, dtype=dt)
    x[:, :-1, 5] = tops
    x[:, :, 11] = every[:, None]
    T = x.numel() // 256
    x = x.view(T, 1, 256).to(DEV)
    page = 128
    kc, vc, ks, vs = pools(T // page, 1, page, 256)
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    fa().paged_append(x, x, kc, vc, slots, k_scale=ks, v_scale=vs)
    codes, scales = paged4_ref.quantise(x.view(T // page, 1, page, 256))
    assert torch.equal(ks, scales) and torch.equal(vs, scales)
    assert torch.equal(kc, codes) and torch.equal(vc, codes)
    back = fa().paged_gather(kc, vc, slots, k_scale=ks, v_scale=vs, dtype=dt)[0]
    finite = (scales != 255).repeat_interleave(32, -1).view(T, 1, 256)
    assert bool(torch.isfinite(back[finite]).all()) and bool(torch.isnan(back[~finite]).all())


def test_every_code_of_every_scale_reads_back():
    """256 scale bytes by 16 codes, 0 (2^-127) and 255 (NaN) among them."""
    scales = torch.arange(256, dtype=torch.uint8, device=DEV).view(16, 1, 16, 1)
    codes = (torch.arange(16, dtype=torch.uint8, device=DEV) * 17).expand(16, 1, 16, 16).contiguous()
    slots = torch.arange(256, dtype=torch.int32, device=DEV)
    exact = paged4_ref.values(codes, scales).view(256, 1, 32)
    for dt in (torch.bfloat16, torch.float16):
        k, v = fa().paged_gather(codes, codes, slots, k_scale=scales, v_scale=scales, dtype=dt)
        for got in (k, v):
            assert torch.equal(got[:255], exact[:255].to(dt)) and bool(torch.isnan(got[255]).all())


def test_append_takes_the_shapes_that_projections_leave():
    """(B, Hkv, N, D) views of (B, N, Hkv, D), rows apart and offset ones, slots (B, N)."""
    B, Hkv, N, D, page, P = 3, 4, 7, 64, 8, 9
    wide = rows((B, N, Hkv + 1, D + 8), torch.bfloat16, 4)
    k, v = (wide[:, :, :Hkv, o:o + D].transpose(1, 2) for o in (0, 8))
    odd = rows((B, Hkv, N, D + 1), torch.bfloat16, 5)[..., 1:]  # (rows on no 16-byte boundary)
    slots = torch.randperm(P * page, generator=torch.Generator().manual_seed(1))[:B * N].view(B, N).to(torch.int32).to(DEV)
    for a, b in ((k, v), (odd, k), (odd.half(), v.half())):
        kc, vc, ks, vs = pools(P, Hkv, page, D)
        fa().paged_append(a, b, kc, vc, slots, k_scale=ks, v_scale=vs)
        x, y = fa().paged_gather(kc, vc, slots, k_scale=ks, v_scale=vs, dtype=a.dtype)
        assert x.shape == (B, Hkv, N, D)
        for got, src in ((x, a), (y, b)):
            assert torch.equal(got, paged4_ref.values(*paged4_ref.quantise(src)).to(a.dtype))


@pytest.mark.parametrize("layout", ["bhnd", "bnhd", "inner"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [8, 40, 80, 128, 256])
def test_gather_copies_rows_of_16_bits(D, dtype, layout):
    P, Hkv, page = 7, 3, 16
    kc, vc = (pool(P, Hkv, page, D, layout, 0, DTYPES[dtype]) for _ in range(2))
    kc.copy_(rows(kc.shape, kc.dtype, 1))
    vc.copy_(rows(vc.shape, vc.dtype, 2))
    kc[2, 1, 3, 0], vc[2, 0, 3, -1] = float("nan"), float("inf")
    slots = torch.tensor([[0, 35, P * page - 1, -1], [35, P * page, 17, 17]], dtype=torch.int32, device=DEV)
    for s in (slots, slots.flatten(), slots.t(), slots[:, ::2], slots[:0], slots[:, :0]):
        got = fa().paged_gather(kc, vc, s)
        live = ((s >= 0) & (s < P * page))
        at = torch.where(live, s, 0).long()
        for x, cache in zip(got, (kc, vc)):
            want = cache[at // page, :, at % page]  # (..., Hkv, D)
            want = torch.where(live[..., None, None], want, torch.zeros_like(want))
            want = want if s.dim() == 1 else want.transpose(1, 2)
            assert x.shape == want.shape and torch.equal(x.view(torch.int16), want.contiguous().view(torch.int16))


def test_rows_past_32_bits():
    """A pool of more than 2^32 bytes: rows near its end, written and read."""
    Hkv, page, D = 8, 256, 256
    P = (1 << 32) // (Hkv * page * D // 2) + 9
    kc = torch.empty(P, Hkv, page, D // 2, dtype=torch.uint8, device=DEV)
    vc = torch.empty_like(kc)
    ks, vs = (torch.empty(P, Hkv, page, D // 32, dtype=torch.uint8, device=DEV) for _ in range(2))
    slots = torch.tensor([0, P * page - 1, (P - 3) * page + 5, 77], dtype=torch.int32, device=DEV)
    k, v = rows((4, Hkv, D), torch.bfloat16, 1), rows((4, Hkv, D), torch.bfloat16, 2)
    fa().paged_append(k, v, kc, vc, slots, k_scale=ks, v_scale=vs)
    for got, x in zip(fa().paged_gather(kc, vc, slots, k_scale=ks, v_scale=vs), (k, v)):
        assert torch.equal(got, paged4_ref.values(*paged4_ref.quantise(x)).bfloat16())
    table = torch.tensor([[P - 1, P - 3]], dtype=torch.int32, device=DEV)
    n = page + 6
    at = torch.arange(n, device=DEV)
    slots = table[0, at // page] * page + (at % page).to(torch.int32)
    k, v = rows((n, Hkv, D), torch.bfloat16, 3), rows((n, Hkv, D), torch.bfloat16, 4)
    fa().paged_append(k, v, kc, vc, slots, k_scale=ks, v_scale=vs)
    q, lens = rows((1, 16, 1, D), torch.bfloat16, 5), torch.tensor([n], dtype=torch.int32, device=DEV)
    o = fa().paged_attn(q, kc, vc, table, lens, k_scale=ks, v_scale=vs)
    small = [t[[P - 1, P - 3]] for t in (kc, vc, ks, vs)]
    ref = paged4_ref.attention(q, paged4_ref.values(small[0], small[2]), paged4_ref.values(small[1], small[3]),
                               torch.tensor([[0, 1]]), [n])
    paged_ref.check(o, None, ref)


# ------------------------------------------------------------------ attention

def cache_of(B, Hkv, D, page, lens, seed, layout="bhnd", spread=1.0, spare=3):
    """(caches and scales, float64 k and v, table): random rows in 4 bits, pages anywhere."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    perm = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((B, max(need + [1]) + 2), 2 ** 30, dtype=torch.int32)  # (entries behind: not read)
    used = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[used:used + n]
        used += n
    kc, vc, ks, vs = pools(P, Hkv, page, D, layout)
    for cache, scale, x in ((kc, ks, 1), (vc, vs, 2)):
        codes, sizes = paged4_ref.quantise(rows((P, Hkv, page, D), torch.bfloat16, seed + x, spread))
        cache.copy_(codes)
        scale.copy_(sizes)
    k, v = paged4_ref.values(kc, ks), paged4_ref.values(vc, vs)
    return (kc, vc, ks, vs), k, v, table.to(DEV)


def hide_rest(caches, table, lens, page):
    """Fills all rows that hold no token with NaN."""
    kc, vc, ks, vs = caches
    live = torch.zeros(kc.size(0), page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            p = int(table[b, j // page])
            if 0 <= p < kc.size(0):
                live[p, j % page] = True
    dead = ~live.to(DEV)[:, None, :, None]
    for cache, scale in ((kc, ks), (vc, vs)):
        scale.copy_(torch.where(dead, torch.full_like(scale, 255), scale))
        cache.copy_(torch.where(dead, torch.full_like(cache, 0x77), cache))


def run(q, caches, table, lens, **kw):
    kc, vc, ks, vs = caches
    return fa().paged_attn(q, kc, vc, table, torch.tensor(lens, dtype=torch.int32, device=DEV),
                           return_lse=True, k_scale=ks, v_scale=vs, **kw)


def long_table(table, page):
    """One for requests so long that several workgroups would share an item."""
    return torch.nn.functional.pad(table, (0, 20000 // page), value=2 ** 30)


LENGTHS = [1, 63, 64, 65, 0, 700, 129, 17]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,N", [(4, 4, 1), (8, 1, 1), (6, 2, 5), (16, 1, 1), (16, 1, 2), (24, 1, 1),
                                      (8, 2, 9), (64, 1, 1), (12, 1, 7), (32, 1, 5)])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention_matches_float64(D, Hq, Hkv, N, dtype):
    """Each row tiling (1, 2, several groups of 2 tiles of 16) at each width, items of a workgroup
    and on the line."""
    page = {32: 1, 64: 16, 96: 8, 128: 32, 160: 2, 192: 4, 224: 64, 256: 16}[D]
    caches, k, v, table = cache_of(len(LENGTHS), Hkv, D, page, LENGTHS, seed=D + N)
    hide_rest(caches, table, LENGTHS, page)
    q = rows((len(LENGTHS), Hq, N, D), DTYPES[dtype], 9)
    want = paged4_ref.attention(q, k, v, table, LENGTHS)
    for t in (table, long_table(table, page)):
        paged_ref.check(*run(q, caches, t, LENGTHS), want)


@pytest.mark.parametrize("layout", ["bhnd", "bnhd", "inner"])
@pytest.mark.parametrize("causal,window,alibi,scale", [(False, None, False, None), (True, 5, False, None),
                                                       (True, 64, True, 0.3), (True, 300, False, None),
                                                       (False, None, True, 0.02), (True, 1, True, None)])
@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16"), (192, "fp16")])
def test_options(D, dtype, causal, window, alibi, scale, layout):
    lens = [3, 64, 0, 257, 1000, 66]
    caches, k, v, table = cache_of(6, 2, D, 16, lens, seed=D, layout=layout)
    hide_rest(caches, table, lens, 16)
    q = rows((6, 3, 10, D), DTYPES[dtype], 9).transpose(1, 2)  # (B, 10 heads, 3 rows)
    slopes = torch.linspace(-0.1, 0.5, 10, device=DEV) if alibi else None
    want = paged4_ref.attention(q, k, v, table, lens, causal=causal, window=window, alibi=slopes,
                                scale=scale)
    for t in (table, long_table(table, 16)):
        o, lse = run(q, caches, t, lens, causal=causal, sliding_window=window, alibi_slopes=slopes,
                     softmax_scale=scale)
        assert o.shape == q.shape and o.stride() == q.stride()
        paged_ref.check(o, lse, want)


@pytest.mark.parametrize("B,Hq,Hkv,N,D,top,page", [(1, 8, 1, 1, 128, 20000, 16), (1, 16, 2, 2, 256, 8000, 8),
                                                   (70, 8, 2, 1, 64, 3000, 32), (200, 4, 1, 1, 128, 400, 16),
                                                   (3, 32, 4, 6, 96, 9000, 128), (1, 4, 4, 1, 32, 60000, 256)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_long_and_many_requests(B, Hq, Hkv, N, D, top, page, dtype):
    """Items that many waves share, waves that hold many items, joins of both kinds."""
    lens = [max(N, int(top * ((0.5 + 0.618034 * i) % 1.0))) for i in range(B)]
    lens[0] = top
    caches, k, v, table = cache_of(B, Hkv, D, page, lens, seed=B)
    q = rows((B, Hq, N, D), DTYPES[dtype], 9)
    o, lse = run(q, caches, table, lens)
    paged_ref.check(o, lse, paged4_ref.attention(q, k, v, table, lens))
    again, lse_again = run(q, caches, table, lens)
    assert torch.equal(o, again) and torch.equal(lse, lse_again)


def test_sizes_far_apart():
    """Scales from 2^-126 to 2^125 beside each other, in K and in V; large scores."""
    lens = [300, 65]
    caches, _, _, table = cache_of(2, 2, 64, 16, lens, seed=5)
    kc, vc, ks, vs = caches
    g = torch.Generator().manual_seed(8)
    # (V: within 2^+-60 a row, so that sums of weights times values stay finite; K's blocks
    # one small, one ordinary)
    vs.copy_(torch.randint(127 - 100, 127 + 60, vs.shape, generator=g).to(torch.uint8))
    ks[..., 0] = 1
    ks[..., 1] = torch.randint(124, 130, ks.shape[:-1], generator=g).to(torch.uint8).to(DEV)
    k, v = paged4_ref.values(kc, ks), paged4_ref.values(vc, vs)
    q = rows((2, 4, 1, 64), torch.bfloat16, 9, 0.5)
    o, lse = run(q, caches, table, lens)
    paged_ref.check(o, lse, paged4_ref.attention(q, k, v, table, lens))


def test_pages_outside_the_pool_are_hidden():
    lens = [200, 64, 33]
    for page in (1, 8, 64):
        caches, k, v, table = cache_of(3, 2, 128, page, lens, seed=page)
        P = caches[0].size(0)
        bad = table.clone()
        bad[0, 0], bad[0, 130 // page], bad[2, :-(-33 // page)] = -1, P, 2 ** 31 - 1
        caches[2][0], caches[3][0] = 255, 255  # (page 0, which hidden keys are read from)
        k, v = paged4_ref.values(caches[0], caches[2]), paged4_ref.values(caches[1], caches[3])
        bad[bad == 0] = -2 ** 31  # (and hidden, whoever has it)
        q = rows((3, 8, 3, 128), torch.bfloat16, 9)
        o, lse = run(q, caches, bad, lens)
        paged_ref.check(o, lse, paged4_ref.attention(q, k, v, bad, lens))
        assert bool((o[2] == 0).all()) and bool((lse[2] == math.inf).all())


def test_a_nan_stays_in_its_request():
    lens = [100, 100, 100]
    caches, k, v, table = cache_of(3, 2, 64, 16, lens, seed=3)
    kc, vc, ks, vs = caches
    ks[int(table[0, 2]), 0, 5], vs[int(table[1, 3]), 1, 7] = 255, 255
    q = rows((3, 8, 1, 64), torch.float16, 9)
    o, lse = run(q, caches, table, lens)
    assert bool(torch.isnan(o[0, :4]).all()) and bool(torch.isnan(lse[0, :4]).all())
    nan_v = torch.isnan(paged4_ref.values(vc, vs)[int(table[1, 3]), 1, 7])
    assert bool(torch.isnan(o[1, 4:][..., nan_v]).all()) and bool(torch.isfinite(lse[1]).all())
    ref = paged4_ref.attention(q, k, v, table, lens)
    for b, heads in ((0, slice(4, 8)), (1, slice(0, 4)), (2, slice(0, 8))):
        paged_ref.check(o[b, heads], lse[b, heads], [t[b, heads] for t in ref])
    # infinite queries: NaN or infinite scores, and no more than theirs
    q[2, 0, 0, 0] = math.inf
    o, lse = run(q, caches, table, lens)
    assert not bool(torch.isfinite(o[2, 0]).all())
    paged_ref.check(o[2, 4:], lse[2, 4:], [t[2, 4:] for t in ref])


def test_captured_steps_replay():
    """Append, attention and tables' lengths in a graph, replayed over changing inputs, with
    eager work between; two captured calls share nothing."""
    Hkv, D, page, B = 2, 128, 16, 4
    lens = [30, 1, 65, 200]
    caches, _, _, table = cache_of(B, Hkv, D, page, lens, seed=11, spare=40)
    P = caches[0].size(0)
    held = set(table[table < 2 ** 30].tolist())
    free = iter(p for p in range(P) if p not in held)
    for b, n in enumerate(lens):
        have = -(-n // page)
        if have < table.size(1):
            table[b, have:] = torch.tensor([next(free) for _ in range(table.size(1) - have)], dtype=torch.int32)
    kv = torch.tensor(lens, dtype=torch.int32, device=DEV)
    k, v, q = (rows((B, h, 1, D), torch.bfloat16, i) for i, h in enumerate((Hkv, Hkv, 8)))
    b_idx = torch.arange(B, device=DEV)

    def step():
        slots = (table[b_idx, ((kv - 1) // page).long()] * page + (kv - 1) % page)[:, None]
        fa().paged_append(k, v, caches[0], caches[1], slots, k_scale=caches[2], v_scale=caches[3])
        one = run2(q)
        return one, run2(q * 2)

    def run2(x):
        return fa().paged_attn(x, caches[0], caches[1], table, kv, k_scale=caches[2], v_scale=caches[3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        for t, s in ((k, 20), (v, 30), (q, 40)):
            t.copy_(rows(t.shape, t.dtype, s + i))
        kv.add_(1)
        graph.replay()
        got = [t.clone() for t in out]
        want = step()  # (appends the same rows again)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_streams_and_order():
    """On another stream than the tensors' own; the result does not depend on it."""
    lens = [500, 3]
    caches, k, v, table = cache_of(2, 2, 64, 16, lens, seed=2)
    q = rows((2, 4, 1, 64), torch.float16, 9)
    want, _ = run(q, caches, table, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = run(q, caches, table, lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_refusals():
    lens = torch.tensor([20, 5], dtype=torch.int32, device=DEV)
    (kc, vc, ks, vs), _, _, table = cache_of(2, 2, 64, 16, [20, 5], seed=2)
    q, k = rows((2, 4, 1, 64), torch.float16, 9), rows((2, 2, 64), torch.float16, 8)
    slots = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    f = fa()
    bad_scales = (ks[:1], ks[..., :1], ks.int(), ks.cpu(), ks.transpose(1, 2), ks[0])
    for s in bad_scales:
        for call in (lambda: f.paged_attn(q, kc, vc, table, lens, k_scale=s, v_scale=s),
                     lambda: f.paged_append(k, k, kc, vc, slots, k_scale=s, v_scale=s),
                     lambda: f.paged_gather(kc, vc, slots, k_scale=s, v_scale=s)):
            with pytest.raises(RuntimeError):
                call()
    four = dict(k_scale=ks, v_scale=vs)
    for call in (lambda: f.paged_attn(q[..., :32].contiguous(), kc, vc, table, lens, **four),
                 lambda: f.paged_attn(q, kc, vc, table, lens),
                 lambda: f.paged_attn(q, kc.half(), vc.half(), table, lens, **four),
                 lambda: f.paged_attn(q, kc[..., ::2], vc[..., ::2], table, lens, **four),
                 lambda: f.paged_attn(q.float(), kc, vc, table, lens, **four),
                 lambda: f.paged_append(k.float(), k.float(), kc, vc, slots, **four),
                 lambda: f.paged_append(k[..., :32], k[..., :32], kc, vc, slots, **four),
                 lambda: f.paged_append(k, k, kc, vc, slots.long(), **four),
                 lambda: f.paged_append(k, k, kc[:1].expand(3, -1, -1, -1), vc[:1].expand(3, -1, -1, -1), slots,
                                        k_scale=ks[:3], v_scale=vs[:3]),
                 lambda: f.paged_append(k, k, kc, kc, slots, **four),
                 lambda: f.paged_append(k, k, kc, vc, slots, k_scale=ks, v_scale=ks),
                 lambda: f.paged_gather(kc, vc, slots, dtype=torch.float32, **four),
                 lambda: f.paged_gather(kc, vc, slots),
                 lambda: f.paged_gather(kc.half(), vc.half(), slots, dtype=torch.bfloat16),
                 lambda: f.paged_gather(kc, vc, slots.long(), **four)):
        with pytest.raises(RuntimeError):
            call()
    grad = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        f.paged_attn(grad, kc, vc, table, lens, **four)
    with torch.no_grad():
        f.paged_attn(grad, kc, vc, table, lens, **four)
