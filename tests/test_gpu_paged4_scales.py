"""Paged caches in 4 bits whose scales lie at any byte: rows, heads and pages an odd number
of bytes apart, pools that begin anywhere in a word. Attention against float64 with its
bounds, the other operators bit for bit or with theirs (paged4_ref.py). No counterpart in the
reference, which has no cache."""
import pytest
import torch

import paged4_ref
import paged_ref
from test_gpu_paged4 import DEV, DTYPES, cache_of, fa, hide_rest, long_table, rows, run
from test_gpu_paged_evict import check_evict, check_weights, row_sums

pytestmark = pytest.mark.gpu

LENGTHS = [1, 65, 300, 0, 17]
# What is odd, and the byte of a word that K's and V's pools begin at.
KINDS = [("row", 0, 1), ("row", 3, 2), ("head", 1, 0), ("page", 2, 3), ("page", 1, 1), ("none", 1, 2),
         ("none", 3, 0), ("none", 2, 1)]


def scattered(scales, what, begin):
    """(the same scales in a buffer of their own, that buffer): `what` lies an odd number of
    bytes apart, the first at byte `begin` of a word; 0xee lies between."""
    P, Hkv, page, W = scales.shape
    row = W + 1 + W % 2 if what == "row" else W
    head = page * row
    head += 1 + head % 2 if what == "head" else 0
    pages = Hkv * head
    pages += 1 + pages % 2 if what == "page" else 0
    buf = torch.full((P * pages + 8,), 0xee, dtype=torch.uint8, device=DEV)
    assert buf.data_ptr() % 4 == 0
    out = buf[begin:].as_strided((P, Hkv, page, W), (pages, head, row, 1))
    out.copy_(scales)
    return out, buf


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,N", [(6, 2, 1), (20, 2, 2), (4, 1, 1)])
@pytest.mark.parametrize("page", [1, 8, 16])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention(D, page, Hq, Hkv, N, dtype):
    """On the line and, for short tables, an item to a workgroup; one and two row tiles."""
    caches, k, v, table = cache_of(len(LENGTHS), Hkv, D, page, LENGTHS, seed=D + page, spread=2.0)
    hide_rest(caches, table, LENGTHS, page)
    q = rows((len(LENGTHS), Hq, N, D), DTYPES[dtype], 9)
    want = paged4_ref.attention(q, k, v, table, LENGTHS)
    for what, in_k, in_v in KINDS:
        ks, vs = scattered(caches[2], what, in_k)[0], scattered(caches[3], what, in_v)[0]
        for t in (table, long_table(table, page)):
            o, lse = run(q, (caches[0], caches[1], ks, vs), t, LENGTHS)
            try:
                paged_ref.check(o, lse, want)
            except AssertionError as e:
                raise AssertionError(f"{what} {in_k} {in_v}: {e}") from e


@pytest.mark.parametrize("page", [1, 8, 16])
@pytest.mark.parametrize("D", [32, 96, 128, 224, 256])
def test_append_and_gather(D, page):
    Hkv, T, P = 3, 40, 48 // page + 3
    k, v = rows((T, Hkv, D), torch.bfloat16, 1, 2.0), rows((T, Hkv, D), torch.bfloat16, 2, 2.0)
    slots = torch.randperm(P * page, generator=torch.Generator().manual_seed(D))[:T].to(torch.int32).to(DEV)
    for what, in_k, in_v in KINDS:
        kc, vc = (torch.zeros(P, Hkv, page, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
        empty = torch.full((P, Hkv, page, D // 32), 0xee, dtype=torch.uint8, device=DEV)
        (ks, k_buf), (vs, v_buf) = scattered(empty, what, in_k), scattered(empty, what, in_v)
        fa().paged_append(k, v, kc, vc, slots, k_scale=ks, v_scale=vs)
        at = slots.long()
        for x, codes, scales, buf in ((k, kc, ks, k_buf), (v, vc, vs, v_buf)):
            want = paged4_ref.quantise(x)
            assert torch.equal(codes[at // page, :, at % page], want[0]), what
            assert torch.equal(scales[at // page, :, at % page], want[1]), what
            assert int((buf != 0xee).sum()) <= want[1].numel(), what  # (nothing between them)
        for got, x in zip(fa().paged_gather(kc, vc, slots, k_scale=ks, v_scale=vs), (k, v)):
            assert torch.equal(got, paged4_ref.values(*paged4_ref.quantise(x)).bfloat16()), what


@pytest.mark.parametrize("Hq,N", [(6, 1), (8, 2), (10, 5)])
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("D", [32, 96, 128, 224, 256])
def test_weights(D, page, Hq, N):
    caches, k, _, table = cache_of(len(LENGTHS), 2, D, page, LENGTHS, seed=D + page, spread=2.0)
    hide_rest(caches, table, LENGTHS, page)
    q = rows((len(LENGTHS), Hq, N, D), torch.float16, 9, 0.5)
    lse = row_sums(q, k, table, LENGTHS)
    for what, in_k, _ in KINDS:
        check_weights(q, (caches[0], scattered(caches[2], what, in_k)[0]), k, table, LENGTHS, lse=lse)


@pytest.mark.parametrize("tables", ["short", "long"])
@pytest.mark.parametrize("D,page", [(32, 1), (96, 8), (256, 16)])
def test_evict(D, page, tables):
    caches, _, _, table = cache_of(len(LENGTHS), 2, D, page, LENGTHS, seed=D)
    w = rows(caches[0].shape[:3], torch.float32, 3).abs()
    t = (table if tables == "short" else long_table(table, page)).cpu()
    for what, in_k, in_v in KINDS:
        (ks, k_buf), (vs, v_buf) = scattered(caches[2], what, in_k), scattered(caches[3], what, in_v)
        between = [b.clone() for b in (k_buf, v_buf)]
        check_evict([caches[0].clone(), caches[1].clone(), ks, vs], w.clone(), t, LENGTHS, 40, 5)
        for scales, buf, before, begin in ((ks, k_buf, between[0], in_k), (vs, v_buf, between[1], in_v)):
            for b in (buf, before):  # (but for the scales themselves)
                b[begin:].as_strided(scales.shape, scales.stride()).fill_(0)
            assert torch.equal(buf, before), what
