"""Paged attention where the division of the keys takes its less common ways: lines of
key blocks past 2^17 units, joins by item over more requests than a wave has lanes.
And the tables' pages counted on what the kernel returns. No counterpart in the
reference."""
import pytest
import torch

import paged_ref
from test_gpu_paged import DEV, attn_inputs, check_attn, fa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.half, torch.bfloat16])
@pytest.mark.parametrize("D,Hq,N,B", [(32, 2, 1, 700), (64, 3, 2, 700), (256, 1, 1, 640), (128, 40, 1, 400)])
def test_lines_past_131072_units(D, Hq, N, B, dtype):
    """Requests of few lengths over the same pages, in no order: more units than the
    join's division in floats takes. Each against its length's float64 result."""
    lens, page = [16384, 9001, 5, 12345, 777], 32
    g = torch.Generator().manual_seed(B + D)
    q, kc, vc, table, _ = attn_inputs([16384], Hq, 1, N, D, page, dtype, seed=D)
    pick = torch.randint(0, 5, (B,), generator=g)
    kv_len = torch.tensor(lens)[pick]
    tiles = -(-Hq * N // 32)
    assert int(((kv_len + 31) // 32).sum()) * tiles >= 1 << 17
    ref = paged_ref.attention(q.expand(5, -1, -1, -1), kc, vc, table.expand(5, -1), lens)
    got, lse = fa().paged_attn(q.expand(B, -1, -1, -1).contiguous(), kc, vc, table.repeat(B, 1),
                               kv_len.to(torch.int32).to(DEV), return_lse=True)
    paged_ref.check(got, lse, [x[pick.to(DEV)] for x in ref])


@pytest.mark.parametrize("B,Hq,Hkv,N,D", [(70, 5, 1, 1, 128), (85, 5, 1, 1, 128), (66, 3, 1, 1, 256),
                                          (65, 2, 1, 1, 128), (68, 9, 1, 1, 64), (80, 7, 1, 3, 32)])
@pytest.mark.parametrize("top", [40, 700, 3000])
def test_joins_by_item_of_more_than_64_requests(B, Hq, Hkv, N, D, top):
    g = torch.Generator().manual_seed(B + top)
    lens = torch.randint(0, top + 1, (B,), generator=g).tolist()
    lens[0], lens[63], lens[64], lens[-1] = top, 0, top, top // 2
    check_attn(attn_inputs(lens, Hq, Hkv, N, D, 16, torch.half, seed=B))


@pytest.mark.parametrize("seed", range(6))
def test_tables_keep_every_page_once(seed):
    """Requests that enter, grow, shrink and end over a pool that some steps exhaust:
    after every call the requests' pages and the free ones are the pool, each once, and
    the slots are distinct rows of the requests' own pages."""
    r = torch.Generator().manual_seed(seed)
    page, B, M = (4, 8)[seed % 2], (7, 70, 300)[seed % 3], 20
    P = 8 * B
    i32 = dict(dtype=torch.int32, device=DEV)
    table, free = torch.full((B, M), -1, **i32), torch.randperm(P, generator=r).to(**i32)
    ring, old = torch.tensor([seed, P], **i32), torch.zeros(B, **i32)
    short = taken = back = 0
    for step in range(25):
        grow = torch.rand(B, generator=r) < 0.5
        new = torch.where(grow, old.cpu() + 3, torch.randint(0, M * page + 1, (B,), generator=r))
        new = new.to(**i32)
        packed = step % 2 == 0
        kw = dict(tokens=B * M * page) if packed else dict(max_new=M * page)
        slots, kv_len, ring = fa().paged_tables(table, old, new, free, ring, page, **kw)
        t, lens, before, got = table.cpu(), kv_len.tolist(), old.tolist(), slots.cpu()
        held = [t[b, :-(-n // page)].tolist() for b, n in enumerate(lens)]
        head, count = ring.tolist()
        rest = free.cpu()[(head + torch.arange(count)) % P].tolist()
        assert sorted(sum(held, []) + rest) == list(range(P)), step
        live = got[got >= 0].tolist()
        want = [held[b][j // page] * page + j % page for b, n in enumerate(lens) for j in range(before[b], n)]
        assert live == want, step
        short += int((kv_len < new.clamp(max=M * page)).sum())
        pages = [-(-n // page) for n in before]
        taken += sum(len(h) > n for h, n in zip(held, pages))
        back += sum(len(h) < n for h, n in zip(held, pages))
        old = kv_len
    assert short and taken > B and back > B
