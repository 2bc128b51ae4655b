"""Paged caches in 4 bits: the launches that sizes choose. Attention with an item to a
workgroup at wide heads, whose tables have to be short for it; writes and reads of more
tokens than workgroups take at once, of tokens that several workgroups share. Against the
definitions (paged4_ref.py). No counterpart in the reference, which has no cache."""
import pytest
import torch

import paged4_ref
import paged_ref
from test_gpu_paged4 import DEV, DTYPES, cache_of, fa, hide_rest, pool, pools, rows, run

pytestmark = pytest.mark.gpu

# An item goes to a workgroup where the tables hold two blocks of 64 keys per wave, four waves
# above head dim 128, and the items are 256 at most.
LENGTHS, MOST = [1, 63, 64, 65, 0, 300, 129, 17], 512


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("Hq,Hkv,N", [(4, 4, 1), (16, 1, 1), (24, 1, 1), (6, 2, 9), (16, 1, 2), (8, 2, 9), (12, 1, 7)])
@pytest.mark.parametrize("D,page", [(160, 2), (192, 4), (192, 32), (224, 8), (224, 64), (256, 1), (256, 8), (256, 16)])
def test_items_of_a_workgroup_at_wide_heads(D, page, Hq, Hkv, N, dtype):
    """One, two and more row tiles of 16 (one or two to a wave), pages of every kind of place."""
    caches, k, v, table = cache_of(len(LENGTHS), Hkv, D, page, LENGTHS, seed=D + N, spread=2.0)
    assert table.size(1) * page <= MOST
    hide_rest(caches, table, LENGTHS, page)
    q = rows((len(LENGTHS), Hq, N, D), DTYPES[dtype], 9)
    o, lse = run(q, caches, table, LENGTHS)
    paged_ref.check(o, lse, paged4_ref.attention(q, k, v, table, LENGTHS))
    again, _ = run(q, caches, table, LENGTHS)
    assert torch.equal(o, again)


@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=5), dict(window=64, alibi=True, scale=0.3),
                                dict(causal=False, alibi=True, scale=0.02), dict(window=200)])
@pytest.mark.parametrize("Hq,N", [(8, 1), (10, 3)])
@pytest.mark.parametrize("D,page", [(192, 16), (256, 8), (256, 2)])
def test_options_of_a_workgroups_items(D, page, Hq, N, kw):
    caches, k, v, table = cache_of(len(LENGTHS), 1, D, page, LENGTHS, seed=D)
    assert table.size(1) * page <= MOST
    hide_rest(caches, table, LENGTHS, page)
    q = rows((len(LENGTHS), Hq, N, D), torch.bfloat16, 9)
    if kw.get("alibi"):
        kw = dict(kw, alibi=torch.linspace(-0.1, 0.5, Hq, device=DEV))
    names = dict(causal="causal", window="sliding_window", alibi="alibi_slopes", scale="softmax_scale")
    o, lse = run(q, caches, table, LENGTHS, **{names[x]: y for x, y in kw.items()})
    paged_ref.check(o, lse, paged4_ref.attention(q, k, v, table, LENGTHS, **kw))


# (heads, head dim): chunks of 16 bytes of a token's dense rows 384, 4 and 36 of the 256 that a
# workgroup takes, so two workgroups to a token, 64 and 7 tokens to a workgroup; a thread goes on
# by 1024, 131072 and 14336 tokens, over the ends of several requests of N.
@pytest.mark.parametrize("Hkv,D,B,N", [(12, 256, 7, 701), (1, 32, 5, 30011), (3, 96, 9, 5003), (3, 96, 30011, 1),
                                       (12, 256, 2, 9), (9, 256, 1, 1)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_many_tokens_of_requests_apart(Hkv, D, B, N, dtype):
    """(B, Hkv, N, D) views of (B, N, Hkv + 1, D + 8), each with strides of its own."""
    page = 16
    P = B * N // page + 9
    wide = rows((B, N, Hkv + 1, D + 8), DTYPES[dtype], 4)
    k, v = (wide[:, :, h:h + Hkv, o:o + D].transpose(1, 2) for h, o in ((0, 8), (1, 0)))
    slots = torch.randperm(P * page, generator=torch.Generator().manual_seed(1))[:B * N].view(B, N).to(torch.int32)
    slots.view(-1)[::97] = -1
    slots = slots.to(DEV)
    kc, vc, ks, vs = pools(P, Hkv, page, D)
    want = [t.clone() for t in (kc, vc, ks, vs)]
    live = slots.view(-1) >= 0
    at = slots.view(-1)[live].long()
    dense = []
    for x, codes, scales in ((k, want[0], want[2]), (v, want[1], want[3])):
        x = x.transpose(1, 2).reshape(B * N, Hkv, D)[live]
        codes[at // page, :, at % page], scales[at // page, :, at % page] = paged4_ref.quantise(x)
        dense.append(x)
    fa().paged_append(k, v, kc, vc, slots, k_scale=ks, v_scale=vs)
    for name, a, b in zip(("k", "v", "k_scale", "v_scale"), (kc, vc, ks, vs), want):
        assert torch.equal(a, b), name

    def check(got, want_rows):
        flat = got.transpose(1, 2).reshape(B * N, Hkv, D)
        assert torch.equal(flat[live], want_rows) and not bool(flat[~live].any())

    for got, x in zip(fa().paged_gather(kc, vc, slots, k_scale=ks, v_scale=vs, dtype=DTYPES[dtype]), dense):
        check(got, paged4_ref.values(*paged4_ref.quantise(x)).to(x.dtype))
    kc, vc = (pool(P, Hkv, page, D, "bnhd", 0, DTYPES[dtype]) for _ in range(2))
    fa().paged_append(k, v, kc, vc, slots)
    for got, x in zip(fa().paged_gather(kc, vc, slots), dense):
        check(got, x)
