"""The paged cache's argument checks that need no GPU (nothing is launched), and its
plain restatement against a second one. No counterpart in the reference."""
import ctypes

import pytest
import torch

import paged_ref
from helpers import fa_opts, load_capi
from oracle import attention as ora


class Cache(ctypes.Structure):
    """struct fa_paged_cache of include/fa_mi355x.h."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("stride_page", ctypes.c_longlong),
                ("stride_head", ctypes.c_longlong), ("stride_row", ctypes.c_longlong),
                ("pages", ctypes.c_int), ("page_size", ctypes.c_int), ("table", ctypes.c_void_p),
                ("table_stride", ctypes.c_longlong), ("table_width", ctypes.c_int),
                ("kv_len", ctypes.c_void_p)]


def cache(**kw):
    c = dict(k=16, v=16, stride_page=2048, stride_head=1024, stride_row=64, pages=4, page_size=16,
             table=16, table_stride=3, table_width=3, kv_len=16)
    return ctypes.pointer(Cache(**{**c, **kw}))


def capi():
    lib = load_capi()
    vp, i, ll, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t
    lib.fa_paged_tables.argtypes = [vp, ll, i, vp, vp, vp, i, vp, i, i, i, i, vp, vp, vp, vp]
    lib.fa_paged_append.argtypes = [vp, vp] + [ll] * 6 + [vp, vp, i, i, i, i, vp]
    lib.fa_paged_attn.argtypes = [vp, vp, vp, vp, vp, sz, i, i, i, i, i, i, vp, vp]
    lib.fa_paged_attn_workspace_bytes.argtypes = [i] * 5
    lib.fa_paged_attn_workspace_bytes.restype = sz
    return lib


def test_tables_refusals():
    lib = capi()
    one = 16

    def call(table=one, stride=4, width=4, old=one, new=one, free=one, n_ring=8, ring=one, page=16,
             B=2, max_new=1, tokens=-1, slots=one, kv_len=one, ring_out=one):
        return lib.fa_paged_tables(table, stride, width, old, new, free, n_ring, ring, page, B,
                                   max_new, tokens, slots, kv_len, ring_out, None)

    for name in ("table", "old", "new", "free", "ring", "slots", "kv_len", "ring_out"):
        assert call(**{name: None}) == 10005, name
    for bad in (dict(page=0), dict(page=-16), dict(page=24), dict(width=0), dict(stride=3),
                dict(n_ring=0), dict(max_new=-1)):
        assert call(**bad) == 10019, bad
    for bad in (dict(width=1 << 28, stride=1 << 28, page=8), dict(B=(1 << 20) + 1),
                dict(n_ring=1 << 30), dict(B=1 << 12, max_new=1 << 19)):
        assert call(**bad) == 10007, bad
    assert call(B=0) == 10004
    assert b"power of two" in lib.fa_error_string(10019)


def test_append_refusals():
    lib = capi()

    def call(k=16, v=16, strides=(1024, 64, 64) * 2, slots=16, c=None, B=1, N=1, Hkv=2, D=64):
        return lib.fa_paged_append(k, v, *strides, slots, c or cache(), B, N, Hkv, D, None)

    assert call(D=60) == 10001 and call(D=264) == 10001
    assert call(Hkv=0) == 10003 and call(N=0) == 10002 and call(B=0) == 10004
    for bad in (dict(k=None), dict(v=None), dict(slots=None), dict(c=cache(k=None))):
        assert call(**bad) == 10005, bad
    assert call(k=24) == 10019 and call(v=17) == 10019 and call(strides=(1024, 60, 64) * 2) == 10019
    for bad in (dict(page_size=12), dict(page_size=0), dict(pages=0), dict(v=24),
                dict(stride_row=60), dict(stride_page=-2048), dict(pages=1 << 28)):
        assert call(c=cache(**bad)) == 10019, bad
    assert call(B=1 << 16, N=1 << 16) == 10007


def test_attn_refusals():
    lib = capi()

    def call(q=16, o=16, lse=None, c=None, ws=16, nbytes=1 << 40, B=1, Hq=4, Hkv=2, N=1, D=64,
             causal=1, opts=None):
        return lib.fa_paged_attn(q, o, lse, c or cache(), ws, nbytes, B, Hq, Hkv, N, D, causal,
                                 opts, None)

    assert call(D=60) == 10001 and call(N=0) == 10002 and call(Hkv=3) == 10003 and call(B=0) == 10004
    for bad in (dict(q=None), dict(o=None), dict(c=cache(table=None)), dict(c=cache(kv_len=None)),
                dict(c=cache(v=None))):
        assert call(**bad) == 10005, bad
    for bad in (dict(page_size=48), dict(stride_head=100), dict(table_width=0), dict(table_stride=2),
                dict(table_width=1 << 28, table_stride=1 << 28)):
        assert call(c=cache(**bad)) == 10019, bad
    assert call(N=1 << 23) == 10007  # rows of a request
    assert call(B=1 << 16, c=cache(table_width=1 << 20, table_stride=1 << 20)) == 10007  # key blocks
    # (2^54 tiles of 2^10 blocks: their product in 64 bits is 0)
    assert call(B=1 << 30, Hq=1 << 24, Hkv=1 << 24, D=8,
                c=cache(table_width=1020, table_stride=1020, page_size=32)) == 10007
    assert call(Hq=1 << 23, Hkv=1, N=2, D=256, opts=fa_opts(layout=1)) == 10007  # a token's elements
    for bad in (fa_opts(kv_len=1), fa_opts(seg_start=1, seg_end=1), fa_opts(mask=1, mask_heads=1),
                fa_opts(drop=1, drop_scale=1.0), fa_opts(bias=1), fa_opts(kv_rows=9),
                fa_opts(block_rows=1), fa_opts(mask_t=1), fa_opts(drop_t=1)):
        assert call(opts=bad) == 10019
    assert call(causal=0, opts=fa_opts(window=4)) == 10010
    assert call(opts=fa_opts(window=-1)) == 10010
    assert call(opts=fa_opts(scale=float("nan"))) == 10012
    assert call(opts=fa_opts(dtype=2)) == 10009 and call(opts=fa_opts(layout=2)) == 10008
    need = lib.fa_paged_attn_workspace_bytes(1, 4, 2, 1, 64)
    assert need > 0 and call(nbytes=need - 1) == 10006 and call(ws=None) == 10005
    for bad in (dict(q=24), dict(o=8), dict(ws=20)):  # alignment
        assert call(**bad) == 10019, bad
    assert call(c=cache(stride_page=1 << 31)) == 10007
    assert lib.fa_paged_attn_workspace_bytes(1, 4, 3, 1, 64) == 0


def test_binding_refuses_host_tensors_and_bad_arguments():
    import fa_p100
    ints = torch.zeros(2, 3, dtype=torch.int32)
    lens = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.half)
    pool = torch.zeros(5, 2, 16, 64, dtype=torch.half)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        fa_p100.paged_attn(q, pool, pool, ints, lens)
    with pytest.raises(RuntimeError, match="k must be a CUDA tensor"):
        fa_p100.paged_append(pool[0], pool[0], pool, pool, lens)
    with pytest.raises(RuntimeError, match="block_table must be a CUDA tensor"):
        fa_p100.paged_tables(ints, lens, lens, lens, lens, 16, max_new=1)
    with pytest.raises(ValueError, match="sliding_window"):
        fa_p100.paged_attn(q, pool, pool, ints, lens, causal=False, sliding_window=4)
    with pytest.raises(ValueError, match="softmax_scale"):
        fa_p100.paged_attn(q, pool, pool, ints, lens, softmax_scale=-1.0)
    with pytest.raises(ValueError, match="alibi_slopes"):
        fa_p100.paged_attn(q, pool, pool, ints, lens, alibi_slopes=torch.ones(3))

    class Wrapped(torch.Tensor):
        pass

    with pytest.raises(TypeError, match="plain tensors"):
        fa_p100.paged_attn(q.as_subclass(Wrapped), pool, pool, ints, lens)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda x: fa_p100.paged_attn(x, pool, pool, ints, lens), q)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.func.vmap(lambda x: fa_p100.paged_attn(x, pool, pool, ints, lens))(q[None])
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(), pytest.raises(RuntimeError, match="cannot be traced"):
        fa_p100.paged_attn(q, pool, pool, ints, lens)


@pytest.mark.parametrize("causal,window,alibi", [(True, None, False), (False, None, False),
                                                 (True, 7, True)])
def test_plain_attention_equals_the_oracle(causal, window, alibi):
    """paged_ref.attention (rows gathered by table) against the dense oracle."""
    g = torch.Generator().manual_seed(3)
    B, Hq, Hkv, N, D, page, P = 3, 4, 2, 3, 16, 4, 40
    kc, vc = (torch.randn(P, Hkv, page, D, generator=g) for _ in range(2))
    q = torch.randn(B, Hq, N, D, generator=g)
    lens = [1, 12, 30]
    table = torch.randperm(P, generator=g)[:B * 9].view(B, 9).to(torch.int32)
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.0]) if alibi else None
    o, lse, _, _ = paged_ref.attention(q, kc, vc, table, lens, causal, window, slopes)
    for b, n in enumerate(lens):
        rows = [(int(table[b, j // page]), j % page) for j in range(n)]
        k, v = (torch.stack([c[p, :, r] for p, r in rows], 1)[None].double().numpy() for c in (kc, vc))
        want, want_lse = ora.attention_fwd(q[b:b + 1].double().numpy(), k, v, causal, window=window,
                                           alibi=None if slopes is None else slopes.double().numpy())
        assert ora.max_abs(o[b:b + 1].numpy(), want) < 1e-9
        some = want_lse < 1e300
        assert ora.max_abs(lse[b:b + 1].numpy()[some], want_lse[some]) < 1e-9
        assert (lse[b:b + 1].numpy() < 1e300).tolist() == some.tolist()


def test_plain_tables_keep_every_page_once():
    """Random growing, shrinking and ending requests over a small pool: the pages of
    the requests and the ring's free ones are the pool, each once, and slots are
    distinct."""
    g = torch.Generator().manual_seed(5)
    page, P, B, M = 4, 50, 7, 20
    table = torch.full((B, M), -1, dtype=torch.int32)
    free, ring = torch.arange(P, dtype=torch.int32), torch.tensor([0, P], dtype=torch.int32)
    old = torch.zeros(B, dtype=torch.int32)
    short = 0
    for step in range(200):
        new = torch.where(torch.rand(B, generator=g) < 0.5, old + 1,
                          torch.randint(0, 90, (B,), generator=g)).to(torch.int32)
        table, free, slots, kv_len, ring = paged_ref.tables(table, old, new, free, ring, page,
                                                            tokens=400)
        short += int((kv_len < new).any())
        held = [int(table[b, p]) for b in range(B) for p in range(-(-int(kv_len[b]) // page))]
        rest = [int(free[(int(ring[0]) + i) % P]) for i in range(int(ring[1]))]
        assert sorted(held + rest) == list(range(P)), step
        live = slots[slots >= 0].tolist()
        assert len(set(live)) == len(live)
        old = kv_len
    assert short > 10
