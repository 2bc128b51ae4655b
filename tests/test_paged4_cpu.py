"""The smaller paged caches' argument checks that need no GPU (nothing is launched), and
their plain restatements against second ones. No counterpart in the reference."""
import ctypes
import subprocess
import sys

import pytest
import torch

import paged4_ref
from helpers import LIB, fa_opts
from test_paged_cpu import cache, capi


class Scales(ctypes.Structure):
    """struct fa_paged_scales of include/fa_mi355x.h."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("stride_page", ctypes.c_longlong),
                ("stride_head", ctypes.c_longlong), ("stride_row", ctypes.c_longlong)]


def scales(**kw):
    return ctypes.pointer(Scales(**{**dict(k=1 << 20, v=1 << 21, stride_page=64, stride_head=32,
                                           stride_row=2), **kw}))


def cache4(**kw):
    """Rows of 32 bytes: 64 values."""
    return cache(**{**dict(k=1 << 24, v=1 << 25, stride_page=1024, stride_head=512, stride_row=32), **kw})


def capi4():
    lib = capi()
    vp, i, ll, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_size_t
    lib.fa_paged4_append.argtypes = [vp, vp] + [ll] * 6 + [vp, vp, vp, i, i, i, i, i, vp]
    lib.fa_paged_gather.argtypes = [vp, vp, ll, ll, ll, vp, vp, vp, i, i, i, i, i, vp]
    lib.fa_paged4_attn.argtypes = [vp] * 6 + [sz] + [i] * 6 + [vp, vp]
    lib.fa_paged4_attn_workspace_bytes.argtypes = [i] * 5
    lib.fa_paged4_attn_workspace_bytes.restype = sz
    lib.fa_paged_weights.argtypes = [vp] * 5 + [ll] * 3 + [i] * 7 + [vp, vp]
    lib.fa_paged_evict.argtypes = [vp] * 3 + [ll] * 3 + [vp, i, vp, vp, sz, i, i, i, vp]
    lib.fa_paged_evict_workspace_bytes.argtypes = [i] * 4
    lib.fa_paged_evict_workspace_bytes.restype = sz
    return lib


def test_append_refusals():
    lib = capi4()

    def call(k=16, v=16, strides=(1024, 64, 64) * 2, slots=16, c=None, s=None, B=1, N=1, Hkv=2, D=64,
             dtype=1):
        return lib.fa_paged4_append(k, v, *strides, slots, c or cache4(), s or scales(), B, N, Hkv, D,
                                    dtype, None)

    for D in (60, 72, 80, 288):
        assert call(D=D) == 10001, D
    assert call(dtype=2) == 10009 and call(dtype=-1) == 10009
    assert call(Hkv=0) == 10003 and call(N=0) == 10002 and call(B=0) == 10004
    for bad in (dict(k=None), dict(v=None), dict(slots=None), dict(c=cache4(k=None)),
                dict(c=cache4(v=None)), dict(s=scales(k=None)), dict(s=scales(v=None))):
        assert call(**bad) == 10005, bad
    for bad in (dict(k=24), dict(v=8), dict(strides=(1024, 60, 64) * 2), dict(c=cache4(page_size=12)),
                dict(c=cache4(stride_row=40)), dict(c=cache4(k=8)), dict(c=cache4(pages=1 << 28)),
                dict(s=scales(stride_row=-2))):
        assert call(**bad) == 10019, bad
    # rows or scales that share a place: of a pool, and of k's and v's
    for bad in (dict(c=cache4(stride_row=16)), dict(c=cache4(stride_head=0)),
                dict(c=cache4(v=(1 << 24) + 32)), dict(s=scales(stride_row=1)),
                dict(s=scales(stride_page=0)), dict(s=scales(v=(1 << 20) + 2))):
        assert call(**bad) == 10019, bad
    for bad in (dict(B=1 << 16, N=1 << 16), dict(c=cache4(stride_page=1 << 31)),
                dict(s=scales(stride_page=1 << 31))):
        assert call(**bad) == 10007, bad


def test_gather_refusals():
    lib = capi4()

    def call(k=16, v=16, strides=(1024, 64, 64), slots=16, c=None, s=None, four=True, B=1, N=1, Hkv=2,
             D=64, dtype=1):
        return lib.fa_paged_gather(k, v, *strides, slots, c or (cache4() if four else cache()),
                                   (s or scales()) if four else None, B, N, Hkv, D, dtype, None)

    for four in (True, False):
        assert call(D=60, four=four) == 10001 and call(dtype=3, four=four) == 10009
        assert call(Hkv=-1, four=four) == 10003 and call(N=0, four=four) == 10002
        assert call(B=0, four=four) == 10004 and call(B=1 << 16, N=1 << 16, four=four) == 10007
        for bad in (dict(k=None), dict(v=None), dict(slots=None)):
            assert call(four=four, **bad) == 10005, bad
        for bad in (dict(k=8), dict(v=24), dict(strides=(1024, 60, 64))):
            assert call(four=four, **bad) == 10019, bad
    assert call(D=72) == 10001 and call(s=scales(k=None)) == 10005


def test_attn_refusals():
    lib = capi4()

    def call(q=16, o=16, lse=None, c=None, s=None, ws=16, nbytes=1 << 40, B=1, Hq=4, Hkv=2, N=1, D=64,
             causal=1, opts=None):
        return lib.fa_paged4_attn(q, o, lse, c or cache4(), s or scales(), ws, nbytes, B, Hq, Hkv, N,
                                  D, causal, opts, None)

    assert lib.fa_paged4_attn(16, 16, None, cache4(), None, 16, 1 << 40, 1, 4, 2, 1, 64, 1, None,
                              None) == 10005
    assert call(D=60) == 10001 and call(D=72) == 10001
    assert call(N=0) == 10002 and call(Hkv=3) == 10003 and call(B=0) == 10004
    for bad in (dict(q=None), dict(o=None), dict(c=cache4(table=None)), dict(c=cache4(kv_len=None)),
                dict(c=cache4(v=None)), dict(s=scales(v=None)), dict(ws=None)):
        assert call(**bad) == 10005, bad
    for bad in (dict(page_size=48), dict(stride_head=100), dict(table_width=0), dict(table_stride=2)):
        assert call(c=cache4(**bad)) == 10019, bad
    assert call(N=1 << 23) == 10007
    assert call(B=1 << 16, c=cache4(table_width=1 << 20, table_stride=1 << 20)) == 10007
    assert call(opts=fa_opts(kv_rows=9)) == 10019 and call(opts=fa_opts(window=-1)) == 10010
    need = lib.fa_paged4_attn_workspace_bytes(1, 4, 2, 1, 64)
    assert need > 0 and call(nbytes=need - 1) == 10006
    for bad in (dict(q=24), dict(o=8), dict(ws=20)):
        assert call(**bad) == 10019, bad
    assert lib.fa_paged4_attn_workspace_bytes(1, 4, 2, 1, 72) == 0
    # what the header says that it is at most
    most = max(lib.fa_paged4_attn_workspace_bytes(1, 64, 1, n, D) for n in (1, 2) for D in (32, 64, 96, 128, 160, 256))
    assert most <= 68.5e6


@pytest.mark.parametrize("entry,units", [("fa_paged_attn", "17paged_workspace_w"), ("fa_paged4_attn", "18paged4_workspace_w")])
@pytest.mark.parametrize("bf", [0, 1])
def test_workspace_is_the_larger_format_s(entry, units, bf, tmp_path):
    """Each format's kernels lay the workspace out for themselves, and the size that a caller
    asks for holds either: where one format's needs more, that (here what a stub in the place of
    that format's answer says, loaded ahead of the library in a process of its own)."""
    stub, need = tmp_path / "stub.so", 1 << 40
    code = f'extern "C" unsigned long _ZN2fa{units}ILi128ELb{bf}EEEmi(int) {{ return {need}ul; }}'
    subprocess.run(["g++", "-shared", "-fPIC", "-x", "c++", "-", "-o", stub], input=code.encode(), check=True)
    ask = (f"import ctypes; ctypes.CDLL({str(stub)!r}, ctypes.RTLD_GLOBAL); "
           f"f = ctypes.CDLL({LIB!r}).{entry}_workspace_bytes; f.restype = ctypes.c_size_t; "
           "print(f(1, 4, 2, 1, 128))")
    assert int(subprocess.run([sys.executable, "-c", ask], check=True, capture_output=True).stdout) == need


def test_weights_refusals():
    lib = capi4()

    def call(q=16, lse=16, c=None, s=None, four=True, w=16, strides=(32, 16, 1), B=1, Hq=4, Hkv=2, N=1,
             D=64, opts=None):
        return lib.fa_paged_weights(q, lse, c or (cache4() if four else cache()),
                                    (s or scales()) if four else None, w, *strides, 0, B, Hq, Hkv, N,
                                    D, 1, opts, None)

    for bad in (dict(q=None), dict(lse=None), dict(w=None), dict(c=cache4(k=None)),
                dict(s=scales(k=None)), dict(c=cache4(table=None))):
        assert call(**bad) == 10005, bad
    for bad in (dict(q=24), dict(strides=(32, 16, 0)), dict(strides=(16, 16, 1)),
                dict(strides=(-32, 16, 1)), dict(opts=fa_opts(bias=1))):
        assert call(**bad) == 10019, bad
    assert call(D=80) == 10001 and call(Hkv=3) == 10003 and call(B=0) == 10004 and call(N=0) == 10002
    assert call(four=False, D=60) == 10001 and call(four=False, strides=(32, 16, 0)) == 10019
    assert call(strides=(1 << 31, 16, 1)) == 10007 and call(strides=(1, 1 << 20, 1 << 31)) == 10007


def test_evict_refusals():
    lib = capi4()

    def call(c=None, s=None, four=True, w=16, strides=(32, 16, 1), max_len=16, recent=0, new=16, ws=16,
             nbytes=1 << 40, B=1, Hkv=2, D=64):
        return lib.fa_paged_evict(c or (cache4() if four else cache(v=1 << 25)),
                                  (s or scales()) if four else None, w, *strides, max_len, recent, new,
                                  ws, nbytes, B, Hkv, D, None)

    for bad in (dict(w=None), dict(max_len=None), dict(new=None), dict(ws=None), dict(c=cache4(v=None)),
                dict(s=scales(v=None)), dict(c=cache4(kv_len=None)), dict(c=cache4(table=None))):
        assert call(**bad) == 10005, bad
    for bad in (dict(strides=(32, 16, 0)), dict(recent=-1), dict(ws=18), dict(c=cache4(table_width=0)),
                dict(c=cache4(stride_row=16)), dict(s=scales(stride_row=1)),
                dict(c=cache4(v=(1 << 24) + 32)), dict(c=cache4(kv_len=1 << 26), new=1 << 26),
                dict(c=cache4(kv_len=1 << 26), new=(1 << 26) + 4, B=2)):
        assert call(**bad) == 10019, bad
    assert call(four=False, c=cache(v=1 << 25, stride_row=32)) == 10019
    assert call(D=72) == 10001 and call(Hkv=0) == 10003 and call(B=0) == 10004
    assert call(B=1 << 20, Hkv=4) == 10007
    need = lib.fa_paged_evict_workspace_bytes(1, 2, 3, 16)
    assert need == 2 * (3 * 16 + 2) * 4 and call(nbytes=need - 1) == 10006
    for bad in ((0, 2, 3, 16), (1, 0, 3, 16), (1, 2, 0, 16), (1, 2, 3, 24), (1 << 21, 2, 3, 16)):
        assert lib.fa_paged_evict_workspace_bytes(*bad) == 0, bad


def test_evict_refuses_new_lengths_across_the_budgets():
    """Budgets are read by all kv heads while new lengths are written: these may lie in their
    place, which changes nothing that is read, but not shifted against them."""
    lib = capi4()
    B = 4

    def call(max_len, new, kv_len=1 << 27):
        return lib.fa_paged_evict(cache4(kv_len=kv_len), scales(), 16, 32, 16, 1, max_len, 0, new, 16,
                                  1 << 40, B, 2, 64, None)

    at = 1 << 26
    for off in range(4, 4 * B, 4):
        assert call(at, at + off) == 10019 and call(at, at - off) == 10019, off
    for off in (0, 4 * B - 4, -4):  # in the lengths' place, or across it
        assert call(1 << 28, at + off, kv_len=at) == 10019, off


def test_binding_refuses_host_tensors_and_bad_arguments():
    import fa_p100
    ints, lens = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.half)
    pool = torch.zeros(5, 2, 16, 32, dtype=torch.uint8)
    sc = torch.zeros(5, 2, 16, 2, dtype=torch.uint8)
    w, lse = torch.zeros(5, 2, 16), torch.zeros(2, 4, 1)
    four = dict(k_scale=sc, v_scale=sc)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        fa_p100.paged_attn(q, pool, pool, ints, lens, **four)
    with pytest.raises(RuntimeError, match="k must be a CUDA tensor"):
        fa_p100.paged_append(q[:, :2], q[:, :2], pool, pool, lens[:, None], **four)
    with pytest.raises(RuntimeError, match="k_cache and v_cache must be on"):
        fa_p100.paged_gather(pool, pool, lens, **four)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        fa_p100.paged_weights(q, pool, ints, lens, lse, w, k_scale=sc)
    with pytest.raises(RuntimeError, match="k_cache and v_cache must be on"):
        fa_p100.paged_evict(pool, pool, w, ints, lens, 4, **four)
    for call in (lambda **kw: fa_p100.paged_attn(q, pool, pool, ints, lens, **kw),
                 lambda **kw: fa_p100.paged_append(q[:, :2], q[:, :2], pool, pool, lens[:, None], **kw),
                 lambda **kw: fa_p100.paged_gather(pool, pool, lens, **kw),
                 lambda **kw: fa_p100.paged_evict(pool, pool, w, ints, lens, 4, **kw)):
        with pytest.raises(RuntimeError, match="given together"):
            call(k_scale=sc)
    with pytest.raises(ValueError, match="sliding_window"):
        fa_p100.paged_weights(q, pool, ints, lens, lse, w, causal=False, sliding_window=4)
    with pytest.raises(ValueError, match="softmax_scale"):
        fa_p100.paged_weights(q, pool, ints, lens, lse, w, softmax_scale=0.0)
    with pytest.raises(ValueError, match="alibi_slopes"):
        fa_p100.paged_weights(q, pool, ints, lens, lse, w, alibi_slopes=torch.ones(3))

    class Wrapped(torch.Tensor):
        pass

    for call in (lambda x: fa_p100.paged_gather(pool, pool, x),
                 lambda x: fa_p100.paged_evict(pool, pool, w, ints, x, 4),
                 lambda x: fa_p100.paged_weights(q, pool, ints, x, lse, w)):
        with pytest.raises(TypeError, match="plain tensors"):
            call(lens.as_subclass(Wrapped))
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, lens)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.func.vmap(lambda x: fa_p100.paged_attn(x, pool, pool, ints, lens, **four))(q[None])


def test_codes_are_the_nearest_levels():
    """paged4_ref.quantise against the distances to all codes of all scales."""
    g = torch.Generator().manual_seed(1)
    levels = torch.tensor(paged4_ref.LEVELS, dtype=torch.float64)
    for dtype in (torch.float16, torch.bfloat16):
        x = (torch.randn(300, 64, generator=g) * torch.exp(3 * torch.randn(300, 64, generator=g))).to(dtype)
        codes, scale = paged4_ref.quantise(x)
        got = paged4_ref.values(codes, scale)
        blocks, back = x.double().unflatten(-1, (-1, 32)), got.unflatten(-1, (-1, 32))
        step = torch.exp2(scale.double() - 127)
        # the scale: the least that reaches the largest value with 7 of it, but where that
        # is past the largest scale (a NaN where the rows overflowed to infinity)
        top = blocks.abs().amax(-1)
        bad, most = scale == 255, scale == 127 + paged4_ref.TOP[dtype]
        assert bool(((top <= 7 * step) | most | bad).all())
        assert bool(((top > 3.5 * step) | bad).all())
        assert torch.equal(bad, torch.isinf(top))
        blocks, back, step = (t[~bad] for t in (blocks, back, step))
        off = (blocks.abs()[..., None] - levels * step[..., None, None]).abs()
        best = off.amin(-1)
        assert bool(((blocks - back).abs() == best).all())
        # ties go to the even code
        tied = (off == best[..., None]).sum(-1) > 1
        half = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32))[~bad]
        assert bool((half[tied] % 2 == 0).all())
    # blocks at the formats' ends: finite in them, zeros of either sign kept, NaN alone
    for dtype in (torch.float16, torch.bfloat16):
        x = torch.zeros(6, 32, dtype=dtype)
        x[0], x[1, 3], x[2] = torch.finfo(dtype).max, torch.finfo(dtype).tiny, -0.0
        x[3, 0], x[4, 9], x[5, 1] = float("inf"), float("nan"), -1.0
        back = paged4_ref.values(*paged4_ref.quantise(x))
        assert bool(torch.isfinite(back[:3].to(dtype)).all()) and bool(torch.isnan(back[3:5]).all())
        assert bool(torch.signbit(back[2]).all()) and float(back[5, 1]) == -1.0
        assert float(back[0, 0]) == (49152.0 if dtype == torch.float16 else 6 * 2.0 ** 125)


def test_plain_eviction_keeps_the_heaviest():
    w = torch.tensor([3.0, 0.0, 5.0, 5.0, -0.0, 1.0, 5.0, 2.0]).view(2, 1, 4)
    rows = torch.arange(8.0).view(2, 1, 4).clone()
    table = torch.tensor([[1, 0]], dtype=torch.int32)  # tokens 0..3: page 1
    for keep, recent, want in ((3, 0, [2, 6, 7]), (4, 1, [2, 5, 6, 7]), (2, 2, [6, 7]), (1, 5, [7]),
                               (0, 3, []), (9, 0, list(range(8)))):
        a, b = rows.clone(), w.clone()
        token = torch.cat([a[1, 0], a[0, 0]])  # what row each token has
        weight = torch.cat([b[1, 0], b[0, 0]])
        new = paged4_ref.evict([a], b, table, [8], [keep], recent)
        assert int(new) == min(keep, 8)
        heavy = sorted(range(8 - min(recent, keep)), key=lambda i: (-float(weight[i]), i))
        kept = sorted(heavy[:keep - min(recent, keep)]) + list(range(8 - min(recent, keep), 8))
        kept = kept if keep < 8 else list(range(8))
        assert torch.cat([a[1, 0], a[0, 0]])[:len(kept)].tolist() == token[kept].tolist(), (keep, recent)
        assert torch.cat([b[1, 0], b[0, 0]])[:len(kept)].tolist() == weight[kept].tolist()
