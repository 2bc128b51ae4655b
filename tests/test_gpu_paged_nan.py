"""What infinities and NaN do in paged attention: lse = +inf says that a row sees no
key and nothing else, a poisoned row is NaN, and other kv heads and requests do not
notice. No counterpart in the reference."""
import math

import pytest
import torch

import paged_ref
from test_gpu_paged import DEV, attn_inputs, fa

pytestmark = pytest.mark.gpu

CALLS = [([40, 700, 5, 0], 4, 2, 3, 64), ([9000, 33], 8, 2, 2, 128), ([20000], 2, 2, 1, 64),
         ([3000, 90], 4, 2, 2, 256), ([300] * 70, 4, 2, 2, 32), ([5000, 1, 40], 66, 2, 1, 96)]


def run(args):
    return fa().paged_attn(*args, return_lse=True)


def same(args, clean, got, rows):
    """The rows of `clean` again. Bit for bit in other kv heads and requests than the
    poisoned ones (request 0, kv head 0); beside a poisoned row a running maximum may
    move earlier, so those are within their rounding of the float64 results."""
    o, lse, o_tol, lse_tol = paged_ref.attention(*args)
    G = o.size(1) // args[1].size(1)
    far = rows.clone()
    far[0, :G] = False
    assert torch.equal(got[0][far], clean[0][far]) and torch.equal(got[1][far], clean[1][far])
    near = rows & torch.isfinite(lse)
    assert bool(((got[0].double() - o).abs() <= o_tol + 2.0 ** -24)[near].all())  # (a subnormal's step)
    assert bool(((got[1].double() - lse).abs() <= lse_tol)[near].all())


def spot(args, b, j):
    """(page, row) of request b's token j."""
    page = args[1].size(2)
    return int(args[3][b, j // page]), j % page


@pytest.mark.parametrize("dtype", [torch.half, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,N,D", CALLS)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_poisoned_query_row(lens, Hq, Hkv, N, D, dtype, bad):
    args = attn_inputs(lens, Hq, Hkv, N, D, 16, dtype, seed=D)
    clean, q = run(args), args[0].clone()
    q[0, 0, N - 1, 3] = bad
    got = run((q, *args[1:]))
    assert bool(torch.isnan(got[0][0, 0, N - 1]).all()) and bool(torch.isnan(got[1][0, 0, N - 1]))
    rest = torch.ones(clean[1].shape, dtype=torch.bool, device=DEV)
    rest[0, 0, N - 1] = False
    same(args, clean, got, rest)


@pytest.mark.parametrize("dtype", [torch.half, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,N,D", CALLS)
@pytest.mark.parametrize("where", ["first", "newest"])
def test_a_poisoned_key(lens, Hq, Hkv, N, D, dtype, where):
    """A NaN key of kv head 0: every row of its heads sees the first token, the last
    row alone the newest."""
    args = attn_inputs(lens, Hq, Hkv, N, D, 16, dtype, seed=D)
    clean, kc = run(args), args[1].clone()
    G, n = Hq // Hkv, lens[0]
    page, row = spot(args, 0, 0 if where == "first" else n - 1)
    kc[page, 0, row, 5] = math.nan
    got = run((args[0], kc, *args[2:]))
    seen = torch.zeros(clean[1].shape, dtype=torch.bool, device=DEV)
    seen[0, :G, (0 if where == "first" else N - 1):] = True
    assert bool(torch.isnan(got[0][seen]).all()) and bool(torch.isnan(got[1][seen]).all())
    same(args, clean, got, ~seen)


@pytest.mark.parametrize("dtype", [torch.half, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,N,D", CALLS)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_poisoned_value(lens, Hq, Hkv, N, D, dtype, bad):
    """In column 5 of the newest token's value: the row that sees it has it there (an
    infinity as one or as NaN), and no sum of weights knows of it."""
    args = attn_inputs(lens, Hq, Hkv, N, D, 16, dtype, seed=D)
    o, lse = run(args)
    G, n = Hq // Hkv, lens[0]
    page, row = spot(args, 0, n - 1)
    args[2][page, 0, row, 5] = bad
    got, got_lse = run(args)
    assert torch.equal(got_lse, lse)
    assert not bool(torch.isfinite(got[0, :G, N - 1, 5]).any())
    columns = torch.arange(D, device=DEV) != 5
    assert torch.equal(got[..., columns], o[..., columns])
    others = torch.ones(lse.shape, dtype=torch.bool, device=DEV)
    others[0, :G] = False
    assert torch.equal(got[others], o[others])


@pytest.mark.parametrize("lens,Hq,Hkv,N,D", CALLS)
def test_an_infinite_key(lens, Hq, Hkv, N, D):
    """One element of a key infinite: where its score is -inf the row is as without that
    key, where it is +inf the row is NaN, and in no row that sees a key is lse +inf."""
    args = attn_inputs(lens, Hq, Hkv, N, D, 16, torch.half, seed=D)
    _, lse = run(args)
    G = Hq // Hkv
    page, row = spot(args, 0, 1)
    args[1][page, 0, row, 5] = math.inf
    _, got_lse = run(args)
    up = args[0][0, :G, :, 5] > 0
    assert bool(torch.isnan(got_lse[0, :G][up]).all()) and bool(torch.isfinite(got_lse[0, :G][~up]).all())
    assert torch.equal(got_lse[0, G:], lse[0, G:]) and torch.equal(got_lse[1:], lse[1:])
