"""Paged attention of rows whose softmax spans many powers of two: one key with nearly
all of the weight and next to no value (an attention sink), and a long flat tail far
below it that makes the output. No counterpart in the reference."""
import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.half, torch.bfloat16])
@pytest.mark.parametrize("B,D,Hq,N", [(2048, 64, 2, 1),  # an item per wave
                                      (1500, 64, 2, 1),  # items that two waves share
                                      (600, 128, 4, 2), (400, 256, 1, 1), (3, 32, 1, 1)])
@pytest.mark.parametrize("peak", [4.125, 4.21875, 4.75])  # tails at 2^-24.5, 2^-25.7 and 2^-32.6
def test_a_sink_over_a_long_flat_tail(peak, B, D, Hq, N, dtype):
    """B requests over the same pages: 16384 keys of score 0 behind one of peak^2.

    The outputs are sums of the tail's weights alone, so these have to be right
    relative to themselves. paged_ref's bound takes every probability as rounded by
    half a step of itself. In fp16 that ends at the smallest normal number: the
    kernel's probabilities are scaled by 2^15, and one below 2^-14 / 2^15 is off by half
    a subnormal step, 2^-25 / 2^15 = 2^-40 of the row's largest, which is 1 and part of
    the sum that divides: n 2^-40 max |v| more."""
    n, page = 16384 + N, 64
    g = torch.Generator().manual_seed(D)
    P = -(-n // page)
    kc, vc = (torch.zeros(P, 1, page, D, dtype=dtype, device=DEV) for _ in range(2))
    vc.copy_(((0.5 + torch.rand(P, 1, page, D, generator=g)) * 100).to(dtype))
    kc[0, 0, 0, 0], vc[0, 0, 0] = peak, 0
    q = torch.zeros(1, Hq, N, D, dtype=dtype, device=DEV)
    q[..., 0] = peak
    table = torch.arange(P, dtype=torch.int32, device=DEV)[None]
    o, lse, o_tol, lse_tol = paged_ref.attention(q, kc, vc, table, [n], scale=1.0)
    if dtype == torch.half:
        o_tol = o_tol + n * 2.0 ** -40 * vc.double().abs().max()
    import fa_p100
    got, got_lse = fa_p100.paged_attn(q.expand(B, -1, -1, -1).contiguous(), kc, vc,
                                      table.repeat(B, 1),
                                      torch.full((B,), n, dtype=torch.int32, device=DEV),
                                      softmax_scale=1.0, return_lse=True)
    ref = [x.expand(B, *x.shape[1:]) for x in (o, lse, o_tol, lse_tol)]
    paged_ref.check(got, got_lse, ref)


@pytest.mark.parametrize("dtype", [torch.half, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,N,D", [
    ([1, 33, 1000, 5000], 8, 1, 1, 128), ([20000], 8, 2, 4, 64), ([700] * 40, 32, 1, 1, 256),
    ([9000, 3, 700], 16, 4, 8, 96), ([300 * i for i in range(30)], 4, 4, 1, 32), ([4000], 31, 1, 1, 80)])
def test_up_to_32_rows_of_a_kv_head_are_rounded_once(lens, Hq, Hkv, N, D, dtype):
    """paged_ref's bound without the probabilities' rounding u A (A = sum_j p_j |v_j|, its
    result of |v|): they are two numbers of q's format, whose sum is off by u^2 of it, in
    fp16 by 2^-40 of the row's largest where it is below 2^-29 of that (see above)."""
    from test_gpu_paged import attn_inputs, fa
    args = attn_inputs(lens, Hq, Hkv, N, D, 16, dtype, seed=D)
    o, lse, o_tol, lse_tol = paged_ref.attention(*args)
    a = paged_ref.attention(args[0], args[1], args[2].abs(), *args[3:])[0]
    u = torch.finfo(dtype).eps / 2
    o_tol = o_tol - (u - u * u) * a
    if dtype == torch.half:
        values = args[2].double()
        o_tol = o_tol + max(lens) * 2.0 ** -40 * values[torch.isfinite(values)].abs().max()
    got, got_lse = fa().paged_attn(*args, return_lse=True)
    paged_ref.check(got, got_lse, (o, lse, o_tol, lse_tol))
