"""Paged attention's slopes in every form that they may have, and a step in inference
mode. No counterpart in the reference."""
import pytest
import torch

from test_gpu_paged import DEV, attn_inputs, check_attn, fa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["fp64", "fp16", "strided", "one", "no_grad"])
def test_slopes(form):
    args = attn_inputs([40, 1, 700], 8, 2, 2, 64, 16, torch.half, seed=1)
    slopes = torch.tensor([2.0 ** -h for h in range(8)], device=DEV)
    given = {"fp64": slopes.double(), "fp16": slopes.half(), "strided": slopes.repeat_interleave(3)[::3],
             "one": slopes[1:2].expand(8), "no_grad": slopes.clone().requires_grad_()}[form]
    with torch.no_grad():
        o, lse = check_attn(args, alibi=given)
    if form == "no_grad":
        with pytest.raises(RuntimeError, match="alibi_slopes requires grad"):
            fa().paged_attn(*args, alibi_slopes=given)
    want, want_lse = check_attn(args, alibi=slopes[1:2].repeat(8) if form == "one" else slopes)
    assert torch.equal(o, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dtype", [torch.half, torch.bfloat16])
def test_converted_slopes_in_a_captured_call(dtype):
    args = attn_inputs([900, 33], 8, 2, 1, 128, 16, dtype, seed=2)
    slopes = torch.tensor([2.0 ** -h for h in range(8)], device=DEV, dtype=dtype)
    want = fa().paged_attn(*args, alibi_slopes=slopes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = fa().paged_attn(*args, alibi_slopes=slopes)
    for _ in range(4):
        o.fill_(float("nan"))
        assert torch.equal(fa().paged_attn(*args, alibi_slopes=slopes), want)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)


def test_a_step_in_inference_mode():
    f, i32 = fa(), dict(dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn(2, h, 3, 64, generator=g).half().to(DEV) for h in (2, 2, 8))

    def step():
        kc, vc = (torch.zeros(6, 2, 16, 64, dtype=torch.half, device=DEV) for _ in range(2))
        table = torch.zeros(2, 3, **i32)
        slots, lens, _ = f.paged_tables(table, torch.zeros(2, **i32), torch.full((2,), 3, **i32),
                                        torch.arange(6, **i32), torch.tensor([0, 6], **i32), 16, max_new=3)
        f.paged_append(k, v, kc, vc, slots)
        return f.paged_attn(q, kc, vc, table, lens)

    want = step()
    with torch.inference_mode():
        got = step()
        assert got.is_inference() and torch.equal(got, want)
