"""The paged entries have no derivative: what carries one into them is refused, in both
modes and before anything else is looked at, so that no GPU is needed to see it."""
import pytest
import torch
from torch.autograd import forward_ad

import fa_p100

NAMES = ("q", "k", "v", "k_cache", "v_cache", "alibi_slopes")


def calls(name, make):
    """The entries that take `name`, with make(tensor) in its place."""
    x = dict(q=torch.zeros(2, 4, 1, 64, dtype=torch.half), k=torch.zeros(2, 2, 1, 64, dtype=torch.half),
             v=torch.zeros(2, 2, 1, 64, dtype=torch.half),
             k_cache=torch.zeros(5, 2, 16, 64, dtype=torch.half),
             v_cache=torch.zeros(5, 2, 16, 64, dtype=torch.half), alibi_slopes=torch.ones(4))
    x[name] = make(x[name])
    ints, lens = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    if name not in ("k", "v"):
        yield lambda: fa_p100.paged_attn(x["q"], x["k_cache"], x["v_cache"], ints, lens,
                                         alibi_slopes=x["alibi_slopes"])
    if name not in ("q", "alibi_slopes"):
        yield lambda: fa_p100.paged_append(x["k"], x["v"], x["k_cache"], x["v_cache"], ints[:, :1])


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name):
    with forward_ad.dual_level():
        for make in (lambda t: forward_ad.make_dual(t, torch.ones_like(t)),
                     lambda t: forward_ad.make_dual(t, torch.ones_like(t))[:]):  # a view of one
            for call in calls(name, make):
                with pytest.raises(RuntimeError, match=f"{name} has a forward-mode tangent"):
                    call()
                with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                    call()
        for call in calls(name, lambda t: t):  # (the level alone is nothing)
            with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
                call()


@pytest.mark.parametrize("name", NAMES)
def test_what_requires_grad_is_refused(name):
    for make in (lambda t: t.clone().requires_grad_(), lambda t: t.clone().requires_grad_() * 2,
                 lambda t: torch.nn.Parameter(t)):
        for call in calls(name, make):
            with pytest.raises(RuntimeError, match=f"{name} requires grad"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="must be a CUDA tensor"):
                call()


def test_slopes_of_a_subclass_are_refused():
    class Wrapped(torch.Tensor):
        pass

    for call in calls("alibi_slopes", lambda t: t.as_subclass(Wrapped)):
        with pytest.raises(TypeError, match="plain tensors"):
            call()
