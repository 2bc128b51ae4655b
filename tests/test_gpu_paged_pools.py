"""Which caches paged_append may write: rows that lie apart, K's from V's too, whatever the
order of their dimensions. No counterpart in the reference."""
import random

import pytest
import torch

from test_gpu_paged import DEV, fa, pool_of

pytestmark = pytest.mark.gpu


def layout(r):
    """(sizes (P, Hkv, page, D), strides, distance of V from K): dimensions in any order,
    each stride passing what lies within it or now and then falling short, and V anywhere
    before, behind or among K's rows."""
    sizes = [r.choice([1, 2, 3, 5]), r.choice([1, 2, 3]), r.choice([1, 2, 4]), r.choice([8, 16, 24])]
    strides, last = [0, 0, 0, 1], sizes[3] - 1
    steps = [8]
    for i in r.sample(range(3), 3):
        least = last // 8 * 8 + 8
        strides[i] = max(8, least + 8 * r.choice([0, 0, 0, 1, 4, -1 if r.random() < 0.3 else 0]))
        strides[i] *= r.choice([1, 1, 2])
        last += (sizes[i] - 1) * strides[i]
        steps.append(strides[i])
    apart = r.choice([last // 8 * 8 + 8, r.choice(steps), sum(r.choice(steps) for _ in range(2)), 0])
    return sizes, strides, apart


def offsets(sizes, strides):
    at = torch.zeros(1, dtype=torch.long)
    for n, s in zip(sizes, strides):
        at = (at[:, None] + s * torch.arange(n)).flatten()
    return at


def check_layout(seed):
    """Against all elements' places, listed."""
    r = random.Random(seed)
    sizes, strides, apart = layout(r)
    at = offsets(sizes, strides)
    places = torch.cat([at, at + apart])
    overlap = places.unique().numel() < places.numel()
    size = int(places.max()) + 1
    pool = torch.full((size + 8,), -5.0, dtype=torch.half, device=DEV)
    kc, vc = (torch.as_strided(pool, sizes, strides, x) for x in (0, apart))
    if r.random() < 0.5:
        kc, vc = vc, kc
    P, Hkv, page, D = sizes
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(P * page, Hkv, D, generator=g).half().to(DEV) for _ in range(2))
    slots = torch.randperm(P * page, generator=g).to(torch.int32).to(DEV)
    if overlap:
        with pytest.raises(RuntimeError):
            fa().paged_append(k, v, kc, vc, slots)
        assert bool((pool == -5).all())
        return True
    fa().paged_append(k, v, kc, vc, slots)
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c[slots.long() // page, :, slots.long() % page], x)
    rest = torch.ones(size + 8, dtype=torch.bool)
    rest[places] = False
    assert bool((pool[rest.to(DEV)] == -5).all())
    return False


@pytest.mark.parametrize("group", range(5))
def test_rows_that_overlap_are_refused(group):
    refused = sum(check_layout(seed) for seed in range(40 * group, 40 * group + 40))
    assert 5 < refused < 35


def test_halves_of_many_kinds():
    """K and V in one pool, side by side at every level."""
    g = torch.Generator().manual_seed(1)
    P, Hkv, page, D = 5, 3, 4, 16
    k, v = (torch.randn(P * page, Hkv, D, generator=g).half().to(DEV) for _ in range(2))
    slots = torch.randperm(P * page, generator=g).to(torch.int32).to(DEV)
    for dim in range(5):
        sizes = [P, Hkv, page, D]
        both = torch.zeros(sizes[:dim] + [2] + sizes[dim:], dtype=torch.half, device=DEV)
        halves = both.unbind(dim)
        if dim == 4:  # (elements in turn: rows that are not dense)
            with pytest.raises(RuntimeError, match="dense rows"):
                fa().paged_append(k, v, *halves, slots)
            continue
        for kc, vc in (halves, halves[::-1]):
            fa().paged_append(k, v, kc, vc, slots)
            for c, x in ((kc, k), (vc, v)):
                assert torch.equal(c[slots.long() // page, :, slots.long() % page], x)
    every_other = torch.zeros(2 * P + 1, Hkv, page, D, dtype=torch.half, device=DEV)
    kc, vc = every_other[0:2 * P:2], every_other[3::2]  # among each other, and V's run past K's
    kc = kc[:vc.size(0)]
    few = slots[slots < kc.size(0) * page]
    fa().paged_append(k[:few.numel()], v[:few.numel()], kc, vc, few)
    assert torch.equal(vc[few.long() // page, :, few.long() % page], v[:few.numel()])


def test_one_cache_for_both():
    """Written twice with different rows it is refused, with the same ones not."""
    kc, _ = pool_of(4, 2, 16, 64, torch.half, "bhnd", fill=1.0)
    k, v = torch.zeros(3, 2, 64, dtype=torch.half, device=DEV), torch.ones(3, 2, 64, dtype=torch.half, device=DEV)
    s = torch.arange(3, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="overlap"):
        fa().paged_append(k, v, kc, kc, s)
    with pytest.raises(RuntimeError, match="overlap"):
        fa().paged_append(k, k, kc[:3], kc[1:], s)  # shifted by a page
    assert bool((kc == 1).all())
    fa().paged_append(k, k, kc, kc, s)
    assert bool((kc[0, :, :3] == 0).all()) and int((kc == 0).sum()) == k.numel()
