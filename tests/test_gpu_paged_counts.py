"""Calls of paged_append with more tokens than its indexes count. No counterpart in the
reference."""
import pytest
import torch

from test_gpu_paged import DEV, fa, pool_of

pytestmark = pytest.mark.gpu


def test_more_tokens_than_2_31_are_refused():
    """2^32 + 3 rows and slots of one place in memory each: their number is not cut to 3."""
    kc, vc = pool_of(4, 1, 16, 8, torch.half, "bhnd", fill=1.0)
    n = 2 ** 32 + 3
    k = torch.zeros(1, 1, 8, dtype=torch.half, device=DEV)
    s = torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="2\\^31"):
        fa().paged_append(k.expand(n, -1, -1), k.expand(n, -1, -1), kc, vc, s.expand(n))
    with pytest.raises(RuntimeError, match="2\\^31"):
        wide = k[:, :, None].expand(2 ** 16, -1, 2 ** 16, -1)
        fa().paged_append(wide, wide, kc, vc, s[None].expand(2 ** 16, 2 ** 16))
    assert bool((kc == 1).all())
