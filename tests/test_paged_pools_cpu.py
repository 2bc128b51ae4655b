"""The C entry refuses to write pools whose rows overlap, without a GPU: nothing is
launched."""
import pytest

from test_paged_cpu import cache, capi


@pytest.mark.parametrize("c", [
    dict(),                                                 # one pool for both
    dict(v=16 + 2 * 64), dict(v=16 + 2 * 2048),             # shifted by a row, by a page
    dict(k=16 + 2 * 1024),                                  # by a head, K behind V
    dict(v=16 + 2 * 32),                                    # by half a row
    dict(v=1 << 40, stride_row=56), dict(v=1 << 40, stride_row=0),  # rows within rows
    dict(v=1 << 40, stride_page=1024), dict(v=1 << 40, stride_head=64),
    dict(v=1 << 40, stride_head=0), dict(v=1 << 40, stride_page=0),
    dict(v=1 << 40, stride_head=1 << 62)])                  # past 64 bits
def test_pools_that_overlap(c):
    lib = capi()
    for D, other in ((64, 1 << 20), (64, 1 << 30)):
        rc = lib.fa_paged_append(1 << 20, (1 << 20) + other, 1024, 64, 64, 1024, 64, 64, 16, cache(**c), 1, 1, 2, D, None)
        assert rc == 10019
    assert b"overlap" in lib.fa_error_string(10019)
