"""What a call of the attention over the pages sets aside, by the C ABI (no launch)."""

import pytest

from cqgdn import _lib


def size(T, N, heads=16, kv=4, D=128, most=1, columns=512, page=16):
    return _lib.lib().cqgdn_kv4_attend_workspace_size(T, N, heads, kv, D, most, columns, page)


def test_a_bound_far_too_small_does_not_grow_the_workspace():
    # rows of one request under a bound of one: as under their own bound
    for rows in (100, 4000, 100000):
        assert size(rows, 1, most=1) == size(rows, 1, most=rows)
    assert size(100000, 1, most=1) <= 2 * 100000 * 16 * 130 * 4
    assert size(8, 8, most=1) == size(8, 8, most=1) > 0


@pytest.mark.parametrize("D", [64, 128, 256])
def test_parts_end_where_the_requests_fill_the_gpu(D):
    assert size(2000, 2000, D=D) == 0            # one part each
    few = size(1, 1, D=D, columns=4096)
    assert few % (16 * (D + 2) * 4) == 0 and 1 < few // (16 * (D + 2) * 4) <= 512
    assert size(1, 1, D=D, columns=1) == 0       # 16 positions are one part


def test_sizes_that_no_call_has():
    assert size(0, 1) == size(4, -1) == size(4, 1, heads=6) == size(4, 1, D=96) == size(4, 1, most=0) == 0
    assert size(4, 1, columns=-1) == size(4, 1, page=24) == 0
