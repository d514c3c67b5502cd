"""In how many parts a call of the attention over the pages takes the positions, by its workspace (no launch): the
join holds the weights of 512, whichever kernel made them."""

import pytest

from cqgdn import _lib


def parts(rows, D, kv, columns, page, N=1):
    """The parts of a call with `rows` rows of one key head a request (16 query heads each): its workspace holds an
    fp32 row of D values, a maximum and a sum for each of them."""
    heads, most = 16 * kv, rows // 16
    size = _lib.lib().cqgdn_kv4_attend_workspace_size(N * most, N, heads, kv, D, most, columns, page)
    n, rest = divmod(size, N * most * heads * (D + 2) * 4)
    assert rest == 0
    return max(n, 1)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [16, 32, 48, 64, 96, 128, 144, 1024])
def test_no_more_parts_than_the_join_reads(D, rows):
    for kv in (1, 2, 3, 8):
        for N in (1, 2, 5):
            for columns, page in ((1, 16), (100, 16), (24576, 16), (25000, 16), (4096, 128), (16384, 128), (30, 65536)):
                assert 1 <= parts(rows, D, kv, columns, page, N) <= 512, (kv, N, columns, page)


def test_long_tables_are_split():
    """One request of 16 to 128 rows does not stay in one workgroup over 393216 positions."""
    for D in (64, 128, 256):
        for rows in (16, 48, 64, 128):
            assert parts(rows, D, 1, 24576, 16) >= 256


@pytest.mark.parametrize("rows", [1, 2, 5, 70])
def test_a_launch_is_for_the_average_request_at_least(rows):
    """Eight requests of `rows` rows each under a bound of one: as under their own bound, so that a bound far too
    small does not multiply the parts of many rows."""
    size = lambda most: _lib.lib().cqgdn_kv4_attend_workspace_size(8 * rows, 8, 16, 4, 128, most, 512, 16)  # noqa: E731
    assert size(1) == size(rows)
    n, rest = divmod(size(rows), 8 * rows * 16 * 130 * 4)
    assert rest == 0 and n == {1: 11, 2: 11, 5: 11, 70: 5}[rows]  # three steps a wave; 512 workgroups over 96
