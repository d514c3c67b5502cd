"""Where the attention over the 4-bit pages once gave a wrong answer, held against the plain 64-bit form.
Tolerances are those of test_gpu_attention.py, from the roundings of the weights and of the result."""

import pytest
import torch

from test_gpu_attention import DEV, _attend_case, _attend_check, i32, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,length", [(64, 49152), (64, 40001), (128, 49152)])
def test_many_rows_over_a_table_of_many_parts(ops, D, length):
    """64 rows of one key head over a table of 393216 positions: no more parts than the join reads, all of which
    hold positions that count."""
    cache, tables, starts, q, k, v = _attend_case(ops, [length], [4], 16, 1, D, 16, "bf16", seed=D)
    wide = torch.full((1, 24576), -1, dtype=torch.int32)
    wide[:, :tables.shape[1]] = tables
    visible = [length - 3 + i for i in range(4)]
    out, lse = ops.kv.attend(q.to(DEV), cache, wide.to(DEV), i32(starts), i32(visible), max_queries=4, return_lse=True)
    _attend_check(out, lse, q, k, v, starts, visible, D ** -0.5)


@pytest.mark.parametrize("heads,rows", [(2, 1), (2, 60)])
def test_a_table_row_of_more_than_32_bits_of_positions(ops, heads, rows):
    """40000 columns of pages of 65536 positions, of which a request uses two."""
    length, page, D = 70000, 65536, 64
    cache, tables, starts, q, k, v = _attend_case(ops, [length], [rows], heads, 1, D, page, "bf16")
    wide = torch.full((1, 40000), -1, dtype=torch.int32)
    wide[:, :tables.shape[1]] = tables
    visible = [length - rows + 1 + i for i in range(rows)]
    out, lse = ops.kv.attend(q.to(DEV), cache, wide.to(DEV), i32(starts), i32(visible), max_queries=rows, return_lse=True)
    _attend_check(out, lse, q, k, v, starts, visible, D ** -0.5)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 60])
def test_entries_that_name_no_page_read_no_page(ops, rows, D):
    """Hidden pages between the others, at a tile's ends and behind the limit, while the cache's first page (which no
    table names) is NaN in every block: nothing of it arrives."""
    cache, tables, starts, q, k, v = _attend_case(ops, [400], [rows], 4, 1, D, 16, "bf16", seed=rows + D)
    data = torch.cat((torch.full_like(cache.data[:1], 255), cache.data))
    cache = ops.kv.KVCache(data, page=16, head_dim=D)
    tables = torch.where(tables >= 0, tables + 1, -1)
    hidden = torch.zeros(1, 400, dtype=torch.bool)
    for c, entry in ((0, -1), (1, cache.pages), (5, 2 ** 31 - 1), (7, -1), (8, -2 ** 31), (17, -1), (24, -1)):
        tables[0, c] = entry
        hidden[0, 16 * c:16 * c + 16] = True
    for limit in (400, 393, 272, 96, 40, 32):
        visible = [max(0, limit - i % 3) for i in range(rows)]
        for window in (0, 90):
            out, lse = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), window=window or None,
                                     max_queries=rows, return_lse=True)
            _attend_check(out, lse, q, k, v, starts, visible, D ** -0.5, window, hidden)


@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("window", [1, 20, 1000])
def test_a_window_whose_limit_lies_beyond_the_table(ops, rows, window):
    """A row sees the last `window` of its first `visible` positions; those beyond the table are among them and are
    not seen, so the window's other end moves with the limit."""
    length = 160
    cache, tables, starts, q, k, v = _attend_case(ops, [length] * 6, [rows] * 6, 4, 2, 128, 16, "bf16", extra_columns=0)
    hidden = torch.zeros(6, 2048, dtype=torch.bool)
    hidden[:, length:] = True
    more = torch.zeros(6, 2048, 2, 128, dtype=torch.float64)
    kw, vw = more.clone(), more.clone()
    kw[:, :length], vw[:, :length] = k, v
    visible = [x for x in (length, length + 1, length + 7, length + 20, 2000, 2 ** 31 - 1) for _ in range(rows)]
    out, lse = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), window=window, max_queries=rows,
                             return_lse=True)
    _attend_check(out, lse, q, kw, vw, starts, visible, 128 ** -0.5, window, hidden)


@pytest.mark.parametrize("requests,rows", [(256, 1), (1, 64)])
def test_large_values_under_scores_that_rise(ops, requests, rows):
    """Values of 2^100, and scores that lie 2^10 in weight above the first positions': the running sums stay
    finite, whatever maximum the weights are taken against."""
    length, D = 2048, 128
    cache, tables, _, _, k, v = _attend_case(ops, [length], [1], 1, 1, D, 64, "bf16", seed=3, extra_columns=0)
    kr, vr = torch.zeros(length, 1, D), torch.full((length, 1, D), 2.0 ** 100)
    kr[:, :, 0] = torch.where(torch.arange(length) % 512 < (256 if rows == 1 else 64), 0.0, 6.0)[:, None]
    if rows == 1:  # each of a workgroup's four waves begins with 64 low positions
        kr[512:, :, 0] = 6.0
    vr[:, :, 1::2] *= -1
    slots = (tables[0, :, None] * 64 + torch.arange(64)).flatten().int().to(DEV)
    ops.kv.write(cache, kr.bfloat16().to(DEV), vr.bfloat16().to(DEV), slots)
    kr, vr = (x.cpu().double() for x in ops.kv.read(cache, slots))
    k[0], v[0] = kr, vr
    q = torch.zeros(requests * rows, 1, D).bfloat16()
    q[:, :, 0] = 1
    starts = [rows * i for i in range(requests + 1)]
    scale = 10 / 6 * 0.6931471805599453
    out, lse = ops.kv.attend(q.to(DEV), cache, tables.expand(requests, -1).contiguous().to(DEV), i32(starts),
                             i32([length] * (requests * rows)), scale=scale, max_queries=rows, return_lse=True)
    assert bool(torch.isfinite(out.float()).all())
    _attend_check(out[:rows], lse[:rows], q[:rows], k, v, [0, rows], [length] * rows, scale)
    assert torch.equal(out, out[:1].expand(requests * rows, -1, -1)) and torch.equal(lse, lse[:1].expand_as(lse))
