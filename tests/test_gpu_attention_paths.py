"""Where the attention over the 4-bit pages takes another way: positions in many parts and their joins, tables
longer than a wave holds at once, maxima that move at every step, rows that begin to see at different steps.
Tolerances are those of test_gpu_attention.py, from the roundings of the weights and of the result."""

import math

import pytest
import torch

from test_gpu_attention import (DEV, DTYPES, R, _attend_case, _attend_check, _pages_case, _pages_check,  # noqa: F401
                                _rotary_case, _rotary_close, i32, ops)

pytestmark = pytest.mark.gpu


def _causal(lengths, news):
    return [max(0, x - m + 1 + i) for x, m in zip(lengths, news) for i in range(m)]


def _run(ops, case, visible, scale=None, window=0, max_queries=None):
    cache, tables, starts, q, k, v = case
    D = q.shape[2]
    news = [b - a for a, b in zip(starts, starts[1:])]
    scale = D ** -0.5 if scale is None else scale
    out, lse = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), window=window or None, scale=scale,
                             max_queries=max_queries or max(news), return_lse=True)
    _attend_check(out, lse, q, k, v, starts, visible, scale, window)
    again, lse2 = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), window=window or None, scale=scale,
                                max_queries=max_queries or max(news), return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)  # nothing depends on timing


@pytest.mark.parametrize("lengths,news,hq,hk,D,page,dtype,window", [
    ([2100, 1025], [70, 13], 8, 2, 128, 32, "bf16", 0),      # many rows, positions in parts, a part that is empty
    ([2600], [33], 8, 1, 64, 16, "fp16", 0),
    ([1600, 700], [50, 64], 4, 2, 256, 64, "bf16", 0),
    ([1900], [140], 16, 2, 128, 16, "fp16", 1300),           # parts within a window
    ([1300], [130], 16, 1, 128, 64, "bf16", 0),              # 2080 rows in parts: joined some lanes a row
])
def test_many_rows_in_parts(ops, lengths, news, hq, hk, D, page, dtype, window):
    case = _attend_case(ops, lengths, news, hq, hk, D, page, dtype, seed=sum(lengths))
    _run(ops, case, _causal(lengths, news), window=window)


@pytest.mark.parametrize("n,length,hq,hk,D,page", [
    (1, 70000, 2, 1, 64, 64),      # more than 256 parts
    (130, 1500, 8, 8, 64, 16),     # one part of more than 64 pages
    (40, 4100, 8, 8, 64, 16),      # parts of more than 64 pages
    (200, 700, 16, 1, 128, 32),    # 3200 rows in parts
])
def test_single_tokens_over_long_tables(ops, n, length, hq, hk, D, page):
    g = torch.Generator().manual_seed(n)
    lengths = [length] + [int(x) for x in torch.randint(1, length + 1, (n - 1,), generator=g)]
    case = _attend_case(ops, lengths, [1] * n, hq, hk, D, page, "bf16", seed=n)
    _run(ops, case, lengths)


@pytest.mark.parametrize("window", [16, 100, 1000, 2 ** 31 - 1])
def test_single_tokens_with_windows(ops, window):
    lengths = [1500, 3, 99, 100, 101, 1024, 64, 0, 1]
    case = _attend_case(ops, lengths, [1] * len(lengths), 4, 2, 128, 16, "bf16", seed=4)
    _run(ops, case, lengths, window=window)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("falling", [False, True])
def test_maxima_that_move_at_every_step(ops, dtype, rows, falling):
    """Keys that grow (or shrink) along the positions: the largest score of every 64 positions is far above, or
    below, that of those before."""
    length, D = 640, 128
    cache, tables, starts, q, k, v = _attend_case(ops, [length], [rows], 2, 1, D, 32, dtype, seed=rows)
    q = q.abs() + 0.5  # scores of one sign
    grow = torch.linspace(0.05, 6.0, length).flip(0) if falling else torch.linspace(0.05, 6.0, length)
    rng = torch.Generator().manual_seed(9)
    kr = ((torch.rand(length, 1, D, generator=rng) + 0.5) * grow[:, None, None]).to(DTYPES[dtype]).to(DEV)
    vr = torch.randn(length, 1, D, generator=rng).to(DTYPES[dtype]).to(DEV)
    slots = (tables[0, :length // 32, None] * 32 + torch.arange(32)).flatten().int().to(DEV)
    ops.kv.write(cache, kr, vr, slots)
    kr, vr = ops.kv.read(cache, slots)
    k[0, :length], v[0, :length] = kr.cpu().double(), vr.cpu().double()
    for scale in (0.02, 0.3):
        _run(ops, (cache, tables, starts, q, k, v), [length - 3] * rows, scale=scale)
        _run(ops, (cache, tables, starts, q, k, v), [length - 3] * rows, scale=-scale)


@pytest.mark.parametrize("rows,D", [(6, 128), (90, 128), (90, 256), (90, 64)])
def test_rows_that_begin_to_see_at_different_steps(ops, rows, D):
    """Limits spread over the positions with a short window: at any step some rows of a tile see everything, some
    a part and some nothing; and a NaN value in a part of its own reaches the rows that see it only."""
    length, window = 1300, 40
    case = _attend_case(ops, [length], [rows], 2, 1, D, 16, "bf16", seed=rows + D)
    g = torch.Generator().manual_seed(D)
    visible = [int(x) for x in torch.randint(0, length + 1, (rows,), generator=g)]
    visible[:5] = [0, 1, 40, 41, length]
    _run(ops, case, visible, window=window)
    cache, tables, starts, q, k, v = case
    good = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), window=window, max_queries=rows)
    at = 700
    slot = i32([int(tables[0, at // 16]) * 16 + at % 16])
    kr, vr = (x[0, at:at + 1].bfloat16().to(DEV) for x in (k, v))
    vr = vr.clone()
    vr[..., 5] = math.nan
    ops.kv.write(cache, kr, vr, slot)
    out = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), window=window, max_queries=rows)
    sees = torch.tensor([x > at and x - window <= at for x in visible], device=DEV)
    assert torch.equal(out[~sees], good[~sees])
    assert torch.equal(out[sees][..., 32:], good[sees][..., 32:]) and bool(torch.isnan(out[sees][..., :32]).all())


@pytest.mark.parametrize("lengths,news,pad,D", [
    ([3000], [1], 11, 128),                # single tokens, positions in parts
    ([300] * 8, [1] * 8, 1, 64),           # in one part
    ([300] * 32, [1] * 32, 320, 64),       # more rows of padding than of requests
    ([3000], [1], 500, 128),               # so many that the launch is for many rows
    ([300, 20, 7], [1, 0, 1], 700, 256),
    ([2100], [70], 300, 128),              # many rows, in parts
    ([200] * 12, [64] * 12, 2000, 64),     # and in one
    ([], [], 90, 128),                     # nothing but padding
    ([], [], 1, 128),
])
def test_rows_behind_the_requests(ops, lengths, news, pad, D):
    """Zero and -inf, and the requests' rows hold beside them."""
    n, rows, hq, hk = len(lengths), sum(news), 8, 2
    cache, tables, starts, q, k, v = _attend_case(ops, lengths or [16], news or [1], hq, hk, D, 16, "bf16", seed=pad)
    tables, starts, q = (tables, starts, q) if n else (tables[:0], [0], q[:0])
    more = torch.cat([q, torch.full((pad, hq, D), math.nan, dtype=q.dtype)]).to(DEV)
    visible = i32(_causal(lengths, news) + [7] * pad)
    junk = [torch.full(s, 3.0, dtype=t, device=DEV) for s, t in ((more.shape, q.dtype), (more.shape[:2], torch.float32))]
    del junk  # what new tensors hold is nobody's zeros
    out, lse = ops.kv.attend(more, cache, tables.to(DEV), i32(starts), visible, max_queries=max(news, default=1),
                             return_lse=True)
    assert bool((out[rows:] == 0).all()) and bool((lse[rows:] == -math.inf).all())
    if n:
        same, lse2 = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), visible[:rows], max_queries=max(news),
                                   return_lse=True)
        _attend_check(out[:rows], lse[:rows], q, k, v, starts, _causal(lengths, news), D ** -0.5, 0)
        _attend_check(same, lse2, q, k, v, starts, _causal(lengths, news), D ** -0.5, 0)


def test_a_row_does_not_depend_on_the_rows_beside_it(ops):
    """The same row alone in its call and among others of its request, by the same kernel."""
    length = 900
    cache, tables, starts, q, k, v = _attend_case(ops, [length], [60], 4, 2, 128, 32, "bf16", seed=8)
    visible = [length - 59 + i for i in range(60)]
    out = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), max_queries=60)
    other = q.clone()
    other[:30] *= 37.0
    again = ops.kv.attend(other.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), max_queries=60)
    assert torch.equal(out[30:], again[30:])


@pytest.mark.parametrize("n,context,most,page,spare,padding", [
    (1500, 50, 9, 16, 3000, 3),     # two rounds of requests, rows by a launch of their own
    (1024, 40, 8, 16, 900, 100),    # a full round, the pool too small
    (2049, 64, 3, 32, 5000, 0),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_step_pages_over_rounds(ops, n, context, most, page, spare, padding, in_place):
    cached, new, tables, free, count = _pages_case(n, context, most, page, spare, n, end=0.3)
    _pages_check(ops, cached, new, tables, free, count, page, int(new.clamp(min=0).sum()) + padding, in_place)


@pytest.mark.parametrize("case", [  # T, Hq, Hk, D, rotary, sections, mixed, adjacent, type, far
    (3, 2, 1, 1030, 514, (100, 100, 57), True, False, "fp32", 5),    # more units than a workgroup has threads
    (2, 1, 1, 1030, 1030, (515,), False, True, "bf16", 0),
    (2, 1, 2, 8448, 8448, (4224,), False, False, "bf16", 3),         # more pairs than its LDS holds
    (2, 1, 1, 8448, 8448, (2000, 2224), False, True, "fp16", 70),
    (1500, 5, 3, 128, 128, (64,), False, True, "bf16", 11),          # ragged numbers of items, a last workgroup short
    (2051, 1, 1, 64, 16, (2, 3, 3), True, False, "fp32", 0),
    (19, 64, 1, 256, 256, (128,), False, False, "fp16", 0),
], ids=str)
def test_rotate_sizes(ops, case):
    p, q, k, pos, freq, axis = _rotary_case(ops, case)
    r, adjacent, dtype = case[4], case[7], case[8]
    y, z = ops.rotary.rotate(q.to(DEV), k.to(DEV), pos.to(DEV), p)
    _rotary_close(y, q, R.rotate_ref(q, pos, freq, axis, adjacent), r, adjacent, dtype)
    _rotary_close(z, k, R.rotate_ref(k, pos, freq, axis, adjacent), r, adjacent, dtype)
    none = torch.empty(case[0], 0, case[3], dtype=q.dtype, device=DEV)  # one of the two may have no heads
    a, b = ops.rotary.rotate(q.to(DEV), none, pos.to(DEV), p)
    assert torch.equal(a, y) and b.shape == none.shape
    a, b = ops.rotary.rotate(none, k.to(DEV), pos.to(DEV), p)
    assert torch.equal(b, z) and a.shape == none.shape


def test_rotate_gradients_of_one_input_and_of_gradients(ops):
    g = torch.Generator().manual_seed(2)
    p = ops.rotary.plan(32, sections=(4, 6, 6), mixed=True, device=DEV)
    q = torch.randn(9, 2, 64, generator=g).to(DEV).requires_grad_()
    k = torch.randn(9, 1, 64, generator=g).to(DEV)
    pos = torch.randint(0, 900, (3, 9), generator=g).to(DEV)
    y, z = ops.rotary.rotate(q, k, pos, p)
    w = torch.randn(9, 2, 64, generator=g).to(DEV).requires_grad_()
    (dq,) = torch.autograd.grad(y, q, w, create_graph=True)
    # dq is linear in w: its gradient is the turn itself
    u = torch.randn(9, 2, 64, generator=g).to(DEV)
    (dw,) = torch.autograd.grad(dq, w, u)
    assert torch.equal(dw, ops.rotary.rotate(u, k, pos, p)[0])
    assert torch.equal(ops.rotary.rotate(q.detach(), k, pos, p)[0], y.detach())
    with torch.no_grad():
        assert not ops.rotary.rotate(q, k, pos, p)[0].requires_grad
    # the turn back of the turn: off by the roundings of two turns, each at most 6 steps of 2^-24 of |a| + |b|
    back = torch.autograd.grad(ops.rotary.rotate(q, k, pos, p)[0], q, y.detach())[0]
    assert float((back - q.detach()).abs().max()) <= 2 * 6 * 2 ** -24 * 2 * 2 ** 0.5 * float(q.detach().abs().max())


def test_rotate_gradient_in_a_graph(ops):
    g = torch.Generator().manual_seed(3)
    p = ops.rotary.plan(64, device=DEV)
    q0, k0 = torch.randn(33, 4, 64, generator=g).to(DEV), torch.randn(33, 2, 64, generator=g).to(DEV)
    w0, w1 = torch.randn(33, 4, 64, generator=g).to(DEV), torch.randn(33, 2, 64, generator=g).to(DEV)
    pos = torch.arange(33, device=DEV)

    def step(q, k):
        return torch.autograd.grad(ops.rotary.rotate(q, k, pos, p), (q, k), (w0, w1))

    want = step(q0.clone().requires_grad_(), k0.clone().requires_grad_())
    q, k = q0.clone().requires_grad_(), k0.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = step(q, k)
    for _ in range(3):
        for x in held:
            x.zero_()
        step(q0.clone().requires_grad_(), k0.clone().requires_grad_())
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


@pytest.mark.parametrize("T,heads,D,dtype", [(2101, 16, 128, "bf16"), (1100, 16, 256, "fp16"), (9001, 8, 64, "bf16")])
def test_write_and_read_of_many_rows(ops, T, heads, D, dtype):
    """Sizes where a thread takes several rows; skipped slots among them, tokens in no order."""
    g = torch.Generator().manual_seed(T)
    t, page = DTYPES[dtype], 32
    pages = -(-T // page) + 2
    cache = ops.kv.KVCache.empty(pages, heads, page=page, head_dim=D, dtype=t, device=DEV)
    rows = (torch.randn(T, 2 * heads, D, generator=g) * torch.exp2(torch.randint(-5, 5, (T, 1, 1), generator=g))).to(t).to(DEV)
    slots = torch.randperm(pages * page, generator=g)[:T].int()
    slots[::11] = -1
    k, v = rows[:, :heads], rows[:, heads:]
    ops.kv.write(cache, k, v, slots.to(DEV))
    real = (slots >= 0).to(DEV)[:, None, None]
    for got, x in zip(ops.kv.read(cache, slots.to(DEV)), (k, v)):
        assert torch.equal(got.cpu().double(), torch.where(real.cpu(), R.encode_ref(x.cpu()), 0.0))
    unwritten = torch.tensor(sorted(set(range(pages * page)) - set(slots.tolist())), dtype=torch.int32, device=DEV)
    assert not any(bool(x.any()) for x in ops.kv.read(cache, unwritten))
