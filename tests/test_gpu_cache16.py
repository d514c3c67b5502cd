"""The 16-bit cache on the GPU: rows appended with their turn, read back, and the attention over the pages, against plain
64-bit forms (core_testlib has the tolerances)."""

import math

import pytest
import torch

import core_testlib as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def ops(gdn):
    from cqgdn import kvcache, rotary

    class Both:
        pass

    Both.rotary, Both.kv = rotary, kvcache
    return Both


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- rows put into the pages -------------------------------------------------------------------------

@pytest.mark.parametrize("T,hq,hk,D,rotary_dim,page,adjacent,axes,dtype", [
    (1, 4, 1, 128, 128, 16, False, 1, "bf16"), (7, 16, 4, 128, 64, 64, True, 3, "fp16"), (130, 3, 3, 256, 64, 32, False, 3, "bf16"),
    (515, 14, 2, 64, 64, 16, True, 2, "bf16"), (33, 2, 2, 64, 10, 16, False, 1, "fp16"), (2100, 8, 2, 128, 128, 128, False, 3, "bf16"),
    (20, 0, 5, 256, 256, 16, False, 1, "bf16"), (9, 4, 2, 128, 0, 16, False, 1, "bf16"),
])
@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("bits", [4, 16])
def test_append_is_rotate_and_write(ops, T, hq, hk, D, rotary_dim, page, adjacent, axes, dtype, strided, bits):
    g = torch.Generator(device=DEV).manual_seed(T)
    t = DTYPES[dtype]
    rows = torch.randn(T, hq + 2 * hk, D + (3 if strided else 0), generator=g, device=DEV).to(t)[..., 1 if strided else 0:][..., :D]
    q, k, v = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
    n = rotary_dim // 2
    if n:
        sections = (n,) if axes == 1 else (n - 2 * (n // 3), n // 3, n // 3) if axes == 3 else (n // 2, n - n // 2)
        plan = ops.rotary.plan(rotary_dim, theta=1e6, sections=sections, adjacent=adjacent, device=DEV)
    else:
        plan = ops.rotary.RotaryPlan(torch.zeros(0, dtype=torch.int64, device=DEV), i32([]), adjacent)
    pos = torch.randint(-1000, 2 ** 30, (axes, T), generator=g, device=DEV)
    pos = pos if axes == 2 else pos.int()
    pages = -(-2 * T // page)
    cache, two = (ops.kv.KVCache.empty(pages, hk, page=page, head_dim=D, dtype=t, bits=bits, device=DEV) for _ in range(2))
    cache.data.random_(0, 100)
    two.data.copy_(cache.data)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:T].int()
    slots[::5] = -1
    if T > 2:
        slots[1], slots[2] = pages * page, 2 ** 31 - 1  # beyond the cache: skipped
    turned, keys = ops.rotary.rotate(q, k, pos, plan)
    ops.kv.write(two, keys, v, slots)
    out = ops.kv.append(cache, q, k, v, pos, plan, slots)
    assert torch.equal(out, turned) and torch.equal(cache.data, two.data)
    if bits == 16:
        real = ((slots >= 0) & (slots < pages * page))[:, None, None]
        gk, gv = ops.kv.read(cache, slots)
        assert torch.equal(gk, torch.where(real, keys, 0)) and torch.equal(gv, torch.where(real, v, 0))


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("loose", [0, 1, 2])
def test_append_with_one_operand_off_alignment(ops, loose, dtype, adjacent):
    """One of q, k and v begins off 16 bytes: the turns are those of the rotary kernel, whichever way either goes."""
    T, hq, hk, D = 201, 6, 2, 128
    g = torch.Generator(device=DEV).manual_seed(loose)
    rows = [torch.randn(T, h, D + 1, generator=g, device=DEV).to(DTYPES[dtype])[..., 1:] if i == loose else
            torch.randn(T, h, D, generator=g, device=DEV).to(DTYPES[dtype]) for i, h in enumerate((hq, hk, hk))]
    plan = ops.rotary.plan(64, theta=1e4, adjacent=adjacent, device=DEV)
    pos = torch.randint(0, 2 ** 20, (T,), generator=g, device=DEV).int()
    cache, two = (ops.kv.KVCache.empty(16, hk, page=16, head_dim=D, dtype=DTYPES[dtype], bits=16, device=DEV) for _ in range(2))
    cache.data.zero_(), two.data.zero_()
    slots = torch.randperm(256, generator=g, device=DEV)[:T].int()
    turned, keys = ops.rotary.rotate(rows[0], rows[1], pos, plan)
    ops.kv.write(two, keys, rows[2], slots)
    assert torch.equal(ops.kv.append(cache, *rows, pos, plan, slots), turned) and torch.equal(cache.data, two.data)


def test_write_changes_its_slots_alone(ops):
    cache = ops.kv.KVCache.empty(9, 3, page=16, head_dim=64, bits=16, device=DEV)
    cache.data.random_(0, 50)
    before = cache.data.clone()
    slots = torch.tensor([3, 143, 17, -1, 144, 100], dtype=torch.int32)
    k, v = (torch.randn(6, 3, 64, device=DEV).bfloat16() for _ in range(2))
    ops.kv.write(cache, k, v, slots.to(DEV))
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < 144:
            before[s // 16, :, 0, s % 16], before[s // 16, :, 1, s % 16] = k[i], v[i]
    assert torch.equal(cache.data, before)
    none = torch.zeros(0, 3, 64, dtype=torch.bfloat16, device=DEV)
    ops.kv.write(cache, none, none, i32([]))
    empty = ops.kv.KVCache.empty(0, 3, page=16, head_dim=64, bits=16, device=DEV)
    ops.kv.write(empty, k, v, slots.to(DEV))
    a, b = ops.kv.read(empty, slots.to(DEV))
    assert torch.equal(cache.data, before) and not bool(a.any()) and not bool(b.any())


# ---- attention ---------------------------------------------------------------------------------------

def make(ops, lengths, news, hq, hk, D, page, dtype, seed=0, size=1.0, extra_columns=1):
    """Requests of `lengths` cached positions with `news` rows, scattered pages; what no request wrote is NaN."""
    g = torch.Generator().manual_seed(seed)
    t, n = DTYPES[dtype], len(lengths)
    held = [-(-x // page) for x in lengths]
    cache = ops.kv.KVCache.empty(sum(held) + 2, hk, page=page, head_dim=D, dtype=t, bits=16, device=DEV)
    cache.data.fill_(math.nan)
    order = torch.randperm(sum(held) + 2, generator=g).tolist()
    tables = torch.full((n, max(held) + extra_columns), -1, dtype=torch.int32)
    rows = []
    for r, x in enumerate(lengths):
        tables[r, :held[r]] = torch.tensor([order.pop() for _ in range(held[r])], dtype=torch.int32)
        k, v = ((torch.randn(x, hk, D, generator=g) * size).to(t).to(DEV) for _ in range(2))
        if x:
            slots = (tables[r, :held[r], None] * page + torch.arange(page)).flatten()[:x].int().to(DEV)
            ops.kv.write(cache, k, v, slots)
        rows.append((k, v))
    starts = [0]
    for m in news:
        starts.append(starts[-1] + m)
    return cache, tables, starts, torch.randn(starts[-1], hq, D, generator=g).to(t).to(DEV), rows


def compare(out, lse, q, rows, starts, visible, *, window=0, hidden=None, scale=None, positions=None, **kw):
    for r, (k, v) in enumerate(rows):
        at = slice(starts[r], starts[r + 1])
        if starts[r] == starts[r + 1]:
            continue
        limit = torch.tensor(visible[at], dtype=torch.int64, device=DEV)
        j = torch.arange(k.shape[0], device=DEV)
        seen = (j < limit[:, None]) & (j >= limit[:, None] - window if window else j >= 0)
        if hidden is not None:
            seen &= ~hidden[r, :k.shape[0]].to(DEV)
        want, tol = R.attend_ref(q[at], k, v, None, limit, scale=q.shape[2] ** -0.5 if scale is None else scale, seen=seen,
                                 positions=None if positions is None else positions[at], **kw)
        R.check(out[at], want["out"], tol["out"], "out", q.dtype)
        if lse is not None:
            R.check(lse[at], want["lse"], tol["lse"], "lse", q.dtype)


CASES = [  # lengths, rows, Hq, Hk, D, page, type, window, cap, slopes
    ([1], [1], 1, 1, 128, 16, "bf16", 0, None, False),
    ([33], [1], 16, 4, 128, 16, "bf16", 0, 10.0, False),
    ([200, 1, 31, 0, 97], [1, 1, 1, 1, 1], 8, 2, 128, 32, "bf16", 0, None, True),
    ([70, 150], [5, 3], 14, 2, 64, 16, "fp16", 0, 20.0, True),
    ([300], [2], 8, 1, 256, 64, "bf16", 0, None, False),
    ([257, 64], [17, 40], 12, 4, 128, 64, "fp16", 0, None, False),
    ([500], [70], 4, 4, 64, 128, "bf16", 100, None, True),
    ([129, 700], [129, 90], 8, 2, 128, 16, "bf16", 37, 5.0, False),
    ([1500, 40], [3, 1], 32, 4, 128, 128, "bf16", 0, None, False),
    ([400, 310], [200, 310], 8, 4, 128, 32, "bf16", 0, None, False),
    ([330], [150], 16, 2, 256, 16, "fp16", 64, None, False),
    ([260], [260], 2, 2, 64, 64, "bf16", 0, 30.0, True),
    ([3000], [1], 4, 2, 256, 16, "fp16", 200, 8.0, True),
    ([5000, 700], [4, 4], 4, 1, 64, 16, "bf16", 0, None, False),
    ([2500], [600], 4, 2, 256, 64, "bf16", 0, None, True),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_attend(ops, case):
    lengths, news, hq, hk, D, page, dtype, window, cap, bias = case
    cache, tables, starts, q, rows = make(ops, lengths, news, hq, hk, D, page, dtype)
    visible = [max(0, x - m + 1 + i) for x, m in zip(lengths, news) for i in range(m)]  # causal; some see nothing
    slopes = torch.tensor([2.0 ** (-1 - i % 8) for i in range(hq)], device=DEV) if bias else None
    for bound in (max(news), 1, None):  # the bound sets the launch, not the result's meaning
        out, lse = ops.kv.attend(q, cache, tables.to(DEV), i32(starts), i32(visible), window=window or None, cap=cap,
                                 slopes=slopes, max_queries=bound, return_lse=True)
        compare(out, lse, q, rows, starts, visible, window=window, cap=cap, slopes=slopes)


@pytest.mark.parametrize("news", [[4, 3], [90, 50]], ids=str)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_of_any_limit(ops, news, D):
    """Limits in no order, zero, below zero and beyond the table; positions anywhere; rows of padding; odd strides of q."""
    cache, tables, starts, q, rows = make(ops, [100, 240], news, 4, 2, D, 16, "bf16", extra_columns=0)
    g = torch.Generator().manual_seed(1)
    n = sum(news)
    visible = [int(x) for x in torch.randint(-5, 100, (n,), generator=g)]
    visible[0], visible[1] = 0, -2 ** 31
    visible[news[0]] = 240
    where = torch.randint(-10, 250, (n + 3,), generator=g).int().to(DEV)
    slopes = torch.tensor([0.25, 0.0, 0.5, -0.01], device=DEV)
    wide = torch.zeros(n + 3, 5, D + 3, dtype=torch.bfloat16, device=DEV)
    wide[:n, :4, 1:-2] = q
    wide[n:] = 1
    x = wide[:, :4, 1:-2]
    for view in (x, x.contiguous(), x.transpose(0, 1).contiguous().transpose(0, 1)):
        out, lse = ops.kv.attend(view, cache, tables.to(DEV), i32(starts), i32(visible + [9, 9, 2 ** 31 - 1]), slopes=slopes,
                                 positions=where, max_queries=max(news), return_lse=True)
        compare(out, lse, q, rows, starts, visible, slopes=slopes, positions=where)
        assert not bool(out[n:].any()) and bool((lse[n:] == -math.inf).all())


@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_entries_that_name_no_page(ops, rows, D):
    cache, tables, starts, q, held = make(ops, [160], [rows], 4, 1, D, 16, "bf16")
    tables[0, 2], tables[0, 5], tables[0, 9] = -1, cache.pages, 2 ** 31 - 1
    hidden = torch.zeros(1, 160, dtype=torch.bool)
    for c in (2, 5, 9):
        hidden[0, 16 * c:16 * c + 16] = True
    for limit in (160, 48, 40):
        out, lse = ops.kv.attend(q, cache, tables.to(DEV), i32(starts), i32([limit] * rows), max_queries=rows, return_lse=True)
        compare(out, lse, q, held, starts, [limit] * rows, hidden=hidden)
    out = ops.kv.attend(q, cache, tables[:, 2:3].to(DEV), i32(starts), i32([16] * rows), max_queries=rows)
    assert not bool(out.any())


@pytest.mark.parametrize("rows,D", [(4, 64), (4, 128), (4, 256), (64, 128), (64, 256), (64, 64)])
@pytest.mark.parametrize("bad", [math.nan, -math.inf])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(ops, rows, D, bad):
    length = 150
    cache, tables, starts, q, _ = make(ops, [length], [rows], 2, 1, D, 32, "bf16")
    visible = [length - rows + 1 + i for i in range(rows)]
    at = length - rows // 2
    page, offset = int(tables[0, at // 32]), at % 32
    call = lambda: ops.kv.attend(q, cache, tables.to(DEV), i32(starts), i32(visible), max_queries=rows, return_lse=True)  # noqa: E731
    good, good_lse = call()
    sees = torch.tensor([x > at for x in visible], device=DEV)
    was = cache.data.clone()
    cache.data[page, :, 1, offset, 33] = bad
    out, lse = call()
    keep = [d for d in range(D) if d != 33]
    assert torch.equal(out[~sees], good[~sees]) and torch.equal(out[..., keep], good[..., keep]) and torch.equal(lse, good_lse)
    assert not bool(torch.isfinite(out[sees][..., 33]).any())
    cache.data.copy_(was)
    cache.data[page, :, 0, offset, D - 1] = math.nan
    out, lse = call()
    assert torch.equal(out[~sees], good[~sees]) and torch.equal(lse[~sees], good_lse[~sees])
    assert bool(torch.isnan(out[sees]).all()) and bool(torch.isnan(lse[sees]).all())


@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("cap", [None, 15.0])
def test_scale_and_large_scores(ops, scale, rows, cap):
    cache, tables, starts, q, held = make(ops, [90], [rows], 2, 2, 64, 16, "bf16", size=4.0)
    visible = [90] * rows
    out, lse = ops.kv.attend(q, cache, tables.to(DEV), i32(starts), i32(visible), scale=scale, cap=cap, max_queries=rows,
                             return_lse=True)
    compare(out, lse, q, held, starts, visible, scale=scale, cap=cap)


def test_nothing(ops):
    cache = ops.kv.KVCache.empty(2, 2, page=16, head_dim=128, bits=16, device=DEV)
    q = torch.randn(3, 4, 128, device=DEV).bfloat16()
    none = torch.empty(0, 4, 128, dtype=torch.bfloat16, device=DEV)
    assert ops.kv.attend(none, cache, i32([[0]]), i32([0, 0]), i32([])).shape == (0, 4, 128)
    out, lse = ops.kv.attend(q, cache, torch.zeros(0, 4, dtype=torch.int32, device=DEV), i32([0]), i32([5, 5, 5]), return_lse=True)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    out = ops.kv.attend(q, cache, torch.zeros(1, 0, dtype=torch.int32, device=DEV), i32([0, 3]), i32([5, 5, 5]))
    assert not bool(out.any())
    empty = ops.kv.KVCache.empty(0, 2, page=16, head_dim=128, bits=16, device=DEV)
    assert not bool(ops.kv.attend(q, empty, i32([[0]]), i32([0, 3]), i32([5, 5, 5])).any())
    # starts out of range are clamped
    cache, tables, starts, q, held = make(ops, [50, 50], [2, 2], 2, 1, 64, 16, "bf16")
    out = ops.kv.attend(q, cache, tables.to(DEV), i32([-3, 2, 900]), i32([50] * 4), max_queries=2)
    compare(out, None, q, held, [0, 2, 4], [50] * 4)


def test_a_cache_beyond_32_bits(ops):
    """Pages whose values lie beyond 2^32: written, read and attended to at the cache's end."""
    pages, heads, page, D = 36000, 8, 64, 128
    data = torch.empty(pages, heads, 2, page, D, dtype=torch.bfloat16, device=DEV)
    assert data.numel() > 2 ** 32
    cache = ops.kv.KVCache(data, page=page, head_dim=D)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32)
    slots = (table.T * page + torch.arange(page)).flatten()[:170].int().to(DEV)
    x = torch.randn(170, 2 * heads, D, generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    ops.kv.write(cache, x[:, :heads], x[:, heads:], slots)
    k, v = ops.kv.read(cache, slots)
    assert torch.equal(k, x[:, :heads]) and torch.equal(v, x[:, heads:])
    for rows in (1, 40):
        q = torch.randn(rows, 16, D, generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
        visible = [170 - rows + 1 + i for i in range(rows)]
        out = ops.kv.attend(q, cache, table.to(DEV), i32([0, rows]), i32(visible), max_queries=rows)
        compare(out, None, q, [(k, v)], [0, rows], visible)


def test_pages_of_many_tokens(ops):
    """A page of 65536 tokens of 256 dimensions, 64 MB a head: offsets within it at its end."""
    cache = ops.kv.KVCache.empty(2, 2, page=65536, head_dim=256, bits=16, device=DEV)
    k, v = (torch.randn(65500, 2, 256, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV).bfloat16() for i in (1, 2))
    ops.kv.write(cache, k, v, 65536 + torch.arange(65500, dtype=torch.int32, device=DEV))
    for rows in (1, 30):
        q = torch.randn(rows, 4, 256, generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
        visible = [65500 - rows + 1 + i for i in range(rows)]
        out, lse = ops.kv.attend(q, cache, i32([[1]]), i32([0, rows]), i32(visible), max_queries=rows, window=700, return_lse=True)
        compare(out, lse, q, [(k, v)], [0, rows], visible, window=700)


# ---- together ----------------------------------------------------------------------------------------

def serving_state(ops, seed, most, D=128):
    g = torch.Generator().manual_seed(seed)
    n, heads = 6, 2
    cached = torch.randint(0, 90, (n,), generator=g).int()
    new = torch.randint(1, most + 1, (n,), generator=g).int()
    tables = torch.full((n, 12), -1, dtype=torch.int32)
    ids = torch.randperm(80, generator=g).int().tolist()
    for r in range(n):
        for c in range(-(-int(cached[r]) // 16)):
            tables[r, c] = ids.pop()
    cache = ops.kv.KVCache.empty(80, heads, page=16, head_dim=D, bits=16, device=DEV)
    past = torch.randn(1280, 2 * heads, D, generator=g).bfloat16().to(DEV)
    ops.kv.write(cache, past[:, :heads], past[:, heads:], torch.arange(1280, dtype=torch.int32, device=DEV))
    x = torch.randn(int(new.sum()) + 3, 8, D, generator=g).bfloat16().to(DEV)
    return dict(cached=cached.to(DEV), new=new.to(DEV), tables=tables.to(DEV), free=i32(ids), count=i32([len(ids)]), cache=cache,
                q=x[:, :4], k=x[:, 4:6], v=x[:, 6:], plan=ops.rotary.plan(D, device=DEV), most=most)


def serving_step(ops, s):
    step = ops.kv.step_pages(s["cached"], s["new"], s["tables"], s["free"], s["count"], page=16, tokens=s["q"].shape[0])
    q = ops.kv.append(s["cache"], s["q"], s["k"], s["v"], step.positions, s["plan"], step.slots)
    return ops.kv.attend(q, s["cache"], s["tables"], step.starts, step.visible, cap=12.0, max_queries=s["most"], return_lse=True)


@pytest.mark.parametrize("most", [1, 30])
def test_a_step_on_another_stream_and_in_a_graph(ops, most):
    s, other = serving_state(ops, 1, most), serving_state(ops, 2, most)
    want = [x.clone() for x in serving_step(ops, s)]
    assert bool(torch.isfinite(want[0][:-3].float()).all()) and float(want[0].float().abs().max()) > 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = serving_step(ops, s)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = serving_step(ops, s)
    for replay in range(4):
        for x in held:
            x.fill_(7)
        serving_step(ops, other)  # eager work of other inputs between the replays
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), replay


@pytest.mark.parametrize("cap", [None, 6.0])
def test_prompt_served_as_it_was_trained(ops, cap):
    """A document through the training attention, and the same through the cache: a chunk, another chunk, single tokens.
    The rows are the same but for what their tolerances allow."""
    from cqgdn import attention

    T, D, hq, hk = 230, 128, 8, 2
    g = torch.Generator().manual_seed(4)
    x = torch.randn(T, hq + 2 * hk, D, generator=g).bfloat16().to(DEV)
    plan = ops.rotary.plan(D, theta=1e6, device=DEV)
    slopes = torch.tensor([2.0 ** -(i + 1) for i in range(hq)], device=DEV)
    q, k = ops.rotary.rotate(x[:, :hq], x[:, hq:hq + hk], torch.arange(T, device=DEV).int(), plan)
    limit = torch.arange(1, T + 1, dtype=torch.int32, device=DEV)
    v = x[:, hq + hk:]
    want, tol = R.attend_ref(q, k, v, torch.zeros_like(limit), limit, scale=D ** -0.5, cap=cap, slopes=slopes)
    R.check(attention.attend(q, k, v, limit, cap=cap, slopes=slopes), want["out"], tol["out"], "out", q.dtype)
    cache = ops.kv.KVCache.empty(20, hk, page=16, head_dim=D, bits=16, device=DEV)
    cached, tables, free, count = i32([0]), torch.full((1, 16), -1, dtype=torch.int32, device=DEV), torch.arange(20, dtype=torch.int32, device=DEV), i32([20])
    at = 0
    for n in (150, 60) + (1,) * 20:
        step = ops.kv.step_pages(cached, i32([n]), tables, free, count, page=16, tokens=n, in_place=True)
        y = ops.kv.append(cache, x[at:at + n, :hq], x[at:at + n, hq:hq + hk], v[at:at + n], step.positions, plan, step.slots)
        out = ops.kv.attend(y, cache, tables, step.starts, step.visible, cap=cap, slopes=slopes, max_queries=n)
        R.check(out, want["out"][at:at + n], tol["out"][at:at + n], "out", q.dtype)
        at += n
    assert at == T
