"""The attention layers' operators on the GPU against plain 64-bit forms, where they can go wrong.

Tolerances: a rounding to a type is off by at most half a step, u = finfo(type).eps / 2 of the value.
Attention rounds each weight p_j and the result once (u each), so |out - exact| <= u (A + |exact|) with
A = sum w_j |v_j|; its scores are fp32 sums of D exact products, off by at most (D + 3) 2^-24 times the
sum of the products' magnitudes, which moves every weight by that factor."""

import math

import pytest
import torch

import attn_testlib as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ops(gdn):
    from cqgdn import kvcache, rotary

    class Both:
        pass

    Both.rotary, Both.kv = rotary, kvcache
    return Both


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---- rotary ----------------------------------------------------------------------------------------

ROTARY = [  # T, Hq, Hk, D, rotary, sections, mixed, adjacent, type, far
    (1, 16, 4, 128, 128, (16, 24, 24), False, False, "bf16", 0),
    (37, 4, 4, 256, 64, (11, 11, 10), True, False, "bf16", 10 ** 6),
    (65, 3, 1, 64, 32, (16,), False, True, "fp16", 2 ** 30),
    (130, 2, 7, 128, 128, (8, 28, 28), True, True, "fp32", -70000),
    (5, 1, 1, 6, 2, (1,), False, False, "bf16", 17),        # heads of no vector's size
    (9, 2, 3, 80, 40, (20,), False, True, "fp32", 0),
    (700, 16, 2, 128, 64, (32,), False, False, "fp32", 2 ** 40),
]


def _rotary_case(ops, case, strided=False):
    T, hq, hk, D, r, sections, mixed, adjacent, dtype, far = case
    g = torch.Generator().manual_seed(T)
    p = ops.rotary.plan(r, theta=1e6, sections=sections, mixed=mixed, adjacent=adjacent, device=DEV)
    rows = torch.randn(T, (hq + hk) * D + (9 if strided else 0), generator=g).to(DTYPES[dtype])
    q = rows[:, 1 if strided else 0:][:, :hq * D].unflatten(1, (hq, D))
    k = rows[:, (hq * D + (2 if strided else 0)):][:, :hk * D].unflatten(1, (hk, D))
    pos = torch.randint(0, 5000, (len(sections), T), generator=g) + far
    if abs(far) < 2 ** 31 - 5000:
        pos = pos.int()
    freq = R.frequencies(10 ** 6, r)
    axis = p.axis.tolist()
    return p, q, k, pos, freq, axis


def _rotary_close(y, x, ref, r, adjacent, dtype):
    """sine, cosine, two products and a sum in fp32: each term off by at most 6 steps of 2^-24 of |a| + |b|
    (angle 2^-32 turns, polynomials 2^-28, their rounding 3 steps, the product and the sum)."""
    u = torch.finfo(DTYPES[dtype]).eps / 2
    a = x.double().abs()
    n = r // 2
    pair = a.clone()
    if adjacent:
        pair[..., 0:r:2] = pair[..., 1:r:2] = a[..., 0:r:2] + a[..., 1:r:2]
    else:
        pair[..., :n] = pair[..., n:r] = a[..., :n] + a[..., n:r]
    tol = 6 * 2 ** -24 * pair * (1 + u) + u * ref.abs() + torch.finfo(DTYPES[dtype]).smallest_normal * u
    err = (y.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    assert torch.equal(y[..., r:].cpu(), x[..., r:]), "values behind rotary_dim pass unchanged"


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("case", ROTARY, ids=str)
def test_rotate_forward_and_gradient(ops, case, strided):
    p, q, k, pos, freq, axis = _rotary_case(ops, case, strided)
    r, adjacent, dtype = case[4], case[7], case[8]
    qd, kd = q.to(DEV), k.to(DEV)
    if strided:  # views of wider, odd rows
        wide = torch.zeros(q.shape[0], q.shape[1] * q.shape[2] + 3, dtype=q.dtype, device=DEV)
        wide[:, 1:-2] = qd.flatten(1)
        qd = wide[:, 1:-2].unflatten(1, q.shape[1:])
    qd.requires_grad_()
    kd.requires_grad_()
    y, z = ops.rotary.rotate(qd, kd, pos.to(DEV), p)
    _rotary_close(y.detach(), q, R.rotate_ref(q, pos, freq, axis, adjacent), r, adjacent, dtype)
    _rotary_close(z.detach(), k, R.rotate_ref(k, pos, freq, axis, adjacent), r, adjacent, dtype)
    dy, dz = torch.randn(y.shape).to(q.dtype), torch.randn(1, k.shape[1], 1).to(q.dtype).expand(k.shape)
    dq, dk = torch.autograd.grad((y, z), (qd, kd), (dy.to(DEV), dz.to(DEV)))
    _rotary_close(dq, dy, R.rotate_ref(dy, pos, freq, axis, adjacent, -1.0), r, adjacent, dtype)
    _rotary_close(dk, dz, R.rotate_ref(dz, pos, freq, axis, adjacent, -1.0), r, adjacent, dtype)


def test_rotate_gradient_against_differences(ops):
    p, q, k, pos, _, _ = _rotary_case(ops, (33, 2, 1, 64, 32, (4, 6, 6), True, False, "fp32", 900))
    q, k, pos = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_(), pos.to(DEV)
    w, v = torch.randn_like(q), torch.randn_like(k)

    def loss(a, b):
        y, z = ops.rotary.rotate(a, b, pos, p)
        return (y.double() * w.double()).sum() + (z.double() * v.double()).sum()

    dq, dk = torch.autograd.grad(loss(q, k), (q, k))
    for x, dx, which in ((q, dq, 0), (k, dk, 1)):
        d = torch.randn_like(x)
        with torch.no_grad():
            h = 0.25  # the map is linear: a difference has rounding error only
            plus, minus = ((q + h * d, k) if which == 0 else (q, k + h * d)), ((q - h * d, k) if which == 0 else (q, k - h * d))
            difference = (loss(*plus) - loss(*minus)) / (2 * h)
        exact = (dx.double() * d.double()).sum()
        # each of the 4 roundings of a value is below 2^-23 of |x| + |y|, random over the values
        assert abs(float(difference - exact)) <= 8 * 2 ** -24 / h * x.numel() ** 0.5 * 40


def test_rotate_empty_one_axis_and_packed(ops):
    p = ops.rotary.plan(64, device=DEV)
    q = torch.zeros(0, 4, 64, device=DEV)
    y, z = ops.rotary.rotate(q, q[:, :1], torch.zeros(0, dtype=torch.int32, device=DEV), p)
    assert y.shape == (0, 4, 64) and z.shape == (0, 1, 64)
    q, pos = torch.randn(1, 5, 2, 64, device=DEV), torch.arange(5, device=DEV)
    y, z = ops.rotary.rotate(q, q, pos, p)
    a, _ = ops.rotary.rotate(q[0], q[0], pos[None].int(), p)
    assert y.shape == q.shape and torch.equal(y[0], a) and torch.equal(y, z)
    assert torch.equal(y[0, 0], q[0, 0]), "position 0 turns nothing"


# ---- pages -----------------------------------------------------------------------------------------

def _pages_case(n, context, most, page, spare, seed, columns=None, end=0.1):
    g = torch.Generator().manual_seed(seed)
    cached = torch.randint(0, context + 1, (n,), generator=g)
    new = torch.randint(0, most + 1, (n,), generator=g)
    new[torch.rand(n, generator=g) < end] = -1
    held = -(-cached // page)
    columns = columns or -(-(context + most) // page)
    ids = torch.randperm(int(held.sum()) + spare, generator=g).int()
    tables = torch.full((n, columns), -1, dtype=torch.int32)
    at = 0
    for r in range(n):
        tables[r, :held[r]] = ids[at:at + held[r]]
        at += int(held[r])
    free = torch.full((len(ids),), -7, dtype=torch.int32)
    free[:spare] = ids[at:]
    return cached.int(), new.int(), tables, free, spare


def _pages_check(ops, cached, new, tables, free, count, page, tokens, in_place=False):
    want = R.pages_ref(cached.tolist(), new.tolist(), tables.tolist(), free.tolist(), count, page, tokens)
    c, t, f, k = cached.to(DEV), tables.to(DEV), free.to(DEV), i32([count])
    step = ops.kv.step_pages(c, new.to(DEV), t, f, k, page=page, tokens=tokens, in_place=in_place)
    got = {name: getattr(step, name).tolist() for name in step._fields} | dict(tables=t.tolist(), free=f.tolist())
    if in_place:
        got |= dict(lengths=c.tolist(), free_count=k.tolist())
    for name, x in want.items():
        assert got[name] == x, name


@pytest.mark.parametrize("n,context,most,page,spare,padding", [
    (1, 0, 1, 16, 1, 0), (1, 40, 7, 16, 0, 3), (64, 300, 1, 64, 70, 0), (7, 100, 33, 32, 6, 11), (5, 64, 64, 64, 2, 1),
    (1000, 50, 3, 16, 120, 5), (1025, 30, 9, 16, 900, 0), (2500, 20, 2, 128, 400, 1), (300, 200, 40, 16, 700, 999),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_step_pages(ops, n, context, most, page, spare, padding, in_place):
    cached, new, tables, free, count = _pages_case(n, context, most, page, spare, n + spare)
    tokens = int(new.clamp(min=0).sum()) + padding
    _pages_check(ops, cached, new, tables, free, count, page, tokens, in_place)


def test_step_pages_edges(ops):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    t = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    # no request; no token; all idle; no table column
    _pages_check(ops, z(0), z(0), z(0, 3), t([4, 5]), 2, 16, 5)
    _pages_check(ops, z(2), z(2), z(2, 3), t([4, 5]), 2, 16, 0)
    _pages_check(ops, z(2), t([1, 0]), z(2, 0), t([4]), 1, 16, 2)
    # rows that do not fit: beyond the table, beyond the buffer, and the one behind that does
    _pages_check(ops, t([30, 0, 5]), t([3, 9, 2]), t([[1, 2], [3, 4], [5, 6]]), t([7, 8, 9]), 3, 16, 11)
    # counts and lengths out of range are clamped: a negative length, a pool count beyond the pool, below 0
    _pages_check(ops, t([-5, 3]), t([2, 1]), t([[-1, -1], [0, -1]]), t([7, 8]), 9, 16, 3)
    _pages_check(ops, t([0, 3]), t([2, 1]), t([[-1, -1], [0, -1]]), t([7, 8]), -4, 16, 3)
    # returned pages beyond the pool's size are dropped; huge lengths return no more than the table holds
    _pages_check(ops, t([64, 2 ** 31 - 1]), t([-1, -1]), t([[1, 2, 3, 4], [5, 6, 7, 8]]), t([9, 0, 0]), 1, 16, 0)
    # an entry that names no page, a slot beyond 32 bits, new tokens beyond any buffer
    _pages_check(ops, t([5, 20]), t([2, 2]), t([[-1, 3], [2, -9]]), t([7]), 1, 16, 4)
    step = ops.kv.step_pages(i32([1]), i32([1]), i32([[2 ** 31 - 1]]), i32([0]), i32([0]), page=64, tokens=1)
    assert step.slots.tolist() == [-1] and step.visible.tolist() == [0]
    step = ops.kv.step_pages(i32([0] * 3), i32([2 ** 31 - 1] * 3), i32([[0]] * 3), i32([0]), i32([1]), page=16, tokens=9)
    assert step.starts.tolist() == [0] + [2 ** 31 - 1] * 3 and step.admitted.tolist() == [0] * 3
    assert step.slots.tolist() == [-1] * 9 and step.free_count.tolist() == [1]


def test_step_pages_wide_table_rows(ops):
    cached, new, tables, free, count = _pages_case(50, 90, 5, 16, 40, 3)
    wide = torch.full((50, tables.shape[1] + 5), 77, dtype=torch.int32, device=DEV)
    wide[:, :tables.shape[1]] = tables.to(DEV)
    tokens = int(new.clamp(min=0).sum())
    ops.kv.step_pages(cached.to(DEV), new.to(DEV), wide[:, :tables.shape[1]], free.to(DEV), i32([count]), page=16,
                      tokens=tokens)
    want = R.pages_ref(cached.tolist(), new.tolist(), tables.tolist(), free.tolist(), count, 16, tokens)
    assert wide[:, :tables.shape[1]].tolist() == want["tables"] and bool((wide[:, tables.shape[1]:] == 77).all())


# ---- the cache -------------------------------------------------------------------------------------

@pytest.mark.parametrize("T,heads,D,page,dtype", [
    (1, 1, 64, 16, "bf16"), (3, 5, 128, 32, "fp16"), (129, 4, 256, 64, "bf16"), (515, 2, 128, 16, "bf16"),
    (40, 16, 64, 128, "fp16"),
])
def test_write_and_read(ops, T, heads, D, page, dtype):
    g = torch.Generator().manual_seed(T)
    t = DTYPES[dtype]
    rows = (torch.randn(T, 2 * heads + 1, D, generator=g) * torch.exp2(torch.randint(-9, 9, (T, 1, 1), generator=g))).to(t)
    pages = -(-2 * T // page)
    cache = ops.kv.KVCache.empty(pages, heads, page=page, head_dim=D, dtype=t, device=DEV)
    cache.data.random_(0, 200)
    before = cache.data.clone()
    slots = torch.randperm(pages * page, generator=g)[:T].int()
    slots[::7] = -1
    if T > 2:
        slots[1] = pages * page  # beyond the cache: skipped too
    d = rows.to(DEV)
    k, v = d[:, 1:heads + 1], d[:, heads + 1:]  # strided views
    ops.kv.write(cache, k, v, slots.to(DEV))
    gk, gv = ops.kv.read(cache, slots.to(DEV))
    real = ((slots >= 0) & (slots < pages * page))[:, None, None]
    for got, x in ((gk, k), (gv, v)):
        assert got.dtype == t and torch.equal(got.cpu().double(), torch.where(real, R.encode_ref(x.cpu()), 0.0))
    # nothing else was written
    other = torch.tensor(sorted(set(range(pages * page)) - set(slots.tolist())), dtype=torch.int32, device=DEV)
    old = ops.kv.KVCache(before, page=page, head_dim=D, dtype=t)
    for a, b in zip(ops.kv.read(cache, other), ops.kv.read(old, other)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_write_special_values(ops, dtype):
    """Zeros, ties to the even code, cuts, magnitudes at both ends, infinities and NaN in a block."""
    rows = torch.zeros(12, 1, 64)
    rows[1, 0, :8] = torch.tensor([4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5])
    rows[2] = -rows[1]
    rows[3, 0, :4] = torch.tensor([7.0, 0.5, -0.25, 1.0])        # 7 / 2^0 stays: cut to 6
    rows[4, 0, :4] = torch.tensor([7.03125, 0.5, -0.25, 1.0])    # above 7: a scale of 2
    rows[5, 0, 0] = 3e38
    rows[6, 0, :3] = torch.tensor([1.2e-38, -1e-38, 9e-41])      # at and below the smallest normal
    rows[7, 0, 1] = math.inf
    rows[8, 0, 40] = -math.inf
    rows[9, 0, 5] = math.nan
    rows[10] = 1.0
    rows[11, 0, :2] = torch.tensor([6.0, -0.0])
    if dtype == "fp16":
        rows[5, 0, :2] = torch.tensor([65504.0, -60000.0])       # a larger scale would round these to infinity
        rows[6, 0, :3] = torch.tensor([6.2e-5, -6e-8, 1.2e-7])
    x = rows.to(DTYPES[dtype]).to(DEV)
    cache = ops.kv.KVCache.empty(1, 1, page=16, head_dim=64, dtype=DTYPES[dtype], device=DEV)
    slots = torch.arange(12, dtype=torch.int32, device=DEV)
    ops.kv.write(cache, x, x, slots)
    for got in ops.kv.read(cache, slots):
        want = R.encode_ref(x.cpu()).to(x.dtype).double()
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=12345.0), torch.nan_to_num(want, nan=12345.0))
    assert bool(torch.isnan(got[7, 0, :32]).all()) and not bool(torch.isnan(got[7, 0, 32:]).any())


def test_write_nothing(ops):
    cache = ops.kv.KVCache.empty(2, 3, page=16, head_dim=128, device=DEV)
    none = torch.empty(0, 3, 128, dtype=torch.bfloat16, device=DEV)
    ops.kv.write(cache, none, none, i32([]))
    k, v = ops.kv.read(cache, i32([]))
    assert k.shape == (0, 3, 128) and not bool(cache.data.any())
    k, _ = ops.kv.read(cache, i32([-1, 5, 32, 2 ** 31 - 1]))
    assert k.shape == (4, 3, 128) and not bool(k.any())


# ---- attention -------------------------------------------------------------------------------------

def _attend_case(ops, lengths, news, hq, hk, D, page, dtype, seed=0, size=1.0, extra_columns=1):
    """Requests of `lengths` cached positions with `news` rows, scattered pages; k, v as the cache holds them."""
    g = torch.Generator().manual_seed(seed)
    t, n = DTYPES[dtype], len(lengths)
    held = [-(-x // page) for x in lengths]
    cache = ops.kv.KVCache.empty(sum(held) + 2, hk, page=page, head_dim=D, dtype=t, device=DEV)
    cache.data.fill_(255)  # what no request wrote reads as NaN
    order = torch.randperm(sum(held) + 2, generator=g).tolist()
    tables = torch.full((n, max(held) + extra_columns), -1, dtype=torch.int32)
    k = torch.zeros(n, max(max(lengths), 1), hk, D, dtype=torch.float64)
    v = torch.zeros_like(k)
    for r, x in enumerate(lengths):
        tables[r, :held[r]] = torch.tensor([order.pop() for _ in range(held[r])])
        if x:
            slots = (tables[r, :held[r], None] * page + torch.arange(page)).flatten()[:x].int().to(DEV)
            kr, vr = ((torch.randn(x, hk, D, generator=g) * size).to(t).to(DEV) for _ in range(2))
            ops.kv.write(cache, kr, vr, slots)
            kr, vr = ops.kv.read(cache, slots)
            k[r, :x], v[r, :x] = kr.cpu().double(), vr.cpu().double()
    starts = [0]
    for m in news:
        starts.append(starts[-1] + m)
    q = torch.randn(starts[-1], hq, D, generator=g).to(t)
    return cache, tables, starts, q, k, v


def _attend_check(out, lse, q, k, v, starts, visible, scale, window=0, hidden=None):
    want, wl, size = R.attend_ref(q, k, v, starts, visible, scale, window, hidden)
    u = torch.finfo(q.dtype).eps / 2
    D = q.shape[2]
    # the largest sum of the products' magnitudes of any score, and what it may move a score by
    reach = float(q.double().abs().sum(-1).max()) * float(torch.nan_to_num(k).abs().max()) * abs(scale)
    moved = 2 * (D + 3) * 2 ** -24 * reach + 2 ** -20
    tiny = torch.finfo(q.dtype).smallest_normal
    tol = u * (size + want.abs()) * (1 + 2 ** -6) + moved * size + tiny
    err = (out.cpu().double() - want).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), int((err > tol).sum()))
    if lse is not None:
        empty = wl == -math.inf
        assert torch.equal(lse.cpu()[empty].double(), wl[empty])
        off = (lse.cpu().double() - wl)[~empty].abs()
        assert bool((off <= moved + 2 ** -22 * (wl[~empty].abs() + 1)).all())


ATTEND = [  # lengths, rows, Hq, Hk, D, page, type, window
    ([1], [1], 1, 1, 128, 16, "bf16", 0),
    ([33], [1], 16, 4, 128, 16, "bf16", 0),
    ([200, 1, 31, 0, 97], [1, 1, 1, 1, 1], 8, 2, 128, 32, "bf16", 0),
    ([70, 150], [5, 3], 14, 2, 64, 16, "fp16", 0),
    ([300], [2], 8, 1, 256, 64, "bf16", 0),
    ([257, 64], [17, 40], 12, 4, 128, 64, "fp16", 0),
    ([500], [70], 4, 4, 64, 128, "bf16", 100),
    ([129, 700], [129, 90], 8, 2, 128, 16, "bf16", 37),
    ([1500, 40], [3, 1], 32, 4, 128, 128, "bf16", 0),
    ([400, 310], [200, 310], 8, 4, 128, 32, "bf16", 0),
    ([330], [150], 16, 2, 256, 16, "fp16", 64),
    ([260], [260], 2, 2, 64, 64, "bf16", 0),
]


@pytest.mark.parametrize("case", ATTEND, ids=str)
def test_attend(ops, case):
    lengths, news, hq, hk, D, page, dtype, window = case
    cache, tables, starts, q, k, v = _attend_case(ops, lengths, news, hq, hk, D, page, dtype)
    visible = [max(0, x - m + 1 + i) for x, m in zip(lengths, news) for i in range(m)]  # causal; some see nothing
    out, lse = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), window=window or None,
                             max_queries=max(news), return_lse=True)
    _attend_check(out, lse, q, k, v, starts, visible, D ** -0.5, window)
    # the bound sets the launch, not the result's meaning: too small and too large ones
    for bound in (1, None):
        again = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), window=window or None,
                              max_queries=bound)
        _attend_check(again, None, q, k, v, starts, visible, D ** -0.5, window)


@pytest.mark.parametrize("news", [[4, 3], [90, 50]], ids=str)
def test_attend_rows_of_any_limit(ops, news):
    """Limits in no order, zero, below zero and beyond the table; rows of padding; odd strides of q."""
    cache, tables, starts, q, k, v = _attend_case(ops, [100, 240], news, 4, 2, 128, 16, "bf16", extra_columns=0)
    g = torch.Generator().manual_seed(1)
    visible = [int(x) for x in torch.randint(-5, 100, (sum(news),), generator=g)]
    visible[0], visible[1] = 0, -2 ** 31
    visible[news[0]] = 240
    pad = torch.randn(3, 4, 128, generator=g).bfloat16()
    wide = torch.zeros(sum(news) + 3, 5, 131, dtype=torch.bfloat16, device=DEV)
    wide[:, :4, 1:129] = torch.cat((q, pad)).to(DEV)
    for view in (wide[:, :4, 1:129], wide[:, :4, 1:129].contiguous(), wide[:, :4, 1:129].transpose(0, 1).contiguous().transpose(0, 1)):
        out, lse = ops.kv.attend(view, cache, tables.to(DEV), i32(starts), i32(visible + [9, 9, 2 ** 31 - 1]),
                                 max_queries=max(news), return_lse=True)
        _attend_check(out[:sum(news)], lse[:sum(news)], q, k, v, starts, visible, 128 ** -0.5)
        assert not bool(out[sum(news):].any()) and bool((lse[sum(news):] == -math.inf).all())
    # a limit beyond the table sees the whole table
    out = ops.kv.attend(q.to(DEV), cache, tables[1:].to(DEV), i32([0, 1]), i32([2 ** 31 - 1] * sum(news)), max_queries=1)
    at = tables.shape[1] * 16
    assert at >= 240
    if at == 240:
        _attend_check(out[:1], None, q[:1], k[1:], v[1:], [0, 1], [240], 128 ** -0.5)


@pytest.mark.parametrize("rows", [1, 60])
def test_attend_entries_that_name_no_page(ops, rows):
    cache, tables, starts, q, k, v = _attend_case(ops, [160], [rows], 4, 1, 128, 16, "bf16")
    tables[0, 2], tables[0, 5], tables[0, 9] = -1, cache.pages, 2 ** 31 - 1
    hidden = torch.zeros(1, 160, dtype=torch.bool)
    for c in (2, 5, 9):
        hidden[0, 16 * c:16 * c + 16] = True
    for limit in (160, 48, 40):
        out, lse = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32([limit] * rows), max_queries=rows,
                                 return_lse=True)
        _attend_check(out, lse, q, k, v, starts, [limit] * rows, 128 ** -0.5, 0, hidden)
    out = ops.kv.attend(q.to(DEV), cache, tables[:, 2:3].to(DEV), i32(starts), i32([16] * rows), max_queries=rows)
    assert not bool(out.any())


@pytest.mark.parametrize("rows,D", [(4, 64), (4, 128), (4, 256), (64, 128), (64, 256), (64, 64)])
def test_attend_nan_reaches_the_rows_that_see_it(ops, rows, D):
    """A NaN block of a key makes a row that sees it NaN; of a value, its 32 dimensions; other rows, and the
    dimensions beside it, stay as they are."""
    length = 150
    cache, tables, starts, q, k, v = _attend_case(ops, [length], [rows], 2, 1, D, 32, "bf16")
    visible = [length - rows + 1 + i for i in range(rows)]
    slot = lambda p: i32([int(tables[0, p // 32]) * 32 + p % 32])  # noqa: E731
    at = length - rows // 2
    good = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), max_queries=rows)
    kr, vr = (x[0, at:at + 1].bfloat16().to(DEV) for x in (k, v))
    bad = vr.clone()
    bad[..., 33] = math.inf
    ops.kv.write(cache, kr, bad, slot(at))
    out = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), max_queries=rows)
    sees = torch.tensor([x > at for x in visible], device=DEV)
    assert torch.equal(out[~sees], good[~sees])
    assert bool(torch.isnan(out[sees][..., 32:64]).all())
    rest = torch.cat((out[sees][..., :32], out[sees][..., 64:]), -1)
    assert torch.equal(rest, torch.cat((good[sees][..., :32], good[sees][..., 64:]), -1))
    bad = kr.clone()
    bad[..., D - 1] = math.nan
    ops.kv.write(cache, bad, vr, slot(at))
    out, lse = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), max_queries=rows, return_lse=True)
    assert torch.equal(out[~sees], good[~sees]) and bool(torch.isnan(out[sees]).all()) and bool(torch.isnan(lse[sees]).all())


@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_attend_scale_and_large_scores(ops, scale, rows):
    cache, tables, starts, q, k, v = _attend_case(ops, [90], [rows], 2, 2, 64, 16, "bf16", size=4.0)
    visible = [90] * rows
    out, lse = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), scale=scale, max_queries=rows,
                             return_lse=True)
    _attend_check(out, lse, q, k, v, starts, visible, scale)


@pytest.mark.parametrize("rows", [2, 80])
def test_attend_a_row_that_is_not_finite_stays_alone(ops, rows):
    cache, tables, starts, q, k, v = _attend_case(ops, [100], [rows], 4, 2, 128, 16, "bf16")
    qd = q.to(DEV)
    good = ops.kv.attend(qd, cache, tables.to(DEV), i32(starts), i32([100] * rows), max_queries=rows)
    qd[1, 2] = math.nan
    qd[0, 0, 5] = math.inf
    out = ops.kv.attend(qd, cache, tables.to(DEV), i32(starts), i32([100] * rows), max_queries=rows)
    bad = torch.zeros(rows, 4, dtype=torch.bool, device=DEV)
    bad[1, 2] = bad[0, 0] = True
    assert bool(torch.isnan(out[1, 2]).all()) and bool(torch.isnan(out[0, 0]).any()) and torch.equal(out[~bad], good[~bad])


def test_attend_nothing(ops):
    cache = ops.kv.KVCache.empty(2, 2, page=16, head_dim=128, device=DEV)
    q = torch.randn(3, 4, 128, device=DEV).bfloat16()
    none = torch.empty(0, 4, 128, dtype=torch.bfloat16, device=DEV)
    assert ops.kv.attend(none, cache, i32([[0]]), i32([0, 0]), i32([])).shape == (0, 4, 128)
    out, lse = ops.kv.attend(q, cache, torch.zeros(0, 4, dtype=torch.int32, device=DEV), i32([0]), i32([5, 5, 5]), return_lse=True)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    out = ops.kv.attend(q, cache, torch.zeros(1, 0, dtype=torch.int32, device=DEV), i32([0, 3]), i32([5, 5, 5]))
    assert not bool(out.any())
    empty = ops.kv.KVCache(torch.zeros(0, 2, 16 * 136, dtype=torch.uint8, device=DEV), page=16, head_dim=128)
    assert not bool(ops.kv.attend(q, empty, i32([[0]]), i32([0, 3]), i32([5, 5, 5])).any())


def test_starts_out_of_range_are_clamped(ops):
    cache, tables, starts, q, k, v = _attend_case(ops, [50, 50], [2, 2], 2, 1, 64, 16, "bf16")
    out = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32([-3, 2, 900]), i32([50] * 4), max_queries=2)
    _attend_check(out, None, q, k, v, [0, 2, 4], [50] * 4, 64 ** -0.5)


def test_a_cache_beyond_32_bits(ops):
    """Pages whose bytes lie beyond 2^32: written, read and attended to at the cache's end."""
    pages, heads, page, D = 80000, 8, 64, 128
    data = torch.empty(pages, heads, page * 136, dtype=torch.uint8, device=DEV)
    assert data.numel() > 2 ** 32
    cache = ops.kv.KVCache(data, page=page, head_dim=D)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32)
    slots = (table.T * page + torch.arange(page)).flatten()[:170].int().to(DEV)
    x = torch.randn(170, 2 * heads, D, generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    ops.kv.write(cache, x[:, :heads], x[:, heads:], slots)
    k, v = ops.kv.read(cache, slots)
    for got, want in ((k, x[:, :heads]), (v, x[:, heads:])):
        assert torch.equal(got.cpu().double(), R.encode_ref(want.cpu()))
    for rows in (1, 40):
        q = torch.randn(rows, 16, D, generator=torch.Generator().manual_seed(6)).bfloat16()
        visible = [170 - rows + 1 + i for i in range(rows)]
        out = ops.kv.attend(q.to(DEV), cache, table.to(DEV), i32([0, rows]), i32(visible), max_queries=rows)
        _attend_check(out, None, q, k.cpu()[None], v.cpu()[None], [0, rows], visible, D ** -0.5)


# ---- streams and graphs ----------------------------------------------------------------------------

def _serving_step(ops, s):
    step = ops.kv.step_pages(s["cached"], s["new"], s["tables"], s["free"], s["count"], page=16, tokens=s["q"].shape[0])
    q, k = ops.rotary.rotate(s["q"], s["k"], step.positions, s["plan"])
    ops.kv.write(s["cache"], k, s["v"], step.slots)
    return ops.kv.attend(q, s["cache"], s["tables"], step.starts, step.visible, max_queries=s["most"], return_lse=True)


def _serving_state(ops, seed, most):
    g = torch.Generator().manual_seed(seed)
    n, heads, D = 6, 2, 128
    cached = torch.randint(0, 90, (n,), generator=g).int()
    new = torch.randint(1, most + 1, (n,), generator=g).int()
    tables = torch.full((n, 12), -1, dtype=torch.int32)
    ids = torch.randperm(80, generator=g).int().tolist()
    for r in range(n):
        for c in range(-(-int(cached[r]) // 16)):
            tables[r, c] = ids.pop()
    cache = ops.kv.KVCache.empty(80, heads, page=16, head_dim=D, device=DEV)
    past = torch.randn(1280, 2 * heads, D, generator=g).bfloat16().to(DEV)
    ops.kv.write(cache, past[:, :heads], past[:, heads:], torch.arange(1280, dtype=torch.int32, device=DEV))
    x = torch.randn(int(new.sum()) + 3, 8, D, generator=g).bfloat16().to(DEV)
    return dict(cached=cached.to(DEV), new=new.to(DEV), tables=tables.to(DEV), free=i32(ids), count=i32([len(ids)]), cache=cache,
                q=x[:, :4], k=x[:, 4:6], v=x[:, 6:], plan=ops.rotary.plan(D, device=DEV), most=most)


@pytest.mark.parametrize("most", [1, 30])
def test_a_step_on_another_stream_and_in_a_graph(ops, most):
    s, other = _serving_state(ops, 1, most), _serving_state(ops, 2, most)
    want = [x.clone() for x in _serving_step(ops, s)]
    assert bool(torch.isfinite(want[0].float()).all()) and float(want[0].float().abs().max()) > 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _serving_step(ops, s)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = _serving_step(ops, s)
    for replay in range(4):
        for x in held:
            x.fill_(7)
        _serving_step(ops, other)  # eager work of other inputs between the replays
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), replay


def test_results_do_not_depend_on_timing(ops):
    s = _serving_state(ops, 3, 30)
    first = [x.clone() for x in _serving_step(ops, s)]
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(_serving_step(ops, s), first))
