"""Attention over packed rows and its gradients on the GPU against plain 64-bit forms (core_testlib has the tolerances)."""

import math

import pytest
import torch

import core_testlib as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def attention(gdn):
    from cqgdn import attention

    return attention


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make(T, S, hq, hk, D, dtype, seed=0, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda n, h: (torch.randn(n, h, D, generator=g, device=DEV) * size).to(DTYPES[dtype])  # noqa: E731
    return r(T, hq), r(S, hk), r(S, hk), r(T, hq)


def run(attention, q, k, v, limit, dy, dlse=None, **kw):
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out, lse = attention.attend(q, k, v, limit, return_lse=True, **kw)
    outs, grads = ((out,), (dy,)) if dlse is None else ((out, lse), (dy, dlse))
    dq, dk, dv = torch.autograd.grad(outs, (q, k, v), grads)
    return dict(out=out.detach(), lse=lse.detach(), dq=dq, dk=dk, dv=dv)


def compare(got, q, k, v, first, limit, dy, dlse=None, **kw):
    first = torch.zeros_like(limit) if first is None else first
    kw.setdefault("scale", q.shape[2] ** -0.5)
    want, tol = R.attend_ref(q, k, v, first, limit, dy=dy, dlse=dlse, **kw)
    for name in got:
        R.check(got[name], want[name], tol[name], name, q.dtype)


CASES = [  # document lengths, queries behind each, Hq, Hk, D, type, window, prefix, cap, slopes
    ([1], 0, 1, 1, 64, "bf16", None, False, None, False),
    ([2, 1, 3], 0, 4, 2, 128, "fp16", None, False, None, False),
    ([33], 5, 4, 1, 128, "bf16", None, False, None, False),
    ([64], 0, 2, 2, 256, "bf16", None, False, None, False),
    ([65, 127, 1, 200], 0, 8, 2, 128, "bf16", None, False, None, False),
    ([300], 64, 4, 4, 64, "fp16", None, False, 3.0, False),
    ([129, 260], 0, 7, 1, 64, "bf16", 50, False, None, True),
    ([129, 260], 3, 14, 2, 128, "bf16", None, True, 20.0, True),
    ([257, 31, 90], 0, 6, 3, 256, "fp16", None, True, None, True),
    ([400], 17, 8, 4, 256, "bf16", 100, False, 5.0, False),
    ([640, 500], 0, 4, 4, 128, "fp16", None, False, None, False),
    ([1000], 0, 3, 1, 128, "bf16", None, True, None, False),
    ([700], 300, 2, 1, 64, "bf16", None, False, None, False),
]


def ranges(docs, queries, window, prefix):
    """first, limit and position of every row: a document's tokens, then its queries, which see a part each."""
    at, rows = 0, []
    for n in docs:
        p = n // 2 if prefix else 0
        rows += [(at + (max(0, i + 1 - window) if window else 0), at + max(i + 1, p), at + i) for i in range(n)]
        for i in range(queries):
            seen = n * (i + 1) // queries
            rows.append((at + (max(0, seen - window) if window else 0), at + seen, at + max(seen - 1, 0)))
        at += n
    return (i32(list(x)) for x in zip(*rows))


@pytest.mark.parametrize("case", CASES, ids=str)
def test_attend_and_its_gradients(attention, case):
    docs, queries, hq, hk, D, dtype, window, prefix, cap, bias = case
    first, limit, position = ranges(docs, queries, window, prefix)
    q, k, v, dy = make(len(limit), sum(docs), hq, hk, D, dtype, seed=len(limit), size=1.5)
    slopes = torch.tensor([2.0 ** (-1 - i) for i in range(hq)], device=DEV) if bias else None
    kw = dict(cap=cap, slopes=slopes, positions=position if bias and prefix else None)
    got = run(attention, q, k, v, limit, dy, first=first, **kw)
    compare(got, q, k, v, first, limit, dy, **kw)
    # without gradients, and without what is not asked for: the same bits
    with torch.no_grad():
        assert torch.equal(attention.attend(q, k, v, limit, first=first, **kw), got["out"])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bent", [False, True])
def test_rows_of_any_range(attention, D, bent):
    """Ranges in no order, empty ones, below 0 and beyond the keys; rows in groups that see nothing at all."""
    T, S = 203, 171
    q, k, v, dy = make(T, S, 6, 2, D, "bf16", seed=3)
    g = torch.Generator().manual_seed(9)
    first, limit = (torch.randint(-20, S + 30, (T,), generator=g) for _ in range(2))
    first[40:90], limit[40:90] = 30, 20
    first[100], limit[100] = -2 ** 31, 2 ** 31 - 1
    first[101], limit[101] = 2 ** 31 - 1, -2 ** 31
    first[102], limit[102] = S, S + 5
    first, limit = first.int().to(DEV), limit.int().to(DEV)
    slopes = torch.tensor([0.5, 0.25, 0.0, 0.125, 1.0, -0.01], device=DEV) if bent else None
    where = torch.randint(-50, S + 50, (T,), generator=g).int().to(DEV) if bent else None
    kw = dict(slopes=slopes, positions=where, cap=7.0 if bent else None)
    got = run(attention, q, k, v, limit, dy, first=first, **kw)
    compare(got, q, k, v, first, limit, dy, **kw)
    none = (first.clamp(min=0) >= limit.clamp(max=S))
    assert bool(none[40:90].all()) and not bool(got["out"][none].any()) and not bool(got["dq"][none].any())
    assert bool((got["lse"][none] == -math.inf).all())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_keys_that_no_row_sees_and_rows_in_many_blocks(attention, D):
    """More rows than 64 blocks of 32, few of which see the keys at hand; keys before, between and behind what is seen."""
    T, S = 1500, 900
    q, k, v, dy = make(T, S, 4, 2, D, "bf16", seed=4)
    t = torch.arange(T, device=DEV)
    first, limit = (100 + t // 300 * 150).int(), (100 + t // 300 * 150 + 1 + t % 140).int()
    got = run(attention, q, k, v, limit, dy, first=first)
    compare(got, q, k, v, first, limit, dy)
    assert not bool(got["dk"][:100].any()) and not bool(got["dv"][840:].any()) and bool(got["dv"][100:240].any())


def test_sizes_of_nothing(attention):
    for T, S in ((0, 5), (5, 0), (0, 0)):
        q, k, v, dy = make(T, S, 4, 2, 128, "bf16")
        got = run(attention, q, k, v, i32([3] * T), dy)
        assert got["out"].shape == q.shape and got["dk"].shape == k.shape
        assert not any(bool(got[n].any()) for n in ("out", "dq", "dk", "dv")) and bool((got["lse"] == -math.inf).all())


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("cap", [None, 4.0])
def test_scale_and_large_scores(attention, scale, cap):
    q, k, v, dy = make(150, 150, 2, 2, 64, "bf16", seed=5, size=4.0)
    limit = torch.arange(1, 151, dtype=torch.int32, device=DEV)
    got = run(attention, q, k, v, limit, dy, scale=scale, cap=cap)
    compare(got, q, k, v, None, limit, dy, scale=scale, cap=cap)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 9])
def test_small_and_large_gradients(attention, dtype, size):
    """Gradients near the ends of fp16, over rows long enough for small weights."""
    q, k, v, dy = make(600, 600, 2, 1, 64, dtype, seed=6)
    q = q / 4
    dy = (dy.float() * size).to(dy.dtype)
    limit = torch.arange(1, 601, dtype=torch.int32, device=DEV)
    got = run(attention, q, k, v, limit, dy)
    compare(got, q, k, v, None, limit, dy)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_gradient_through_the_logarithms(attention, D):
    q, k, v, dy = make(100, 90, 4, 2, D, "bf16", seed=7)
    limit = torch.randint(0, 95, (100,), generator=torch.Generator().manual_seed(1)).int().to(DEV)
    dlse = torch.randn(100, 4, generator=torch.Generator().manual_seed(2)).to(DEV)
    got = run(attention, q, k, v, limit, dy, dlse)
    compare(got, q, k, v, None, limit, dy, dlse)
    # through them alone
    a = q.detach().requires_grad_()
    _, lse = attention.attend(a, k, v, limit, return_lse=True)
    dq, = torch.autograd.grad(torch.where(lse == -math.inf, 0.0, lse).sum(), a)
    want, tol = R.attend_ref(q, k, v, torch.zeros_like(limit), limit, scale=D ** -0.5, dy=torch.zeros_like(q),
                             dlse=torch.ones_like(dlse))
    R.check(dq, want["dq"], tol["dq"], "dq", q.dtype)


def test_gradient_against_differences(attention):
    """The directional derivative of the float64 form by central differences.  With steps of h in each input (+-1 each) the
    difference is off by h^2 / 6 of the third derivative, below 2^3 of the gradient's norm over these scores (below 5, the
    cap), and the kernel's by some 4 roundings a value, of random signs."""
    q, k, v, dy = make(120, 120, 4, 2, 64, "fp16", seed=8)
    limit = torch.arange(1, 121, dtype=torch.int32, device=DEV)
    kw = dict(cap=5.0, slopes=torch.tensor([0.1, 0.2, 0.05, 0.0], device=DEV))
    got = run(attention, q, k, v, limit, dy, **kw)
    u, h = torch.finfo(torch.float16).eps / 2, 2.0 ** -10
    for i, name in enumerate(("dq", "dk", "dv")):
        step = torch.where(torch.rand(got[name].shape, generator=torch.Generator().manual_seed(i)) < 0.5, -1.0, 1.0).double().to(DEV)

        def loss(s):
            x = [q.double(), k.double(), v.double()]
            x[i] = x[i] + s * h * step
            return float((R.attend_ref(*x, torch.zeros_like(limit), limit, scale=64 ** -0.5, **kw)[0]["out"] * dy.double()).sum())

        difference, mine = (loss(1) - loss(-1)) / (2 * h), float((got[name].double() * step).sum())
        norm = float(got[name].double().square().sum().sqrt())
        assert abs(difference - mine) <= 4 * (4 * u + 8 * h * h) * norm * 4, (name, difference, mine, norm)


def test_rows_of_other_strides(attention):
    """Columns of a fused projection, transposed heads, odd rows that are copied, broadcast keys and gradients."""
    T, hq, hk, D = 140, 4, 2, 128
    g = torch.Generator(device=DEV).manual_seed(1)
    rows = torch.randn(T, hq + 2 * hk, D, generator=g, device=DEV).bfloat16()
    limit = torch.arange(1, T + 1, dtype=torch.int32, device=DEV)
    dy = torch.randn(1, hq, 1, generator=g, device=DEV).bfloat16().expand(T, hq, D)
    q, k, v = rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:]
    want = run(attention, q.contiguous(), k.contiguous(), v.contiguous(), limit, dy.contiguous())
    compare(want, q, k, v, None, limit, dy)
    wide = torch.zeros(T, hq + 2 * hk, D + 3, dtype=rows.dtype, device=DEV)
    wide[..., 1:-2] = rows
    turned = rows.transpose(0, 1).contiguous().transpose(0, 1)
    for x in (rows, wide[..., 1:-2], turned):
        got = run(attention, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], limit, dy)
        assert all(torch.equal(got[n], want[n]) for n in want)
    flipped = run(attention, q, k, v, torch.stack((limit, limit), 1)[:, 0], dy)  # a strided limit
    assert all(torch.equal(flipped[n], want[n]) for n in want)
    one = k[:1].expand(T, hk, D)  # every key the same row
    compare(run(attention, q, one, v, limit, dy), q, one, v, None, limit, dy)
    # [1, T, H, D], as the GDN operators take it
    out, lse = attention.attend(q[None], k[None], v[None], limit, return_lse=True)
    assert torch.equal(out[0], want["out"]) and torch.equal(lse[0], want["lse"])


def test_gradients_of_some_inputs(attention):
    q, k, v, dy = make(70, 70, 2, 1, 64, "bf16", seed=2)
    limit = torch.arange(1, 71, dtype=torch.int32, device=DEV)
    want = run(attention, q, k, v, limit, dy)
    for names in ("q", "k", "v", "qv", "kv"):
        x = dict(q=q, k=k, v=v)
        x = {n: t.detach().requires_grad_(n in names) for n, t in x.items()}
        out = attention.attend(x["q"], x["k"], x["v"], limit)
        for n, grad in zip(names, torch.autograd.grad(out, [x[n] for n in names], dy)):
            assert torch.equal(grad, want["d" + n])
    # shared leaves: the gradient is the sum
    a = k.detach().requires_grad_()
    g, = torch.autograd.grad(attention.attend(q, a, a, limit), a, dy)
    both = run(attention, q, k, k, limit, dy)
    assert torch.equal(g, both["dk"] + both["dv"])


def test_documents_is_what_its_words_say(attention):
    first, limit = attention.documents([0, 5, 5, 9], device=DEV)
    assert first.tolist() == [0] * 5 + [5] * 4 and limit.tolist() == list(range(1, 10))
    first, limit = attention.documents([0, 5, 9], window=2, prefix=(3, 7), device=DEV)
    assert first.tolist() == [0, 0, 1, 2, 3, 5, 5, 6, 7] and limit.tolist() == [3, 3, 3, 4, 5, 9, 9, 9, 9]
    _, limit = attention.documents([0, 5, 9], causal=False, device=DEV)
    assert limit.tolist() == [5] * 5 + [9] * 4


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite_reach_only_who_sees_them(attention, D, bad):
    """Two documents in one tile, the second with a bad key, value, query or gradient in its middle, and padding of
    NaN: the first document's results, and the second's rows before the bad one, are the same bits as without."""
    docs, at = [70, 90], 110
    first, limit = attention.documents([0, 70, 160], device=DEV)
    first, limit = (torch.cat((x, i32([0] * 9))) for x in (first, limit))  # rows of padding see nothing
    q, k, v, dy = make(169, 169, 4, 2, D, "bf16", seed=11)
    good = run(attention, q, k, v, limit, dy, first=first)
    for x in (q, k, v, dy):
        x[sum(docs):] = bad
    got = run(attention, q, k, v, limit, dy, first=first)
    assert all(torch.equal(got[n], good[n]) for n in got), "padding reaches nobody"
    sees = (torch.arange(169, device=DEV) >= at) & (torch.arange(169, device=DEV) < 160)
    own = (torch.arange(169, device=DEV) >= 70) & (torch.arange(169, device=DEV) < 160)
    before = ~own
    for name in ("k", "v", "q", "dy"):
        x = dict(q=q.clone(), k=k.clone(), v=v.clone(), dy=dy.clone())
        x[name][at, :, 5] = bad
        got = run(attention, x["q"], x["k"], x["v"], limit, x["dy"], first=first)
        for n in ("dk", "dv", "dq", "out", "lse"):
            assert torch.equal(got[n][before], good[n][before]), (name, n)
        if name in "kv":
            assert torch.equal(got["out"][~sees], good["out"][~sees]) and torch.equal(got["dq"][~sees], good["dq"][~sees])
        else:  # a row's own: other rows keep their results, keys behind it their gradients
            other = torch.arange(169, device=DEV) != at
            assert torch.equal(got["out"][other], good["out"][other]) and torch.equal(got["dq"][other], good["dq"][other])
            behind = torch.arange(169, device=DEV) > at
            assert torch.equal(got["dk"][behind], good["dk"][behind]) and torch.equal(got["dv"][behind], good["dv"][behind])
        if name == "v":
            out = got["out"][sees].float()
            assert not bool(torch.isfinite(out[..., 5]).any())
            keep = [d for d in range(D) if d != 5]
            assert torch.equal(got["out"][sees][..., keep], good["out"][sees][..., keep])
        if name == "dy":
            assert not bool(torch.isfinite(got["dv"][70:at + 1, :, 5].float()).any())
        if name == "k" and bad != bad:
            assert bool(torch.isnan(got["out"][sees]).all()) and bool(torch.isnan(got["lse"][sees]).all())


def test_same_inputs_same_bits(attention):
    first, limit, _ = ranges([900, 340], 40, None, False)
    q, k, v, dy = make(len(limit), 1240, 8, 2, 128, "bf16", seed=12)
    want = run(attention, q, k, v, limit, dy, first=first)
    for _ in range(5):
        got = run(attention, q, k, v, limit, dy, first=first)
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_offsets_beyond_32_bits(attention):
    """More than 2^31 values of q, and of k and v, in windows of 16: the last rows and keys against the form for those alone
    (rows and keys whose windows lie within the last 100)."""
    T, hq, D, n, w = 70000, 256, 128, 100, 16
    assert T * hq * D > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(21)
    q, k, v, dy = (torch.randn(T, hq, D, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(4))
    row = torch.arange(T, device=DEV)
    first, limit = (row + 1 - w).clamp(min=0).int(), (row + 1).int()
    got = run(attention, q, k, v, limit, dy, first=first)
    for heads in (slice(0, 2), slice(hq - 2, hq)):
        part = [x[T - n:, heads] for x in (q, k, v)]
        want, tol = R.attend_ref(*part, first[T - n:] - (T - n), limit[T - n:] - (T - n), scale=D ** -0.5, dy=dy[T - n:, heads])
        for x in want:
            R.check(got[x][T - n + w:, heads], want[x][w:], tol[x][w:], x, q.dtype)


def test_another_stream_and_a_graph(attention):
    first, limit, _ = ranges([500, 77], 13, None, True)
    q, k, v, dy = make(len(limit), 577, 8, 2, 128, "bf16", seed=13)
    other = make(len(limit), 577, 8, 2, 128, "bf16", seed=14)
    kw = dict(first=first, cap=9.0)
    want = run(attention, q, k, v, limit, dy, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(attention, q, k, v, limit, dy, **kw)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = run(attention, q, k, v, limit, dy, **kw)
    for replay in range(4):
        for x in held.values():
            x.fill_(7)
        run(attention, *other[:3], limit, other[3], **kw)  # eager work of other inputs between the replays
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(held[n], want[n]) for n in want), replay


def test_derivatives_that_are_refused(attention):
    q, k, v, dy = make(20, 20, 2, 1, 64, "bf16")
    limit = torch.arange(1, 21, dtype=torch.int32, device=DEV)
    a = q.detach().requires_grad_()
    out = attention.attend(a, k, v, limit)
    with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad(out, a, dy, create_graph=True)
    slopes = torch.ones(2, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="constants"):
        attention.attend(a, k, v, limit, slopes=slopes)
    with torch.no_grad():
        attention.attend(q, k, v, limit, slopes=slopes)
    from torch.autograd import forward_ad

    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        attention.attend(forward_ad.make_dual(q, dy), k, v, limit)
    # a tensor of the forward pass that was written to since
    b = k.clone()
    out = attention.attend(a, b, v, limit)
    b.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, a, dy)


@pytest.mark.parametrize("D", [64, 256])
def test_rows_that_stand_far_away(attention, D):
    """Positions of any size: beyond 2^24 they count as that."""
    T, S = 150, 130
    q, k, v, dy = make(T, S, 2, 1, D, "bf16", seed=22)
    limit = torch.randint(1, S + 1, (T,), generator=torch.Generator().manual_seed(4)).int().to(DEV)
    where = torch.arange(T, device=DEV).int()
    where[::3], where[1::7], where[2::11], where[5::13] = 2 ** 31 - 1, -2 ** 31, 2 ** 24 - 3, -2 ** 24 + 1
    slopes = torch.tensor([2.0 ** -18, -2.0 ** -21], device=DEV)
    got = run(attention, q, k, v, limit, dy, slopes=slopes, positions=where)
    compare(got, q, k, v, None, limit, dy, slopes=slopes, positions=where.clamp(-2 ** 24, 2 ** 24))


@pytest.mark.parametrize("adjacent", [False, True])
def test_a_layer_with_rotary_positions(attention, adjacent):
    """Rows turned, attended, and turned back in the backward pass: what the operators give one after the other, bit for bit,
    and the attention's part against the plain form."""
    from cqgdn import rotary

    bounds = [0, 70, 71, 200]
    first, limit = attention.documents(bounds, prefix=[10, 0, 40], device=DEV)
    T, hq, hk, D = 200, 8, 2, 128
    q, k, v, dy = make(T, T, hq, hk, D, "bf16", seed=23)
    plan = rotary.plan(64, theta=1e5, adjacent=adjacent, device=DEV)
    positions = torch.cat([torch.arange(b - a) for a, b in zip(bounds, bounds[1:])]).int().to(DEV)
    a, b, c = (x.clone().requires_grad_() for x in (q, k, v))
    out = attention.attend(*rotary.rotate(a, b, positions, plan), c, limit, first=first, cap=30.0)
    grads = torch.autograd.grad(out, (a, b, c), dy)
    x, y = q.clone().requires_grad_(), k.clone().requires_grad_()
    turned = rotary.rotate(x, y, positions, plan)
    part = run(attention, turned[0], turned[1], v, limit, dy, first=first, cap=30.0)
    compare(part, turned[0].detach(), turned[1].detach(), v, first, limit, dy, cap=30.0)
    dq, dk = torch.autograd.grad(turned, (x, y), (part["dq"], part["dk"]))
    assert torch.equal(out, part["out"])
    assert torch.equal(grads[0], dq) and torch.equal(grads[1], dk) and torch.equal(grads[2], part["dv"])


def test_two_calls_at_once(attention):
    """Calls on two streams that wait for nothing of each other's, in many parts each."""
    args = []
    for seed in (24, 25):
        first, limit, _ = ranges([700, 90], 0, None, False)
        args.append((make(len(limit), 790, 4, 2, 64, "fp16", seed=seed), first, limit))
    want = [run(attention, *x[:3], limit, x[3], first=first) for x, first, limit in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, (stream, (x, first, limit)) in enumerate(zip(streams, args)):
            with torch.cuda.stream(stream):
                got[i].append(run(attention, *x[:3], limit, x[3], first=first))
    torch.cuda.synchronize()
    for w, all_of in zip(want, got):
        assert all(torch.equal(g[n], w[n]) for g in all_of for n in w)


def test_a_leaf_in_every_place(attention):
    """Queries, keys and values are one tensor: its gradient is the sum of the three."""
    x, _, _, dy = make(200, 200, 2, 2, 64, "bf16", seed=26)
    limit = torch.arange(1, 201, dtype=torch.int32, device=DEV)
    parts = run(attention, x, x, x, limit, dy)
    compare(parts, x, x, x, None, limit, dy)
    leaf = x.clone().requires_grad_()
    attention.attend(leaf, leaf, leaf, limit).backward(dy)
    total = sum(parts[n].double() for n in ("dq", "dk", "dv"))
    # two sums in bf16, each rounded, of values no larger than the three magnitudes
    size = sum(parts[n].double().abs() for n in ("dq", "dk", "dv"))
    assert bool(((leaf.grad.double() - total).abs() <= 2 * 2 ** -8 * (1 + 2 ** -8) * size).all())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_rows_of_one_key_move_no_score(attention, dtype, D):
    """The weight of a row's only key is 1 whatever its score: the gradients of q and k are 0, or the gradient of the
    logarithm's alone.  Values that are not finite still show."""
    T = 90
    q, k, v, dy = make(T, T, 4, 2, D, dtype, seed=27)
    first = torch.arange(T, dtype=torch.int32, device=DEV)
    got = run(attention, q, k, v, first + 1, dy, first=first, cap=20.0)
    assert not bool(got["dq"].any()) and not bool(got["dk"].any()) and torch.equal(got["out"][:, ::2], v)
    compare(got, q, k, v, first, first + 1, dy, cap=20.0)
    dlse = torch.randn(T, 4, device=DEV)
    compare(run(attention, q, k, v, first + 1, dy, dlse, first=first), q, k, v, first, first + 1, dy, dlse)
    dy[7, 1, 3] = math.inf
    got = run(attention, q, k, v, first + 1, dy, first=first)
    assert bool(got["dq"][7, 1].isnan().all()) and bool(got["dk"][7, 0].isnan().all())
    assert not bool(got["dq"][:7].any()) and not bool(got["dk"][8:].any()) and bool(got["dv"][8:].isfinite().all())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cap", [None, 20.0])
def test_rows_of_few_keys_are_held_in_two_terms(attention, D, cap):
    """Causal rows of 63 tokens, every step of which the mask cuts: no score's gradient is rounded to one bf16 term."""
    docs = [63, 5, 2, 40]
    first, limit, _ = ranges(docs, 0, None, False)
    q, k, v, dy = make(sum(docs), sum(docs), 4, 2, D, "bf16", seed=28, size=1.5)
    got = run(attention, q, k, v, limit, dy, first=first, cap=cap)
    compare({n: got[n] for n in ("dq", "dk")}, q, k, v, first, limit, dy, cap=cap, terms=2)
