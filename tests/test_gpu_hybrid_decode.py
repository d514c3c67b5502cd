"""A decode step of a GDN layer and an attention layer together, with a content token and a read-only query a
sequence: the query's rows see what the step has written and are not written themselves."""

import pytest
import torch

from test_gpu_attention import DEV, _attend_case, _attend_check, i32, ops  # noqa: F401

pytestmark = pytest.mark.gpu

N, H, K, W, HEADS, KV, D, PAGE, COLUMNS = 5, 4, 4, 256, 8, 2, 64, 16, 9


def _layers(g):
    S = H * 128
    m = lambda *s: (torch.randn(*s, generator=g) * s[0] ** -0.5).bfloat16().to(DEV)  # noqa: E731
    return dict(gdn=m(W, 4 * S + 2 * H), conv=(torch.rand(3 * S, K, generator=g) - 0.5).bfloat16().to(DEV),
                A=torch.rand(H, generator=g).add(0.1).log().to(DEV), dt=torch.randn(H, generator=g).to(DEV) * 0.5,
                norm=1 + 0.1 * torch.randn(128, generator=g).to(DEV), gdn_out=m(S, W),
                qkv=m(W, (HEADS + 2 * KV) * D), out=m(HEADS * D, W))


def _state(ops, g):
    S, cached = H * 128, torch.randint(0, 100, (N,), generator=g).int()
    pages = N * COLUMNS
    ids = torch.randperm(pages, generator=g).int().tolist()
    tables = torch.full((N, COLUMNS), -1, dtype=torch.int32)
    for r in range(N):
        for c in range(-(-int(cached[r]) // PAGE)):
            tables[r, c] = ids.pop()
    cache = ops.kv.KVCache.empty(pages, KV, page=PAGE, head_dim=D, device=DEV)
    past = torch.randn(pages * PAGE, 2 * KV, D, generator=g).bfloat16().to(DEV)
    ops.kv.write(cache, past[:, :KV], past[:, KV:], torch.arange(pages * PAGE, dtype=torch.int32, device=DEV))
    return dict(x=torch.randn(N, 2, W, generator=g).bfloat16().to(DEV), data=cache.data,
                conv=torch.randn(N, K - 1, 3 * S, generator=g).bfloat16().to(DEV),
                state=torch.randn(N, H, 128, 128, generator=g).to(DEV) * 0.05, cached=cached.to(DEV), tables=tables.to(DEV),
                free=i32(ids + [0] * (pages - len(ids))), count=i32([len(ids)]))


def _step(ops, w, s, plan, one):
    """x [N, 2, W]: content token and query of each sequence; the next step's in its place."""
    from cqgdn import events

    x = s["x"]
    y = events.layer_decode_step(x @ w["gdn"], w["conv"], w["A"], w["dt"], w["norm"], dict(conv=s["conv"], state=s["state"]),
                                 heads=H)
    x = x + y @ w["gdn_out"]
    step = ops.kv.step_pages(s["cached"], one, s["tables"], s["free"], s["count"], page=PAGE, tokens=N, in_place=True)
    cache = ops.kv.KVCache(s["data"], page=PAGE, head_dim=D)
    rows = (x @ w["qkv"]).unflatten(2, (-1, D))  # [N, 2, heads, D]
    content, query = rows[:, 0], rows[:, 1]
    q, k = ops.rotary.rotate(content[:, :HEADS], content[:, HEADS:HEADS + KV], step.positions, plan)
    ops.kv.write(cache, k, content[:, HEADS + KV:], step.slots)
    a = ops.kv.attend(q, cache, s["tables"], step.starts, step.visible, max_queries=1)
    # the query stands behind its token and sees the whole request: a call of its own, a row a request
    q, _ = ops.rotary.rotate(query[:, :HEADS], query[:, :0], step.lengths, plan)
    b = ops.kv.attend(q, cache, s["tables"], s["each"], step.lengths, max_queries=1)
    x = x + torch.stack((a, b), 1).flatten(2) @ w["out"]
    s["x"].copy_(x / x.float().square().mean(-1, keepdim=True).sqrt().bfloat16())


def test_a_hybrid_step_in_a_graph(ops):
    """Steps replayed from a HIP graph, the program's own eager steps between them, give what the same steps give
    run eagerly from the same start."""
    g = torch.Generator().manual_seed(1)
    w, plan, one = _layers(g), ops.rotary.plan(D, device=DEV), torch.ones(N, dtype=torch.int32, device=DEV)
    start = _state(ops, g)
    start["each"] = torch.arange(N + 1, dtype=torch.int32, device=DEV)
    copy = lambda s: {n: x.clone() for n, x in s.items()}  # noqa: E731
    eager, want = copy(start), []
    for _ in range(4):
        _step(ops, w, eager, plan, one)
        want.append(eager["x"].clone())
    assert bool(torch.isfinite(want[-1].float()).all()) and not torch.equal(want[0], want[1])
    s, other = copy(start), copy(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(ops, w, other, plan, one)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _step(ops, w, s, plan, one)
    for x in want:
        _step(ops, w, other, plan, one)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(s["x"], x)
    for name in ("data", "conv", "state", "cached", "tables", "free", "count"):
        assert torch.equal(s[name], eager[name]), name
    assert s["cached"].tolist() == [c + 4 for c in start["cached"].tolist()]


@pytest.mark.parametrize("queries", [1, 3])
def test_query_rows_beside_content_rows(ops, queries):
    """Read-only rows in a call of their own, and in one call with the content rows (starts and limits made by hand):
    both against the plain form."""
    lengths = [130, 1, 77, 600]
    n = len(lengths)
    cache, tables, starts, q, k, v = _attend_case(ops, lengths, [1 + queries] * n, 8, 2, 128, 16, "bf16", seed=queries)
    visible = [x for x in lengths for _ in range(1 + queries)]
    out, lse = ops.kv.attend(q.to(DEV), cache, tables.to(DEV), i32(starts), i32(visible), max_queries=1 + queries,
                             return_lse=True)
    _attend_check(out, lse, q, k, v, starts, visible, 128 ** -0.5)
    alone = q.view(n, 1 + queries, 8, 128)[:, 1:].reshape(-1, 8, 128)
    each = torch.arange(n + 1, dtype=torch.int32, device=DEV) * queries
    out, lse = ops.kv.attend(alone.to(DEV), cache, tables.to(DEV), each, i32(lengths).repeat_interleave(queries),
                             max_queries=queries, return_lse=True)
    _attend_check(out, lse, alone, k, v, each.tolist(), [x for x in lengths for _ in range(queries)], 128 ** -0.5)
