"""The operators that the attention layers of a hybrid stack are trained with, and a 16-bit cache for serving them.

Beside the GDN layers, which have their forward and backward passes, a stack's attention layers take:

* ``attend``  attention over packed documents, forward and backward.  Row t sees the keys first[t] .. limit[t] - 1,
              which covers documents, causal rows, windows, prefixes that see each other and read-only query rows;
              scores may be capped (cap tanh(x / cap)) and get a bias that grows with the distance, a slope a head;
* ``append``  the queries and keys of new tokens turned by their positions, and keys and values put into the
              pages of a 16-bit cache on the way;
* ``cached``  attention of new rows over those pages, one token or many a request, with the cap and the bias that
              the model was trained with.

``run`` computes each in its plain form (elementary torch operations, 32 bits, rounded once at the end) or, with
``own``, through the framework's entry points.  ``exact`` restates each in float64.
"""

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False  # True: run() calls the framework's operators

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # a short document with read-only queries behind its content: a debugging run, or the tail of a microbatch
        dict(name="train_short", kind="attend", documents=1, tokens=253, queries=64, ragged=False, heads=16, kv_heads=4,
             head_dim=128, mask="causal", window=0, cap=0.0, slopes=False, dtype="bf16", padding=0, backward=True),
        # 2048 content tokens and 256 read-only queries, a training step's short form
        dict(name="train_2304", kind="attend", documents=1, tokens=2048, queries=256, ragged=False, heads=16, kv_heads=4,
             head_dim=128, mask="causal", window=0, cap=0.0, slopes=False, dtype="bf16", padding=0, backward=True),
        # 8192 content tokens and four blocks of 256 queries, its long form
        dict(name="train_9216", kind="attend", documents=1, tokens=8192, queries=1024, ragged=False, heads=16, kv_heads=4,
             head_dim=128, mask="causal", window=0, cap=0.0, slopes=False, dtype="bf16", padding=0, backward=True),
        # the largest: a packed microbatch of ragged documents, capped scores, as many key heads as query heads
        dict(name="train_packed", kind="attend", documents=13, tokens=4096, queries=0, ragged=True, heads=16, kv_heads=16,
             head_dim=128, mask="causal", window=0, cap=30.0, slopes=False, dtype="bf16", padding=77, backward=True),
        # wide heads, prefixes that see each other (an image before its text)
        dict(name="train_wide", kind="attend", documents=5, tokens=1531, queries=0, ragged=True, heads=8, kv_heads=2,
             head_dim=256, mask="prefix", window=0, cap=0.0, slopes=True, dtype="bf16", padding=0, backward=True),
        # evaluation: forward only with the scores' logarithms, a distance bias and a sliding window
        dict(name="eval_window", kind="attend", documents=7, tokens=4000, queries=0, ragged=True, heads=12, kv_heads=4,
             head_dim=64, mask="causal", window=1024, cap=0.0, slopes=True, dtype="fp16", padding=0, backward=False),
        # the new tokens of a decode step, scattered over the pool
        dict(name="append_decode", kind="append", tokens=64, heads=16, kv_heads=4, head_dim=128, rotary_dim=128, page=64,
             mixed=False, adjacent=False, far=70000, dtype="bf16"),
        # a prompt's chunk of text and images, an odd number of tokens; a quarter of each head turns
        dict(name="append_prefill", kind="append", tokens=8191, heads=16, kv_heads=4, head_dim=256, rotary_dim=64, page=64,
             mixed=True, adjacent=False, far=0, dtype="bf16"),
        # one interactive session: a content token and its read-only query over 9216 tokens
        dict(name="cached_one", kind="cached", requests=1, new=2, context=9216, ragged=False, heads=16, kv_heads=4,
             head_dim=128, page=64, window=0, cap=30.0, slopes=False, rows="query", dtype="bf16", padding=0, lse=True),
        # a serving batch of ragged lengths, one token each
        dict(name="cached_batch", kind="cached", requests=64, new=1, context=8192, ragged=True, heads=16, kv_heads=4,
             head_dim=128, page=64, window=0, cap=0.0, slopes=True, rows="causal", dtype="bf16", padding=0, lse=False),
        # a few long documents, wide heads, small pages
        dict(name="cached_long", kind="cached", requests=5, new=1, context=65536, ragged=True, heads=16, kv_heads=2,
             head_dim=256, page=16, window=0, cap=50.0, slopes=False, rows="causal", dtype="fp16", padding=3, lse=False),
        # a long prompt's next 4096 tokens over the 4096 before them
        dict(name="cached_chunk", kind="cached", requests=1, new=4096, context=4096, ragged=False, heads=16, kv_heads=4,
             head_dim=128, page=64, window=0, cap=30.0, slopes=False, rows="causal", dtype="bf16", padding=0, lse=False),
    ]


def spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "append", "cached", "cached"))
    dtype, d = rng.choice(("bf16", "bf16", "fp16")), rng.choice((64, 128, 128, 256))
    kv, group = rng.choice(((4, 4), (2, 4), (8, 1), (8, 2), (1, 8), (2, 7), (16, 1)))
    if kind == "attend":
        tokens, queries = spread(rng, 1, 8192), rng.choice((0, 0, spread(rng, 1, 1024)))
        # the plain form's scores, were every document the longest: no more than a half of the largest listed case's
        most = 13 * 16 * 4096 * 4096 * 128 // (2 * kv * group * d * tokens * (tokens + queries))
        return dict(kind=kind, documents=spread(rng, 1, max(1, min(64, most))), tokens=tokens, queries=queries,
                    ragged=rng.random() < 0.7, heads=kv * group, kv_heads=kv, head_dim=d,
                    mask=rng.choice(("causal", "causal", "prefix")), window=rng.choice((0, 0, spread(rng, 16, 4096))),
                    cap=rng.choice((0.0, 0.0, 20.0, 50.0)), slopes=rng.random() < 0.3, dtype=dtype,
                    padding=rng.choice((0, 0, 5, 200)), backward=rng.random() < 0.75)
    if kind == "append":
        return dict(kind=kind, tokens=spread(rng, 1, 8191 * 24 * 256 // ((kv * group + 2 * kv) * d)), heads=kv * group,
                    kv_heads=kv, head_dim=d, rotary_dim=rng.choice((d, d // 2, d // 4)), page=rng.choice((16, 32, 64, 128)),
                    mixed=rng.random() < 0.5, adjacent=rng.random() < 0.5, far=rng.choice((0, 5000, 300000, 20000000)),
                    dtype=dtype)
    if rng.random() < 0.5:
        new, context = rng.choice((1, 1, 1, 2, 4)), spread(rng, 1, 65536)
        requests = spread(rng, 1, max(1, min(128, (64 * 8192 * 4 * 128) // (context * kv * d))))
    else:
        new, context = spread(rng, 16, 4096), spread(rng, 1, 8192)
        requests = spread(rng, 1, max(1, min(16, (4096 * 8192 * 16) // (2 * new * (context + new) * kv * group))))
    return dict(kind=kind, requests=requests, new=new, context=context, ragged=rng.random() < 0.7, heads=kv * group,
                kv_heads=kv, head_dim=d, page=rng.choice((16, 32, 64, 128)),
                window=rng.choice((0, 0, 0, spread(rng, 16, 4096))), cap=rng.choice((0.0, 20.0, 50.0)),
                slopes=rng.random() < 0.4, rows="query" if new == 2 else "causal", dtype=dtype,
                padding=rng.choice((0, 0, 5)), lse=rng.random() < 0.5)


# ---- lengths: a case's own, the same for every seed ---------------------------------------------

def documents(case):
    """(tokens, queries, prefix) of every document."""
    r = random.Random("%d %d %d" % (case["documents"], case["tokens"], case["queries"]))
    got = []
    for i in range(case["documents"]):
        n = r.randint(max(1, case["tokens"] // 4), case["tokens"]) if case["ragged"] and i else case["tokens"]
        got.append((n, case["queries"], r.randint(0, n) if case["mask"] == "prefix" else 0))
    return got


def mask_rows(case):
    """(first key, limit, position) of every row, a document's queries behind its tokens; keys are the tokens.
    Queries come in blocks of up to 256, each of which sees the document up to a place of its own."""
    w, at, got = case["window"], 0, []
    for n, m, prefix in documents(case):
        seen = [(i, max(i + 1, prefix)) for i in range(n)]
        blocks = -(-m // 256)
        seen += [(e - 1, e) for e in (n * (i // 256 + 1) // blocks for i in range(m))]
        got += [(at + (max(0, p + 1 - w) if w else 0), at + limit, at + p) for p, limit in seen]
        at += n
    return got + [(0, 0, 0)] * case["padding"]


def lengths(case):
    """(tokens in the cache before the step, tokens of the step) of every request."""
    r = random.Random("%d %d %d" % (case["requests"], case["context"], case["new"]))
    n = case["requests"]
    if not case["ragged"]:
        return [case["context"]] * n, [case["new"]] * n
    before = [case["context"]] + [r.randint(case["context"] // 8, case["context"]) for _ in range(n - 1)]
    new = [case["new"]] + [case["new"] if case["new"] <= 4 else r.randint(1, case["new"]) for _ in range(n - 1)]
    return before, new


def limits(case):
    """How many positions of its request each row of the step sees: itself and all before it; with read-only
    queries, all that the step has written."""
    before, new = lengths(case)
    if case["rows"] == "query":
        return [b + 1 for b, m in zip(before, new) for _ in range(m)]
    return [b + 1 + i for b, m in zip(before, new) for i in range(m)]


# ---- inputs --------------------------------------------------------------------------------------

def rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def heads_of(gen, tokens, heads, d, dtype):
    """Rows as a projection gives them, some channels several times larger than the others."""
    wide = 1 + 3 * (torch.rand(heads, d, generator=gen, device=DEV) < 0.05)
    return (rand(gen, tokens, heads, d) * wide).to(dtype)


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def slopes_of(case):
    """One a head, falling from 2^(-8 / heads) to 2^-8."""
    n = case["heads"]
    return torch.tensor([2.0 ** (-8 * (i + 1) / n) for i in range(n)], device=DEV) if case["slopes"] else None


def prepare_attend(case, gen):
    hq, hk, d, dtype = case["heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    rows, docs = mask_rows(case), documents(case)
    t, n = len(rows), sum(x[0] for x in docs)
    first, limit, position = (int32(list(x)) for x in zip(*rows))
    s = dict(q=heads_of(gen, t, hq, d, dtype), k=heads_of(gen, n, hk, d, dtype), v=heads_of(gen, n, hk, d, dtype),
             first=first, limit=limit, position=position, slopes=slopes_of(case),
             rows=int32([0] + [a + b for a, b, _ in docs]).cumsum(0), keys=int32([0] + [a for a, _, _ in docs]).cumsum(0),
             most=max(a + b for a, b, _ in docs), longest=max(a for a, _, _ in docs))
    if case["backward"]:
        for x in "qkv":
            s[x].requires_grad_()
        s["dy"] = rand(gen, t, hq, d).to(dtype)
    return s


def prepare_append(case, gen):
    t, hq, hk, d, r, page = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim", "rotary_dim", "page"))
    dtype = DTYPES[case["dtype"]]
    rows = heads_of(gen, t, hq + 2 * hk, d, dtype)  # the fused projection: q, k and v are its columns
    i = torch.arange(t, device=DEV)
    # runs of 64 tokens of text (the three axes alike) and images of 16 x 16 in turn
    base, at = i // 320 * 80 + case["far"], i % 320
    image, p = at >= 64, (at - 64).clamp(min=0)
    positions = torch.stack((torch.where(image, base + 64, base + at), torch.where(image, base + 64 + p // 16, base + at),
                             torch.where(image, base + 64 + p % 16, base + at))).int()
    n = r // 2
    freq = [1e6 ** (-2 * j / r) for j in range(n)]
    first, second = n // 4, (n - n // 4) // 2
    axis = [j % 3 if case["mixed"] else 0 if j < first else 1 if j < first + second else 2 for j in range(n)]
    pages = -(-t * 5 // (4 * page))
    slots = torch.randperm(pages * page, generator=gen, device=DEV)[:t].int()  # every token at a place of its own
    if t > 64:  # a prompt's tokens fill whole pages, which lie anywhere
        order = torch.randperm(pages, generator=gen, device=DEV)
        slots = (order[:, None] * page + torch.arange(page, device=DEV)).flatten()[:t].int()
    slots[t // 2 :: 97] = -1  # padding rows, not written
    return dict(q=rows[:, :hq], k=rows[:, hq : hq + hk], v=rows[:, hq + hk :], slots=slots, positions=positions,
                freq=torch.tensor(freq, dtype=torch.float64, device=DEV), axis=int32(axis),
                # the same frequencies as turns a position, in units of 2^-64 of a turn
                turns=torch.tensor([round(f / (2 * math.pi) * 2.0**64) for f in freq], dtype=torch.int64, device=DEV),
                data=torch.zeros(pages, hk, 2, page, d, dtype=dtype, device=DEV))


def prepare_cached(case, gen):
    before, new = lengths(case)
    hq, hk, d, page = (case[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    dtype, n = DTYPES[case["dtype"]], case["requests"]
    held = [-(-(b + m) // page) for b, m in zip(before, new)]
    data = torch.empty(sum(held) + 3, hk, 2, page, d, dtype=dtype, device=DEV)
    wide = 1 + 3 * (torch.rand(hk, 2, 1, d, generator=gen, device=DEV) < 0.05)
    step = max(1, (1 << 26) // (hk * page * d))
    for at in range(0, data.shape[0], step):
        data[at : at + step] = rand(gen, *data[at : at + step].shape) * wide
    tables = torch.full((n, max(held) + 1), -1, dtype=torch.int32, device=DEV)
    tables[torch.arange(max(held) + 1, device=DEV)[None] < torch.tensor(held, device=DEV)[:, None]] = torch.randperm(
        data.shape[0], generator=gen, device=DEV)[: sum(held)].int()
    see = limits(case)
    return dict(q=heads_of(gen, len(see) + case["padding"], hq, d, dtype), data=data, tables=tables,
                starts=int32([0] + new).cumsum(0).int(), visible=int32(see + [0] * case["padding"]),
                slopes=slopes_of(case), longest=max(b + m for b, m in zip(before, new)), most=max(new))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return dict(dict(attend=prepare_attend, append=prepare_append, cached=prepare_cached)[case["kind"]](case, gen), case=case)


# ---- the plain forms -----------------------------------------------------------------------------

def scored(case, x, distance, slopes, seen):
    """Scores [n, hk, rows, group, keys] of the products x, and what a change of x changes them by.  ``distance``
    and ``seen`` [n, 1, rows, 1, keys] say how far a key lies from a row, and whether the row sees it."""
    x = x * case["head_dim"] ** -0.5
    rate = None
    if case["cap"]:
        rate = torch.tanh(x / case["cap"])
        x = case["cap"] * rate
        rate = 1 - rate * rate
    if slopes is not None:
        x = x - slopes.view(1, case["kv_heads"], 1, -1, 1) * distance
    return torch.where(seen, x, -math.inf), rate


def normal(x):
    """Softmax over the last axis, 0 for rows without a key, and the logarithms of the sums."""
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    w = (x - top).exp()
    total = w.sum(-1, keepdim=True)
    return torch.where(total > 0, w / total, 0.0), (top + total.log()).squeeze(-1)


def plain_attend(s):
    case, q = s["case"], s["q"].detach()
    hq, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    group = hq // hk
    row = s["rows"][:-1, None] + torch.arange(s["most"], device=q.device)
    key = s["keys"][:-1, None] + torch.arange(s["longest"], device=q.device)
    real, there = row < s["rows"][1:, None], key < s["keys"][1:, None]
    row, key = row.clamp(max=q.shape[0] - 1), key.clamp(max=s["k"].shape[0] - 1)
    n = row.shape[0]
    apart = lambda x: x[:, None, :, None, None]  # noqa: E731
    near = key[:, None, None, None, :]
    seen = (near >= apart(s["first"][row])) & (near < apart(s["limit"][row])) & apart(real) & there[:, None, None, None, :]
    distance = (apart(s["position"][row]) - near).abs()
    queries = lambda x: x[row].float().view(n, -1, hk, group, d).transpose(1, 2).flatten(2, 3)  # noqa: E731
    keys = lambda x: x.detach()[key].float().transpose(1, 2).contiguous()  # noqa: E731
    rows = lambda x: x.view(n, hk, -1, group, d).transpose(1, 2).flatten(2, 3)  # noqa: E731
    x, k, v = queries(q), keys(s["k"]), keys(s["v"])  # [n, hk, rows * group, d], [n, hk, keys, d]
    w, rate = scored(case, (x @ k.transpose(2, 3).contiguous()).view(n, hk, -1, group, key.shape[1]), distance,
                     s["slopes"], seen)
    w, sums = normal(w)
    w = w.flatten(2, 3)
    out = torch.zeros(q.shape, device=q.device)
    out[row[real]] = rows(w @ v)[real]
    got = {"out": out.to(q.dtype)}
    if not case["backward"]:
        lse = torch.full(q.shape[:2], -math.inf, device=q.device)
        lse[row[real]] = sums.transpose(1, 2).flatten(2)[real]
        return got | {"lse": lse}
    dy = queries(s["dy"]) * real[:, None, :, None, None].expand(n, 1, -1, group, 1).flatten(2, 3)
    dv = w.transpose(2, 3).contiguous() @ dy
    dw = dy @ v.transpose(2, 3).contiguous()
    dw = w * (dw - (w * dw).sum(-1, keepdim=True)) * d**-0.5
    if rate is not None:
        dw = dw * rate.flatten(2, 3)
    dk = dw.transpose(2, 3).contiguous() @ x
    dq = torch.zeros(q.shape, device=q.device)
    dq[row[real]] = rows(dw @ k)[real]
    back = lambda x: x.transpose(1, 2)[there].to(q.dtype)  # noqa: E731
    return got | {"dq": dq.to(q.dtype), "dk": back(dk), "dv": back(dv)}


def plain_append(s):
    case, slots = s["case"], s["slots"].long()
    r, page = case["rotary_dim"], case["page"]
    angle = s["positions"][s["axis"].long()].t().double() * s["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x):
        y = x.float()
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if case["adjacent"] else (y[..., : r // 2], y[..., r // 2 : r])
        a, b = a * cos - b * sin, b * cos + a * sin
        both = torch.stack((a, b), -1).flatten(-2) if case["adjacent"] else torch.cat((a, b), -1)
        return torch.cat((both, y[..., r:]), -1).to(x.dtype)

    real = slots >= 0
    p, o = slots[real] // page, slots[real] % page
    s["data"][p, :, 0, o] = turned(s["k"])[real]
    s["data"][p, :, 1, o] = s["v"][real]
    return {"q": turned(s["q"]), "data": s["data"]}


def plain_cached(s):
    case, q, starts = s["case"], s["q"], s["starts"].long()
    hq, hk, d, page = (case[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    n, group, most = starts.numel() - 1, hq // hk, s["most"]
    columns = -(-s["longest"] // page)
    held = s["data"][s["tables"][:, :columns].clamp(min=0).long()]  # [n, columns, hk, 2, page, d]
    k, v = (held[:, :, :, i].transpose(1, 2).flatten(2, 3).float() for i in (0, 1))  # [n, hk, columns * page, d]
    row = starts[:-1, None] + torch.arange(most, device=q.device)
    real = row < starts[1:, None]
    row = row.clamp(max=q.shape[0] - 1)
    see = torch.where(real, s["visible"][row], 0)[:, None, :, None, None]
    at = torch.arange(columns * page, device=q.device)
    seen = (at < see) & (at >= see - case["window"]) if case["window"] else at < see
    x = q[row].float().view(n, most, hk, group, d).transpose(1, 2).flatten(2, 3)  # [n, hk, most * group, d]
    x = (x @ k.transpose(2, 3).contiguous()).view(n, hk, most, group, -1)
    w, sums = normal(scored(case, x, (see - 1 - at).abs(), s["slopes"], seen)[0])
    out = torch.zeros(q.shape, device=q.device)
    out[row[real]] = (w.flatten(2, 3) @ v).view(n, hk, most, group, d).transpose(1, 2).flatten(2, 3)[real]
    got = {"out": out.to(q.dtype)}
    if case["lse"]:
        lse = torch.full(q.shape[:2], -math.inf, device=q.device)
        lse[row[real]] = sums.transpose(1, 2).flatten(2)[real]
        got["lse"] = lse
    return got


# ---- the framework's operators -------------------------------------------------------------------

@functools.cache
def framework():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "cq-pretrain_amd"))
    from cqgdn import attention, kvcache, rotary

    return attention, kvcache, rotary


def own_attend(s):
    attention, _, _ = framework()
    case = s["case"]
    given = dict(first=s["first"], cap=case["cap"] or None, slopes=s["slopes"],
                 positions=s["position"] if case["slopes"] else None)
    if not case["backward"]:
        out, lse = attention.attend(s["q"], s["k"], s["v"], s["limit"], return_lse=True, **given)
        return {"out": out, "lse": lse}
    out = attention.attend(s["q"], s["k"], s["v"], s["limit"], **given)
    dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dy"])
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def own_append(s):
    _, kvcache, rotary = framework()
    case = s["case"]
    cache = kvcache.KVCache(s["data"], page=case["page"], head_dim=case["head_dim"], dtype=s["k"].dtype)
    plan = rotary.RotaryPlan(s["turns"], s["axis"], adjacent=case["adjacent"])
    return {"q": kvcache.append(cache, s["q"], s["k"], s["v"], s["positions"], plan, s["slots"]), "data": s["data"]}


def own_cached(s):
    _, kvcache, _ = framework()
    case = s["case"]
    cache = kvcache.KVCache(s["data"], page=case["page"], head_dim=case["head_dim"], dtype=s["q"].dtype)
    got = kvcache.attend(s["q"], cache, s["tables"], s["starts"], s["visible"], window=case["window"] or None,
                         cap=case["cap"] or None, slopes=s["slopes"], max_queries=s["most"], return_lse=case["lse"])
    return dict(zip(("out", "lse"), got)) if case["lse"] else {"out": got}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return dict(attend=own_attend, append=own_append, cached=own_cached)[kind](state)
    return dict(attend=plain_attend, append=plain_append, cached=plain_cached)[kind](state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    d, hq, hk = case["head_dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        t = case["tokens"]
        return {"bytes": 2 * 2 * t * (hq + 2 * hk) * d + 16 * t, "flops": 3 * t * (hq + hk) * case["rotary_dim"]}
    if case["kind"] == "attend":
        rows, keys = mask_rows(case), sum(x[0] for x in documents(case))
        seen = sum(max(0, limit - first) for first, limit, _ in rows) * hq
        # q and the output, k and v; backward: those and the output's gradient in, three gradients out
        q, k = 2 * len(rows) * hq * d, 2 * keys * hk * d
        if case["backward"]:
            return {"bytes": 2 * q + 2 * k + 4 * q + 4 * k + 8 * len(rows), "flops": (4 + 10) * seen * d}
        return {"bytes": 2 * q + 2 * k + 4 * len(rows) * hq + 8 * len(rows), "flops": 4 * seen * d}
    before, new = lengths(case)
    see, w = limits(case), case["window"]
    seen = sum(min(x, w) if w else x for x in see)
    held, at = 0, 0
    for m in new:  # what the rows of a request see together
        held += see[at + m - 1] - (max(0, see[at] - w) if w else 0)
        at += m
    rows = (len(see) + case["padding"]) * hq
    return {"bytes": held * hk * 4 * d + 4 * rows * d + (4 * rows if case["lse"] else 0), "flops": 4 * seen * hq * d}


# ---- the operators' definitions, in 64 bits ------------------------------------------------------

def scores64(case, q, k, distance, slope, hidden):
    """Scores of one head's rows in float64 and the derivative of the cap."""
    x = torch.matmul(q, k.t()) / math.sqrt(case["head_dim"])
    rate = None
    if case["cap"]:
        e = torch.exp(-2 * x.abs() / case["cap"])  # tanh |y| = (1 - e) / (1 + e), and its derivative 4 e / (1 + e)^2
        rate = 4 * e / (1 + e) ** 2
        x = torch.sign(x) * case["cap"] * (1 - e) / (1 + e)
    if slope is not None:
        x = x - float(slope) * distance.double()
    return x.masked_fill(hidden, -math.inf), rate


def exact_attend(case, s):
    hk, group, d = case["kv_heads"], case["heads"] // case["kv_heads"], case["head_dim"]
    q, k, v = (s[x].detach() for x in "qkv")
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    dq, dk, dv = torch.zeros_like(out), torch.zeros(k.shape, dtype=torch.float64, device=DEV), torch.zeros(
        k.shape, dtype=torch.float64, device=DEV)
    r, c = 0, 0
    for n, m, _ in documents(case):
        rows, keys = slice(r, r + n + m), slice(c, c + n)
        at = torch.arange(c, c + n, device=DEV)
        hidden = (at < s["first"][rows, None]) | (at >= s["limit"][rows, None])
        distance = (s["position"][rows, None] - at).abs()
        r, c = r + n + m, c + n
        for h in range(hk * group):
            a, b, g = q[rows, h].double(), k[keys, h // group].double(), v[keys, h // group].double()
            x, rate = scores64(case, a, b, distance, None if s["slopes"] is None else s["slopes"][h], hidden)
            total = torch.logsumexp(x, -1)
            w = torch.exp(x - torch.where(total == -math.inf, 0.0, total)[:, None])
            out[rows, h], lse[rows, h] = torch.matmul(w, g), total
            if not case["backward"]:
                continue
            dy = s["dy"][rows, h].double()
            dv[keys, h // group] += torch.matmul(w.t(), dy)
            dx = w * (torch.matmul(dy, g.t()) - (dy * out[rows, h]).sum(-1, keepdim=True)) / math.sqrt(d)
            dx = dx if rate is None else dx * rate
            dq[rows, h] = torch.matmul(dx, b)
            dk[keys, h // group] += torch.matmul(dx.t(), a)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if case["backward"] else {"out": out, "lse": lse}


def exact_append(case, s):
    n, page = case["rotary_dim"] // 2, case["page"]
    i = torch.arange(n, device=DEV)
    one, two = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + n)
    at = torch.stack([s["positions"][int(a)] for a in s["axis"]], 1).double()
    turn = torch.polar(torch.ones_like(at), at * s["freq"])[:, None]

    def turned(x):
        y = x.double()
        z = torch.complex(y[..., one], y[..., two]) * turn
        y[..., one], y[..., two] = z.real, z.imag
        return y

    data, slots = s["data"].double(), s["slots"].long()
    k, t = turned(s["k"]), torch.nonzero(slots >= 0)[:, 0]
    flat = data.permute(0, 3, 1, 2, 4).reshape(-1, case["kv_heads"], 2, case["head_dim"])  # a row a slot
    flat[slots[t]] = torch.stack((k[t], s["v"][t].double()), 2)
    return {"q": turned(s["q"]), "data": flat.unflatten(0, (-1, page)).permute(0, 2, 3, 1, 4).contiguous()}


def exact_cached(case, s):
    d, page, hk, w = case["head_dim"], case["page"], case["kv_heads"], case["window"]
    group, starts, see = case["heads"] // hk, s["starts"].tolist(), s["visible"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for r in range(case["requests"]):
        a, b = starts[r], starts[r + 1]
        last = max(see[a:b])
        held = s["data"][s["tables"][r, : -(-last // page)].long()]
        limit, at = s["visible"][a:b, None], torch.arange(last, device=DEV)
        hidden = (at >= limit) | (at < limit - w) if w else at >= limit
        for h in range(hk * group):
            k, v = (held[:, h // group, i].flatten(0, 1)[:last].double() for i in (0, 1))
            x, _ = scores64(case, s["q"][a:b, h].double(), k, (limit - 1 - at).abs(),
                            None if s["slopes"] is None else s["slopes"][h], hidden)
            lse[a:b, h] = torch.logsumexp(x, -1)
            out[a:b, h] = torch.matmul(torch.softmax(x, -1), v)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def exact(case, seed):
    s = prepare(case, seed)
    return dict(attend=exact_attend, append=exact_append, cached=exact_cached)[case["kind"]](case, s)
