"""The operators of the attention layers beside the GDN layers, and what they are timed on.

A hybrid stack has one attention layer after every three GDN layers.  Serving it takes, for each
attention layer, the rotary positions of its queries and keys, a paged cache of keys and values
(held here in 4 bits), the attention that reads it, and once a step the pages themselves:

* ``rotary``  rotary positions with several axes (time, height, width), forward and backward;
* ``pages``   block tables, slot maps and row limits of a step, built from request lengths;
* ``write``   keys and values rounded into the 4-bit pages, and the values those hold read back;
* ``attend``  attention of a step's query rows over the pages, one token or many a request.

``run`` computes each in its plain form (elementary torch operations, 32 bits, rounded once at the
end) or, with ``own``, through the framework's entry points.  ``exact`` restates each in float64.

A page of the cache holds, for one head, the codes of its keys [page][D/2], then those of its values,
then the scale bytes of its keys [page][D/32] and of its values.  A code is a sign, two exponent bits
and one mantissa bit (0, .5, 1, 1.5, 2, 3, 4, 6), the even value of a pair in the low half of its byte;
a scale byte b multiplies 32 neighbouring values by 2^(b - 127), and 255 makes them NaN.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False  # True: run() calls the framework's operators

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decode step of 23 sequences, a content token and its read-only query each
        dict(name="rotary_decode", kind="rotary", tokens=46, heads=16, kv_heads=4, head_dim=128, rotary_dim=128,
             mixed=False, adjacent=False, dtype="bf16", far=70000, backward=False),
        # a training step on images between text: 8192 content tokens and four blocks of 256 queries; a quarter
        # of each 256-wide head turns, the axes taking turns over the frequencies
        dict(name="rotary_train", kind="rotary", tokens=9216, heads=16, kv_heads=4, head_dim=256, rotary_dim=64,
             mixed=True, adjacent=False, dtype="bf16", far=0, backward=True),
        # the largest: a packed microbatch of a model with as many key heads as query heads
        dict(name="rotary_packed", kind="rotary", tokens=32768, heads=16, kv_heads=16, head_dim=128, rotary_dim=128,
             mixed=False, adjacent=True, dtype="bf16", far=0, backward=True),
        # a decode step of a serving batch: one token a request, a page begun now and then
        dict(name="pages_decode", kind="pages", requests=64, new=1, context=8192, page=64, padding=0),
        # admission of many prompts at once beside running requests, into a buffer of fixed size
        dict(name="pages_prefill", kind="pages", requests=1000, new=61, context=2000, page=16, padding=531),
        # the tokens of a decode step, scattered over the pool
        dict(name="write_decode", kind="write", tokens=64, kv_heads=4, head_dim=128, page=64, dtype="bf16"),
        # a prompt's chunk, an odd number of tokens
        dict(name="write_prefill", kind="write", tokens=8191, kv_heads=16, head_dim=128, page=64, dtype="bf16"),
        # one interactive session: a content token and its read-only query over 9216 tokens
        dict(name="attend_one", kind="attend", requests=1, new=2, context=9216, ragged=False, heads=16, kv_heads=4,
             head_dim=128, page=64, window=0, rows="query", dtype="bf16", padding=0, lse=True),
        # a serving batch of ragged lengths, one token each
        dict(name="attend_batch", kind="attend", requests=64, new=1, context=8192, ragged=True, heads=16, kv_heads=4,
             head_dim=128, page=64, window=0, rows="causal", dtype="bf16", padding=0, lse=False),
        # a few long documents, wide heads, small pages
        dict(name="attend_long", kind="attend", requests=5, new=1, context=65536, ragged=True, heads=16, kv_heads=2,
             head_dim=256, page=16, window=0, rows="causal", dtype="bf16", padding=3, lse=False),
        # a long prompt's next 4096 tokens over the 4096 before them
        dict(name="attend_prefill", kind="attend", requests=1, new=4096, context=4096, ragged=False, heads=16,
             kv_heads=4, head_dim=128, page=64, window=0, rows="causal", dtype="bf16", padding=0, lse=False),
        # ragged prompts together in fp16, a sliding window, rows of padding behind
        dict(name="attend_packed", kind="attend", requests=7, new=1531, context=700, ragged=True, heads=16,
             kv_heads=8, head_dim=128, page=32, window=1024, rows="causal", dtype="fp16", padding=77, lse=True),
    ]


def spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("rotary", "pages", "write", "attend", "attend"))
    if kind == "rotary":
        d = rng.choice((64, 128, 256))
        heads, kv = rng.choice(((16, 4), (16, 16), (8, 2), (12, 1), (7, 7)))
        most = 32768 * 32 * 128 // ((heads + kv) * d)
        return dict(kind=kind, tokens=spread(rng, 1, min(32768, most)), heads=heads, kv_heads=kv, head_dim=d,
                    rotary_dim=rng.choice((d, d // 2, d // 4)), mixed=rng.random() < 0.5, adjacent=rng.random() < 0.5,
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), far=rng.choice((0, 5000, 300000, 20000000)),
                    backward=rng.random() < 0.6)
    if kind == "pages":
        return dict(kind=kind, requests=spread(rng, 1, 2000), new=spread(rng, 1, 64), context=spread(rng, 1, 8192),
                    page=rng.choice((16, 32, 64, 128)), padding=rng.randrange(0, 300))
    if kind == "write":
        kv, d = rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 128, 256))
        return dict(kind=kind, tokens=spread(rng, 1, 8192 * 16 * 128 // (kv * d)), kv_heads=kv, head_dim=d,
                    page=rng.choice((16, 32, 64, 128)), dtype=rng.choice(("bf16", "bf16", "fp16")))
    kv, group = rng.choice(((4, 4), (2, 8), (8, 1), (8, 2), (1, 8), (2, 7), (16, 1)))
    d = rng.choice((64, 128, 128, 256))
    decode = rng.random() < 0.5
    if decode:
        new = rng.choice((1, 1, 1, 2, 4))
        context = spread(rng, 1, 65536)
        requests = spread(rng, 1, max(1, min(128, (64 * 8192 * 4 * 128) // (context * kv * d))))
    else:
        new, context = spread(rng, 16, 4096), spread(rng, 1, 8192)
        requests = spread(rng, 1, max(1, min(16, (4096 * 8192 * 16) // (2 * new * (context + new) * kv * group))))
    return dict(kind=kind, requests=requests, new=new, context=context, ragged=rng.random() < 0.7, heads=kv * group,
                kv_heads=kv, head_dim=d, page=rng.choice((16, 32, 64, 128)),
                window=rng.choice((0, 0, 0, spread(rng, 16, 4096))),
                rows="query" if new == 2 else "causal", dtype=rng.choice(("bf16", "bf16", "fp16")),
                padding=rng.choice((0, 0, 5)), lse=rng.random() < 0.5)


# ---- lengths: a case's own, the same for every seed ---------------------------------------------

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

def encode(x):
    """The codes (two a byte) and scale bytes of x [..., D]."""
    x = x.float().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    part, e = torch.frexp(top)
    # the scale under which the largest value lies in [4, 8); one more where it would be cut by over 1
    s = torch.where(part > 0.875, e - 2, e - 3).clamp(-125, 127)
    fine = torch.isfinite(top)
    y = torch.where(fine, torch.ldexp(x, -s), 0.0)
    a = y.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = (code | (torch.signbit(y).to(torch.uint8) << 3)).to(torch.uint8).flatten(-2)
    scale = torch.where(fine, s + 127, 255).to(torch.uint8).squeeze(-1)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def decode(code, scale):
    """The fp32 values of codes [..., D/2] and scale bytes [..., D/32]."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=code.device)
    v = torch.stack((grid[(code & 15).long()], grid[(code >> 4).long()]), -1).flatten(-2)
    f = torch.ldexp(torch.ones((), device=code.device), scale.int() - 127)
    f = torch.where(scale == 255, float("nan"), f)
    return (v.unflatten(-1, (-1, 32)) * f.unsqueeze(-1)).flatten(-2)


def parts(data, page, d):
    """The four parts of pages [..., bytes]: key codes, value codes, key scales, value scales."""
    c, s = page * d // 2, page * d // 32
    k, v, ks, vs = data.split((c, c, s, s), -1)
    return (k.unflatten(-1, (page, d // 2)), v.unflatten(-1, (page, d // 2)), ks.unflatten(-1, (page, d // 32)),
            vs.unflatten(-1, (page, d // 32)))


def page_bytes(page, d):
    return page * (d + d // 16)


def rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def heads_of(gen, tokens, heads, d, dtype):
    """Rows as a projection gives them, some channels several times larger than the others."""
    wide = 1 + 3 * (torch.rand(heads, d, generator=gen, device=DEV) < 0.05)
    return (rand(gen, tokens, heads, d) * wide).to(dtype)


def prepare_rotary(case, gen):
    t, hq, hk, d, r = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim", "rotary_dim"))
    dtype = DTYPES[case["dtype"]]
    rows = rand(gen, t, (hq + 2 * hk) * d).to(dtype)  # the fused projection: q, k and v are its columns
    i = torch.arange(t, device=DEV)
    # runs of 64 tokens of text (the three axes alike) and images of 16 x 16 in turn
    run, at = i // 320, i % 320
    base = run * 80 + case["far"]
    image = at >= 64
    p = (at - 64).clamp(min=0)
    positions = torch.stack((torch.where(image, base + 64, base + at), torch.where(image, base + 64 + p // 16, base + at),
                             torch.where(image, base + 64 + p % 16, base + at))).int()
    n = r // 2
    freq = [1e6 ** (-2 * j / r) for j in range(n)]
    first, second = n // 4, (n - n // 4) // 2
    axis = [j % 3 if case["mixed"] else 0 if j < first else 1 if j < first + second else 2 for j in range(n)]
    s = dict(q=rows[:, : hq * d].view(t, hq, d), k=rows[:, hq * d : (hq + hk) * d].view(t, hk, d),
             positions=positions, freq=torch.tensor(freq, dtype=torch.float64, device=DEV),
             # the same frequencies as turns a position, in units of 2^-64 of a turn
             turns=torch.tensor([round(f / (2 * math.pi) * 2.0**64) for f in freq], dtype=torch.int64, device=DEV),
             axis=torch.tensor(axis, dtype=torch.int32, device=DEV))
    if case["backward"]:
        s["q"].requires_grad_()
        s["k"].requires_grad_()
        s |= dict(dq=rand(gen, t, hq, d).to(dtype), dk=rand(gen, t, hk, d).to(dtype))
    return s


def page_lengths(case):
    """(cached, new) of every request: some finished (-1), some idle, most running, new prompts among them."""
    r = random.Random("%d %d %d" % (case["requests"], case["context"], case["new"]))
    cached, new = [], []
    for _ in range(case["requests"]):
        what = r.random()
        cached.append(0 if what < 0.1 else r.randint(1, case["context"]))
        new.append(-1 if 0.1 < what < 0.15 else 0 if 0.15 < what < 0.2 else r.randint(1, case["new"]))
    return cached, new


def prepare_pages(case, gen):
    cached, new = page_lengths(case)
    page, n = case["page"], case["requests"]
    up = lambda x: -(-x // page)  # noqa: E731
    held, total = [up(c) for c in cached], sum(max(m, 0) for m in new) + case["padding"]
    columns = up(case["context"] + case["new"])
    needed = sum(max(0, up(c + m) - up(c)) for c, m in zip(cached, new))
    spare = max(1, needed - case["requests"] // 8 if case["requests"] % 2 else needed + 5)  # odd batches run out of pages
    ids = torch.randperm(sum(held) + spare, generator=gen, device=DEV).int()
    tables = torch.full((n, columns), -1, dtype=torch.int32, device=DEV)
    h = torch.tensor(held, device=DEV)
    tables[torch.arange(columns, device=DEV)[None] < h[:, None]] = ids[: sum(held)]
    free = torch.zeros(sum(held) + spare, dtype=torch.int32, device=DEV)
    free[:spare] = ids[sum(held):]
    return dict(cached=torch.tensor(cached, dtype=torch.int32, device=DEV), tables=tables, free=free,
                new=torch.tensor(new, dtype=torch.int32, device=DEV), tokens=total,
                free_count=torch.tensor([spare], dtype=torch.int32, device=DEV))


def prepare_write(case, gen):
    t, h, d, page = (case[k] for k in ("tokens", "kv_heads", "head_dim", "page"))
    dtype = DTYPES[case["dtype"]]
    rows = torch.cat((heads_of(gen, t, h, d, dtype), heads_of(gen, t, h, d, dtype)), 1)
    pages = -(-t * 5 // (4 * page))
    slots = torch.randperm(pages * page, generator=gen, device=DEV)[:t].int()  # every token at a place of its own
    if t > 64:  # a prompt's tokens fill whole pages, which lie anywhere
        order = torch.randperm(pages, generator=gen, device=DEV)
        slots = (order[:, None] * page + torch.arange(page, device=DEV)).flatten()[:t].int()
    slots[t // 2 :: 97] = -1  # padding rows, not written
    return dict(k=rows[:, :h], v=rows[:, h:], slots=slots,
                data=torch.zeros(pages, h, page_bytes(page, d), dtype=torch.uint8, device=DEV))


def prepare_attend(case, gen):
    before, new = lengths(case)
    hq, hk, d, page = (case[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    dtype, n = DTYPES[case["dtype"]], case["requests"]
    held = [-(-(b + m) // page) for b, m in zip(before, new)]
    data = torch.empty(sum(held) + 3, hk, page_bytes(page, d), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (hk * page * d))
    wide = [1 + 3 * (torch.rand(hk, 1, d, generator=gen, device=DEV) < 0.05) for _ in range(2)]
    for at in range(0, data.shape[0], step):
        part = data[at : at + step]
        for x, c, s in zip(wide, parts(part, page, d)[:2], parts(part, page, d)[2:]):
            code, scale = encode((rand(gen, part.shape[0], hk, page, d) * x).to(dtype))
            c.copy_(code)
            s.copy_(scale)
    tables = torch.full((n, max(held) + 1), -1, dtype=torch.int32, device=DEV)
    tables[torch.arange(max(held) + 1, device=DEV)[None] < torch.tensor(held, device=DEV)[:, None]] = torch.randperm(
        data.shape[0], generator=gen, device=DEV)[: sum(held)].int()
    starts = torch.tensor([0] + new, device=DEV).cumsum(0).int()
    see = limits(case)
    t = len(see) + case["padding"]
    visible = torch.tensor(see + [0] * case["padding"], dtype=torch.int32, device=DEV)
    return dict(q=heads_of(gen, t, hq, d, dtype), data=data, tables=tables, starts=starts, visible=visible,
                longest=max(b + m for b, m in zip(before, new)), most=max(new))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    make = dict(rotary=prepare_rotary, pages=prepare_pages, write=prepare_write, attend=prepare_attend)[case["kind"]]
    return dict(make(case, gen), case=case)


# ---- the plain forms -----------------------------------------------------------------------------

def plain_rotary(s):
    case = s["case"]
    r = case["rotary_dim"]
    angle = s["positions"][s["axis"].long()].t().double() * s["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, sin):
        y = x.detach().float()
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if case["adjacent"] else (y[..., : r // 2], y[..., r // 2 : r])
        a, b = a * cos - b * sin, b * cos + a * sin
        both = torch.stack((a, b), -1).flatten(-2) if case["adjacent"] else torch.cat((a, b), -1)
        return torch.cat((both, y[..., r:]), -1).to(x.dtype)

    out = {"q": turned(s["q"], sin), "k": turned(s["k"], sin)}
    if case["backward"]:
        out |= {"dq": turned(s["dq"], -sin), "dk": turned(s["dk"], -sin)}
    return out


def plain_pages(s):
    page, tokens, cached, new, tables = s["case"]["page"], s["tokens"], s["cached"], s["new"], s["tables"]
    n, columns = tables.shape
    zero = torch.zeros(1, dtype=torch.int64, device=new.device)
    up = lambda x: (x + page - 1) // page  # noqa: E731
    cached, new, free, count = cached.long(), new.long(), s["free"].clone(), s["free_count"].long()
    starts = torch.cat((zero, new.clamp(min=0).cumsum(0)))
    # the pages of finished requests go on top of the pool
    gone = torch.where(new < 0, up(cached), 0)
    column = torch.arange(columns, device=new.device)
    at = (count + gone.cumsum(0) - gone)[:, None] + column
    put = (column < gone[:, None]) & (at < free.numel())
    free[at[put]] = tables[put]
    count = (count + gone.sum()).clamp(max=free.numel())
    # each request that fits takes what it needs from the top, in order
    fits = (new > 0) & (cached + new <= columns * page) & (starts[:-1] + new <= tokens)
    need = torch.where(fits, up(cached + new) - up(cached), 0)
    before = need.cumsum(0) - need
    admitted = (new <= 0) | (fits & ((need == 0) | (before + need <= count)))
    take = torch.where(admitted, need, 0)
    j = column - up(cached)[:, None]
    fresh = (j >= 0) & (j < take[:, None])
    tables[fresh] = free[(count - 1 - before[:, None] - j)[fresh]]
    t = torch.arange(tokens, device=new.device)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    real = r < n
    r = r.clamp(max=n - 1)
    p = torch.where(real, cached[r] + t - starts[r], 0)
    entry = tables[r, (p // page).clamp(max=columns - 1)].long()
    good = real & admitted[r] & (entry >= 0)
    return {"starts": starts.int(), "lengths": torch.where(new < 0, 0, cached + torch.where(admitted, new, 0)).int(),
            "admitted": admitted.int(), "free_count": (count - take.sum()).int(), "free": free,
            "slots": torch.where(good, entry * page + p % page, -1).int(), "positions": p.int(),
            "visible": torch.where(good, p + 1, 0).int(), "tables": tables}


def plain_write(s):
    case, slots = s["case"], s["slots"].long()
    page, dtype = case["page"], s["k"].dtype
    kc, vc, ks, vs = parts(s["data"], page, case["head_dim"])
    real = slots >= 0
    p, o = slots[real] // page, slots[real] % page
    for x, c, f in ((s["k"], kc, ks), (s["v"], vc, vs)):
        code, scale = encode(x[real])
        c[p, :, o] = code
        f[p, :, o] = scale
    p, o = slots.clamp(min=0) // page, slots.clamp(min=0) % page
    return {name: torch.where(real[:, None, None], decode(c[p, :, o], f[p, :, o]), 0.0).to(dtype)
            for name, c, f in (("k", kc, ks), ("v", vc, vs))}


def plain_attend(s):
    case, q, starts = s["case"], s["q"], s["starts"].long()
    hq, hk, d, page = (case[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    n, group, most = starts.numel() - 1, hq // hk, s["most"]
    columns = -(-s["longest"] // page)
    held = s["data"][s["tables"][:, :columns].clamp(min=0).long()]  # [n, columns, hk, bytes]
    kc, vc, ks, vs = (x.transpose(1, 2).flatten(2, 3) for x in parts(held, page, d))
    k, v = decode(kc, ks), decode(vc, vs)  # [n, hk, columns * page, d]
    row = starts[:-1, None] + torch.arange(most, device=q.device)
    real = row < starts[1:, None]
    row = row.clamp(max=q.shape[0] - 1)
    see = torch.where(real, s["visible"][row], 0)[:, None, :, None, None]
    at = torch.arange(columns * page, device=q.device)
    mask = at < see if not case["window"] else (at < see) & (at >= see - case["window"])
    x = q[row].float().view(n, most, hk, group, d).transpose(1, 2).flatten(2, 3)  # [n, hk, most * group, d]
    w = (x @ k.transpose(2, 3).contiguous()) * d**-0.5
    w = torch.where(mask, w.view(n, hk, most, group, -1), -math.inf).view_as(w)
    top = w.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    w = (w - top).exp()
    total = w.sum(-1, keepdim=True)
    y = torch.where(total > 0, (w @ v) / total, 0.0)
    out = torch.zeros(q.shape, device=q.device)
    out[row[real]] = y.view(n, hk, most, group, d).transpose(1, 2).flatten(2, 3)[real]
    got = {"out": out.to(q.dtype)}
    if case["lse"]:
        lse = torch.full(q.shape[:2], -math.inf, device=q.device)
        lse[row[real]] = (top + total.log()).view(n, hk, most, group).transpose(1, 2).flatten(2)[real]
        got["lse"] = lse
    return got


# ---- the framework's operators -------------------------------------------------------------------

def own_rotary(s):
    from cqgdn import rotary

    case = s["case"]
    plan = rotary.RotaryPlan(s["turns"], s["axis"], adjacent=case["adjacent"])
    q, k = rotary.rotate(s["q"], s["k"], s["positions"], plan)
    out = {"q": q, "k": k}
    if case["backward"]:
        out["dq"], out["dk"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return out


def own_pages(s):
    from cqgdn import kvcache

    free = s["free"].clone()  # the pool of the state stays as it was, for the next pass
    step = kvcache.step_pages(s["cached"], s["new"], s["tables"], free, s["free_count"], page=s["case"]["page"],
                              tokens=s["tokens"])
    return {"starts": step.starts, "lengths": step.lengths, "admitted": step.admitted, "free_count": step.free_count,
            "free": free, "slots": step.slots, "positions": step.positions, "visible": step.visible,
            "tables": s["tables"]}


def own_write(s):
    from cqgdn import kvcache

    cache = kvcache.KVCache(s["data"], page=s["case"]["page"], head_dim=s["case"]["head_dim"], dtype=s["k"].dtype)
    kvcache.write(cache, s["k"], s["v"], s["slots"])
    k, v = kvcache.read(cache, s["slots"])
    return {"k": k, "v": v}


def own_attend(s):
    from cqgdn import kvcache

    case = s["case"]
    cache = kvcache.KVCache(s["data"], page=case["page"], head_dim=case["head_dim"], dtype=s["q"].dtype)
    out, lse = kvcache.attend(s["q"], cache, s["tables"], s["starts"], s["visible"], window=case["window"] or None,
                              max_queries=s["most"], return_lse=True) if case["lse"] else (
        kvcache.attend(s["q"], cache, s["tables"], s["starts"], s["visible"], window=case["window"] or None,
                       max_queries=s["most"]), None)
    return {"out": out} if lse is None else {"out": out, "lse": lse}


def run(state):
    kind = state["case"]["kind"]
    if own:
        package = str(Path(__file__).resolve().parents[1] / "cq-pretrain_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        return dict(rotary=own_rotary, pages=own_pages, write=own_write, attend=own_attend)[kind](state)
    return dict(rotary=plain_rotary, pages=plain_pages, write=plain_write, attend=plain_attend)[kind](state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    if case["kind"] == "rotary":
        size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        turned = values * case["rotary_dim"] // case["head_dim"]
        passes = 2 if case["backward"] else 1
        return {"bytes": passes * 2 * values * size + 12 * case["tokens"], "flops": passes * 3 * turned}
    if case["kind"] == "pages":
        cached, new = page_lengths(case)
        n, t, page = case["requests"], sum(max(m, 0) for m in new) + case["padding"], case["page"]
        fresh = sum(max(0, -(-(c + m) // page) - -(-c // page)) for c, m in zip(cached, new))
        return {"bytes": 4 * (2 * n + 2 * fresh + 3 * n + 3 * t + 2), "flops": 0}
    if case["kind"] == "write":
        rows = case["tokens"] * case["kv_heads"]
        d = case["head_dim"]
        # the rows in, codes and scales out, and those in and the values out
        return {"bytes": 2 * rows * (2 * 2 * d + 2 * (d // 2 + d // 32)) + 4 * case["tokens"], "flops": 8 * rows * d}
    before, new = lengths(case)
    see, w, d = limits(case), case["window"], case["head_dim"]
    seen = sum(min(x, w) if w else x for x in see)
    held, at = 0, 0
    for m in new:  # what the rows of a request see together
        first, last = see[at], see[at + m - 1]
        held += last - (max(0, first - w) if w else 0)
        at += m
    rows = (len(see) + case["padding"]) * case["heads"]
    return {"bytes": held * case["kv_heads"] * (d + d // 16) + 4 * rows * d + (4 * rows if case["lse"] else 0),
            "flops": 4 * seen * case["heads"] * d}


# ---- the operators' definitions, in 64 bits ------------------------------------------------------

def values64(code, scale):
    """Codes and scale bytes by the formula of the format: (-1)^s 2^(e - 1) (1 + m / 2), without an exponent m / 2."""
    half = torch.stack((code & 15, code >> 4), -1).flatten(-2).double()
    sign, e, m = 1 - 2 * (half >= 8), torch.floor(half / 2) % 4, half % 2
    v = sign * torch.where(e > 0, (1 + m / 2) * 2.0 ** (e - 1), m / 2)
    return v * (2.0 ** (scale.double() - 127)).repeat_interleave(32, -1)


def exact_rotary(case, s):
    out, n = {}, case["rotary_dim"] // 2
    i = torch.arange(n, device=DEV)
    first, second = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + n)
    at = torch.stack([s["positions"][int(a)] for a in s["axis"]], 1).double()
    turn = torch.polar(torch.ones_like(at), at * s["freq"])[:, None]
    for name in ("q", "k", "dq", "dk"):
        if name in s:
            y = s[name].detach().double().clone()
            z = torch.complex(y[..., first], y[..., second]) * (turn.conj() if name[0] == "d" else turn)
            y[..., first], y[..., second] = z.real, z.imag
            out[name] = y
    return out


def exact_write(case, s):
    out, real = {}, s["slots"] >= 0
    grid = torch.tensor(GRID, dtype=torch.float64, device=DEV)
    for name in ("k", "v"):
        x = s[name].double().unflatten(-1, (-1, 32))
        top = x.abs().amax(-1, keepdim=True)
        e = torch.floor(torch.log2(top.clamp(min=2.0**-140))) - 2
        e = torch.where(top * 2.0**-e > 7, e + 1, e).clamp(-125, 127)
        a = (x.abs() * 2.0**-e).unsqueeze(-1)
        far = (a - grid).abs()
        far = far + 1e-9 * (torch.arange(8, device=DEV) % 2)  # halfway: the even code
        y = torch.sign(x) * grid[far.argmin(-1)] * 2.0**e
        out[name] = torch.where(real[:, None, None], y.flatten(-2), 0.0)
    return out


def exact_attend(case, s):
    d, page, hk, w = case["head_dim"], case["page"], case["kv_heads"], case["window"]
    group, starts, see = case["heads"] // hk, s["starts"].tolist(), s["visible"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for r in range(case["requests"]):
        a, b = starts[r], starts[r + 1]
        if a == b:
            continue
        last = max(see[a:b])
        held = s["data"][s["tables"][r, : -(-last // page)].long()]
        limit = s["visible"][a:b].double()[:, None, None]
        at = torch.arange(last, device=DEV)
        for h in range(hk):
            kc, vc, ks, vs = (x.flatten(0, 1)[:last] for x in parts(held[:, h].contiguous(), page, d))
            k, v = values64(kc, ks), values64(vc, vs)
            mine = slice(h * group, (h + 1) * group)
            x = torch.matmul(s["q"][a:b, mine].double(), k.t()) / math.sqrt(d)
            hidden = (at >= limit) | (at < limit - w) if w else at >= limit
            x = x.masked_fill(hidden, -math.inf)
            lse[a:b, mine] = torch.logsumexp(x, -1)
            out[a:b, mine] = torch.matmul(torch.softmax(x, -1), v)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def exact(case, seed):
    if case["kind"] == "pages":
        return None  # whole numbers
    s = prepare(case, seed)
    return dict(rotary=exact_rotary, write=exact_write, attend=exact_attend)[case["kind"]](case, s)
