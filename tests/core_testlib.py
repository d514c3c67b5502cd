"""Plain 64-bit forms of the attention over 16-bit keys and values, with the sums that its tolerances are made of.

Tolerances.  A rounding to a type is off by at most half a step, u = finfo(type).eps / 2 of the value.  Each weight p_j
is rounded once for its product with v, and the result once: |out - exact| <= u (A + |out|), A = sum p_j |v_j|.  Scores are
fp32 sums of D exact products, off by at most (D + 3) 2^-24 of the sum of their magnitudes, the cap by 2^-22 of itself and a
bias by 2^-22 of its size, so a weight's relative error is at most twice that of the scores (`moved`; the row's sum has
its share of it).
The smallest weights are lost: bf16's, and fp32's, exponents end at 2^-126; in fp16 half a step of the smallest numbers is
2^-25, of weights held 2^7 times as large as the row's largest one's 1 (2^15 times in the backward pass), so a weight is
off by that much (`floor`) beside.  A dx below 2^-126 is lost likewise.
In the backward pass delta = dy.out takes the rounded out: off by at most E = sum |dy| u (A + |out|).  dx = p (dp - delta) is
rounded to one term (or `terms`): off by u |dx| (u^terms) + p E + moved p (|dp| + |delta|).  A gradient is the sum of those, times |k| or |q|, and rounded."""

import math

import torch


def scores(q, k, scale, cap, slope, distance, seen):
    """Scores [T, S] of one head in float64, the cap's derivative, and the largest error of the fp32 ones."""
    d = q.shape[1]
    x = torch.matmul(q, k.t()) * scale
    moved = (d + 3) * 2 ** -24 * abs(scale) * torch.matmul(q.abs(), k.abs().t()) + 2 ** -21
    rate = torch.ones_like(x)
    if cap:
        y = torch.tanh(x / cap)
        rate, x = 1 - y * y, cap * y
        moved = moved + cap * 2 ** -21
    if slope is not None:
        x = x - slope * distance
        moved = moved + 2 ** -21 * abs(slope) * distance
    moved = moved + 2 ** -22 * x.abs()
    return x.masked_fill(~seen, -math.inf), rate, torch.where(seen, moved, 0.0)


def attend_ref(q, k, v, first, limit, *, scale, cap=None, slopes=None, positions=None, dy=None, dlse=None, seen=None, terms=1):
    """Attention and its gradients in float64, each with its tolerance (but for the results' own rounding)."""
    T, hq, D = q.shape
    S, hk, _ = k.shape
    u = torch.finfo(q.dtype).eps / 2
    at = torch.arange(S, device=q.device)
    if seen is None:
        seen = (at >= first[:, None]) & (at < limit[:, None])
    stands = (limit.long() - 1 if positions is None else positions.long())[:, None]
    distance = (stands - at).abs().double()
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)  # noqa: E731
    r = dict(out=z(T, hq, D), lse=torch.full((T, hq), -math.inf, dtype=torch.float64, device=q.device), dq=z(T, hq, D),
             dk=z(S, hk, D), dv=z(S, hk, D))
    tol = {n: torch.zeros_like(x) for n, x in r.items()}
    tol["lse"] = z(T, hq)
    floor, floor_back = (2 ** -32, 2 ** -40) if q.dtype == torch.float16 else (2 ** -126, 2 ** -126)
    there = seen.double()
    for h in range(hq):
        g = h // (hq // hk)
        a, b, c = q[:, h].double(), k[:, g].double(), v[:, g].double()
        x, rate, moved = scores(a, b, scale, cap, None if slopes is None else float(slopes[h]), distance, seen)
        total = torch.logsumexp(x, -1) if S else torch.full((T,), -math.inf, dtype=torch.float64, device=q.device)
        p = torch.exp(x - torch.where(total == -math.inf, 0.0, total)[:, None])
        off = 2 * (moved.amax(-1, keepdim=True) if S else z(T, 1))  # of a weight, relative
        r["out"][:, h], r["lse"][:, h] = torch.matmul(p, c), total
        size = torch.matmul(p, c.abs())
        tol["out"][:, h] = (u + off + 2 ** -22) * size + floor * torch.matmul(there, c.abs())
        tol["lse"][:, h] = off[:, 0] + 2 ** -22
        if dy is None:
            continue
        y = dy[:, h].double()
        dp = torch.matmul(y, c.t())
        delta = (y * r["out"][:, h]).sum(-1, keepdim=True)
        more = 0 if dlse is None else dlse[:, h, None].double()
        around = (y.abs() * (u * (size + r["out"][:, h].abs()) + off * size)).sum(-1, keepdim=True)  # of delta
        reach = torch.matmul(y.abs(), c.abs().t()) + (y * r["out"][:, h]).abs().sum(-1, keepdim=True)
        dx = p * (dp - delta + more) * rate
        # the fp32 sums dp and delta, and the cap's derivative, 4 r (1 - r), whose parts are off by 2^-22 each
        dx_off = u ** terms * dx.abs() + there * 2 ** -126 * (1 + reach + abs(more)) + p * (around + (off + (2 * D + 8) * 2 ** -24) * (reach + abs(more)) +
                                     (2 ** -20 if cap else 0) * (dp - delta + more).abs())
        tiny = 2.0 ** -24 * (dx.abs().amax() if dx.numel() else 0)  # fp16: what its power of two leaves of the smallest
        dx_off = torch.where(seen, dx_off + tiny * 2 ** -8, 0.0) if q.dtype == torch.float16 else dx_off
        r["dq"][:, h] = torch.matmul(dx, b) * scale
        tol["dq"][:, h] = torch.matmul(dx_off, b.abs()) * abs(scale)
        r["dk"][:, g] += torch.matmul(dx.t(), a) * scale
        tol["dk"][:, g] += torch.matmul(dx_off.t(), a.abs()) * abs(scale)
        r["dv"][:, g] += torch.matmul(p.t(), y)
        tol["dv"][:, g] += torch.matmul((p * (u + off + 2 ** -22) + there * floor_back).t(), y.abs())
    return r, tol


def check(got, want, tol, name, dtype):
    """got within the sums' tolerance and half a step of the result's own type."""
    u = 2 ** -22 if name == "lse" else torch.finfo(dtype).eps / 2
    tiny = 2 ** -40 if name == "lse" else torch.finfo(dtype).smallest_normal
    got = got.double()
    empty = want == -math.inf
    assert torch.equal(got[empty], want[empty]), name
    err = torch.where(empty, 0.0, got - want).abs()
    bound = tol * (1 + 2 ** -6) + u * torch.where(empty, 0.0, want).abs() * (1 + 2 ** -6) + tiny
    assert bool((err <= bound).all()), (name, float((err / bound).max()), int((err > bound).sum()))
