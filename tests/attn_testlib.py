"""Plain 64-bit forms of the attention layers' operators, for their tests."""

import decimal
import math

import torch

PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494")


def frequencies(theta, rotary_dim):
    """theta^(-2i / rotary_dim) to 60 digits."""
    with decimal.localcontext() as c:
        c.prec = 60
        return [decimal.Decimal(theta) ** (decimal.Decimal(-2 * i) / rotary_dim) for i in range(rotary_dim // 2)]


GRID = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def rotate_ref(x, positions, freq, axis, adjacent, sign=1.0):
    """x [T, H, D] on the CPU turned in float64; positions [A, T], freq (Decimal) and axis of each pair."""
    y = x.double().clone()
    n = len(freq)
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + n)
        # positions reach 2^40 in the tests: whole turns go in integers, with 120 bits of the frequency
        with decimal.localcontext() as c:
            c.prec = 60
            turn = int(freq[i] / (2 * PI) * 2 ** 120)
        at = torch.tensor([((int(p) * turn) % 2 ** 120) / 2 ** 120 * 2 * math.pi for p in positions[axis[i]]],
                          dtype=torch.float64)[:, None]
        u, v = x[..., a].double(), x[..., b].double()
        y[..., a] = u * at.cos() - sign * v * at.sin()
        y[..., b] = v * at.cos() + sign * u * at.sin()
    return y


def encode_ref(x):
    """The values the cache holds for x [..., D] (float64), NaN for blocks that are not finite."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    part, e = torch.frexp(torch.where(fine, top, 1.0))
    s = torch.where(part > 0.875, e - 2, e - 3).clamp(-125, 13 if x.dtype == torch.float16 else 125)
    y = torch.ldexp(torch.where(fine, b, 0.0), -s)
    far = (y.abs().unsqueeze(-1) - GRID.to(x.device)).abs()
    best = far.amin(-1, keepdim=True)
    # halfway between two codes: the even one
    even = torch.where(far == best, torch.arange(8, device=x.device) % 2, 2).argmin(-1)
    v = torch.ldexp(torch.sign(y) * GRID.to(x.device)[even], s)
    return torch.where(fine, v, math.nan).flatten(-2)


def pages_ref(cached, new, tables, free, free_count, page, tokens):
    """step_pages on lists, by its definition; returns a dict of lists (tables and free among them)."""
    up = lambda x: -(-x // page)  # noqa: E731
    n, columns = len(cached), len(tables[0]) if tables else 0
    tables, pool = [list(t) for t in tables], list(free[:max(0, min(free_count, len(free)))])
    starts = [0]
    for m in new:
        starts.append(starts[-1] + max(m, 0))
    for r in range(n):
        if new[r] < 0:
            pool += tables[r][:min(up(max(cached[r], 0)), columns)]
    pool = pool[:len(free)]
    free = pool + list(free[len(pool):])
    count, need, left = len(pool), 0, len(pool)
    lengths, admitted = [], []
    for r in range(n):
        c = max(cached[r], 0)
        if new[r] <= 0:
            lengths.append(0 if new[r] < 0 else c)
            admitted.append(1)
            continue
        fits = c + new[r] <= columns * page and starts[r] + new[r] <= tokens
        mine = up(c + new[r]) - up(c) if fits else 0
        ok = fits and (mine == 0 or need + mine <= count)
        if ok:
            for j in range(mine):
                tables[r][up(c) + j] = pool[count - 1 - need - j]
            left -= mine
        need += mine
        lengths.append(c + new[r] if ok else c)
        admitted.append(int(ok))
    slots, positions, visible = [-1] * tokens, [0] * tokens, [0] * tokens
    for r in range(n):
        for i in range(max(new[r], 0)):
            t, p = starts[r] + i, max(cached[r], 0) + i
            if t >= tokens:
                break
            positions[t] = p
            if admitted[r] and tables[r][p // page] >= 0:
                slots[t] = tables[r][p // page] * page + p % page
                visible[t] = p + 1
    return dict(starts=starts, lengths=lengths, admitted=admitted, free_count=[left], slots=slots,
                positions=positions, visible=visible, tables=tables, free=free)


def attend_ref(q, k, v, starts, visible, scale, window=0, hidden=None):
    """Attention in float64.  k, v [N, L, Hk, D] are each request's positions in order; ``hidden`` bool
    [N, L] marks positions no row sees.  Returns out, lse and the sums of weight * |v| (for tolerances)."""
    t, hq, d = q.shape
    n, length, hk, _ = k.shape
    out, lse = torch.zeros(t, hq, d, dtype=torch.float64), torch.full((t, hq), -math.inf, dtype=torch.float64)
    size = torch.zeros(t, hq, d, dtype=torch.float64)
    for r in range(n):
        for row in range(starts[r], min(starts[r + 1], t)):
            hi = min(max(int(visible[row]), 0), length)
            lo = max(0, hi - window) if window else 0
            at = [p for p in range(lo, hi) if hidden is None or not hidden[r, p]]
            if not at:
                continue
            for h in range(hk):
                mine = slice(h * (hq // hk), (h + 1) * (hq // hk))
                x = q[row, mine].double() @ k[r, at, h].double().t() * scale
                lse[row, mine] = torch.logsumexp(x, -1)
                w = torch.softmax(x, -1)
                out[row, mine] = w @ v[r, at, h].double()
                size[row, mine] = w @ v[r, at, h].double().abs()
    return out, lse, size
