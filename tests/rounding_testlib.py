"""Inputs that show which numbers of the attention's backward pass are rounded, and how far its gradients may be off there.

All values lie on grids so coarse that q.k and dy.v have no rounding in fp32, whatever the order of their sums.  Keys have a
large value in a dimension where the queries have 0, and queries one where the keys have 0: the scores know nothing of
it, but an error that the dx of a row (of a key) have in common is multiplied by it in dq (dk), where the exact dx of a row
cancel.  Values may have a large one, `shift`, as well: the rounded output is then off by up to half a step of it, which a
delta = dy.out would carry into every dx of the row.

Bounds, with e = 2^-24, n the most keys that a row sees, D the head's dimensions, and X the size of the exponents (scores
and logarithm in units of log2, and the 16 by which weights are held larger at most):
* a weight: the exponent is off by no more than 16 e X (the factor, the product, the logarithm and its way there and back, a
  sum each), the exponential by 2 e, the sum of n weights by n e: off = e (n + 16 X + 16) of itself;
* delta = sum p dp, formed in fp32 from exact dp: (off + (n + 8) e) sum p |dp|;
* dp - delta, a sum of D products and delta: (D + 2) e (sum |dy||v| + |delta|);
* dx = p (dp - delta): its own rounding, u in one term of the type and u^2 in two, and p times the above; in fp16 it is
  held beside the largest dx so far by a power of two that leaves 2^-32 of that one at most;
* dq = scale sum dx k, dk = scale sum dx q: fp32 sums of as many terms as there are."""

import torch

E = 2.0 ** -24


def inputs(docs, hq, hk, D, dtype, shift, seed, device="cpu"):
    """q, k, v, dy, first, limit of packed causal documents."""
    n, g = sum(docs), torch.Generator().manual_seed(seed)
    r = lambda h: torch.randint(-2, 3, (n, h, D), generator=g).float() / 2  # noqa: E731
    q, k, v, dy = r(hq), r(hk), r(hk), r(hq)
    q[..., 0], k[..., 0] = 0.0, 32.0
    q[..., 1], k[..., 1] = 32.0, 0.0
    if shift:
        v[..., 2] += shift
        dy[..., 2] = 1.0
    at = [sum(docs[:i]) for i in range(len(docs))]
    first = torch.tensor([a for a, m in zip(at, docs) for _ in range(m)], dtype=torch.int32)
    limit = torch.arange(1, n + 1, dtype=torch.int32)
    return [x.to(dtype).to(device) for x in (q, k, v, dy)] + [first.to(device), limit.to(device)]


def scale_of(D):
    return 0.0625 if D == 256 else 0.125  # a power of two, so that the factor of a score has one rounding


def head_parts(q, k, v, dy, first, limit, h):
    """float64 parts of one query head, and the mask."""
    at = torch.arange(k.shape[0], device=q.device)
    seen = (at >= first[:, None]) & (at < limit[:, None])
    g = h // (q.shape[1] // k.shape[1])
    return g, q[:, h].double(), k[:, g].double(), v[:, g].double(), dy[:, h].double(), seen


def expected(q, k, v, dy, first, limit, *, terms):
    """dq and dk in float64, and their bounds but for the results' own rounding."""
    D, u, scale = q.shape[2], torch.finfo(q.dtype).eps / 2, scale_of(q.shape[2])
    want = {"dq": torch.zeros_like(q, dtype=torch.float64), "dk": torch.zeros_like(k, dtype=torch.float64)}
    tol = {n: torch.zeros_like(x) for n, x in want.items()}
    for h in range(q.shape[1]):
        g, a, b, c, y, seen = head_parts(q, k, v, dy, first, limit, h)
        x = torch.where(seen, torch.matmul(a, b.t()) * scale, -torch.inf)
        total = torch.logsumexp(x, -1, keepdim=True)
        p, dp = torch.exp(x - total), torch.matmul(y, c.t())
        delta = (p * dp).sum(-1, keepdim=True)
        n = float(seen.sum(-1).max())
        size = 1.4427 * float(torch.where(seen, x.abs() + total.abs(), 0.0).max()) + 16
        off = E * (n + 16 * size + 16)
        dx = p * (dp - delta)
        around = (off + (n + 8) * E) * (p * dp.abs()).sum(-1, keepdim=True)
        reach = torch.matmul(y.abs(), c.abs().t()) + delta.abs()
        wrong = (u ** terms + 2 * E) * dx.abs() + p * (off * (dp - delta).abs() + around + (D + 2) * E * reach)
        if q.dtype == torch.float16:
            wrong = wrong + seen * 2.0 ** -32 * float(dx.abs().max())
        wrong = wrong + (p.shape[0] + 8) * E * dx.abs()  # the last sums
        want["dq"][:, h] = torch.matmul(dx, b) * scale
        tol["dq"][:, h] = torch.matmul(wrong, b.abs()) * scale
        want["dk"][:, g] += torch.matmul(dx.t(), a) * scale
        tol["dk"][:, g] += torch.matmul(wrong.t(), a.abs()) * scale
    return want, tol


def excess(got, want, tol):
    """How far the gradients are off, in units of their bounds (half a step of their own type included)."""
    u = torch.finfo(got.dtype).eps / 2
    bound = tol * (1 + 2 ** -6) + u * want.abs() * (1 + 2 ** -6) + torch.finfo(got.dtype).smallest_normal
    return float(((got.double() - want).abs() / bound).max())


def backward(q, k, v, dy, first, limit, *, terms, delta_from_out=False):
    """dq and dk as kernels form them that hold weights, dp and delta in fp32 and dx in `terms` terms of the type; or with
    delta = dy.out of the rounded out."""
    scale, dtype = scale_of(q.shape[2]), q.dtype
    dq, dk = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(k, dtype=torch.float64)
    for h in range(q.shape[1]):
        g, a, b, c, y, seen = head_parts(q, k, v, dy, first, limit, h)
        x = torch.where(seen, torch.matmul(a, b.t()) * scale, -torch.inf).float()
        p, dp = torch.softmax(x, -1), torch.matmul(y, c.t()).float()
        delta = (p * dp).sum(-1, keepdim=True)
        if delta_from_out:
            out = torch.matmul(p.double(), c).to(dtype).double()
            delta = (out * y).sum(-1, keepdim=True).float()
        dx = p * (dp - delta)
        f = 2.0 ** 10 / float(dx.abs().max()) if dtype == torch.float16 else 1.0
        held, left = torch.zeros_like(dx), dx * f
        for _ in range(terms):
            part = left.to(dtype).float()
            held, left = held + part, left - part
        held = held.double() / f
        dq[:, h] = torch.matmul(held, b) * scale
        dk[:, g] += torch.matmul(held.t(), a) * scale
    return {"dq": dq.to(dtype), "dk": dk.to(dtype)}
