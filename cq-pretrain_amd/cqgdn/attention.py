"""Attention over packed documents for training the attention layers of a hybrid stack.

``attend`` is differentiable and stands between ``rotary.rotate`` and the output projection, as
``events.layer_core`` does in the GDN layers.  Which keys a row sees is a range of its own, which covers packed
documents, causal rows, windows, prefixes and read-only query rows; ``documents`` makes the ranges of the usual
ones.  Everything is enqueued on the current stream; ranges stay on the device.
"""

from __future__ import annotations

import torch

from . import _lib
from .gated_delta_net import CALLS


def documents(bounds, *, causal=True, window=None, prefix=None, device="cuda"):
    """(first, limit) int32 [T] for the rows of packed documents: row t of the document bounds[i] .. bounds[i + 1] - 1
    sees its document's rows up to itself, or all of them if not ``causal``; with ``window`` those of them that lie less
    than ``window`` rows away.  Rows of the first ``prefix[i]`` tokens of document i see the later ones of them too; rows
    before the window stay unseen also there.  Made on the host, once for all layers of a step."""
    bounds = torch.as_tensor([int(b) for b in bounds])
    if bounds.numel() < 1 or int(bounds[0]) != 0 or bool((bounds.diff() < 0).any()):
        raise ValueError("bounds must begin with 0 and not fall")
    if window is not None and window <= 0:
        raise ValueError("window must be positive")
    lengths = bounds.diff()
    if prefix is not None and len(prefix) != lengths.numel():
        raise ValueError("prefix must hold a value a document")
    row = torch.arange(int(bounds[-1]))
    start, end = bounds[:-1].repeat_interleave(lengths), bounds[1:].repeat_interleave(lengths)
    limit = row + 1 if causal else end if window is None else torch.minimum(end, row + window)
    first = start if window is None else torch.maximum(start, row + 1 - window)
    if prefix is not None:
        ends = (bounds[:-1] + torch.as_tensor([int(p) for p in prefix])).repeat_interleave(lengths)
        limit = torch.where(row < ends, torch.maximum(limit, torch.minimum(ends, end)), limit)
    return first.int().to(device), limit.int().to(device)


def attend(q, k, v, limit, *, first=None, positions=None, scale=None, cap=None, slopes=None, return_lse=False):
    """Attention of the rows q [T, Hq, D] to the rows k, v [S, Hk, D] (bf16 or fp16, D = 64, 128 or 256, any strides;
    or [1, T, H, D]).  Row t sees the keys ``first[t]`` (default 0) .. ``limit[t]`` - 1 (int32 [T]; beyond S there are
    none); a row that sees none is zero, one that sees only scores of -infinity NaN.  Query head h reads key head
    h // (Hq // Hk).

    The score of key j is scale q k_j (``scale`` defaults to D^-0.5), capped to cap tanh(score / cap) with ``cap``, less
    ``slopes[h]`` |positions[t] - j| with ``slopes`` (fp32 [Hq], constants; ``positions`` int32 [T] is the key that row t
    stands at, by default limit[t] - 1; beyond 2^24 either way it counts as that, and S may be 2^24 at most).  With
    ``return_lse`` also fp32 [T, Hq]: the logarithm of the sum of exp(score), -inf for rows that see nothing.

    Scores, sums and results are held in fp32, and each weight, and in the backward pass each score's gradient, is
    rounded once to the rows' type for its product (in bf16 a score's gradient to two terms where a range cuts 64 keys).
    The sum p dy.v of a row is formed in fp32 from its keys, not from the rounded result.  A capped score is off by up to
    2^-22 of the cap.  Differentiable in q, k and v, once (a backward pass with ``create_graph`` is refused), through both
    results; the same inputs give the same bits.  A value that is not finite reaches the rows that see it (a gradient's,
    the keys that are seen), and no other."""
    packed = q.dim() == 4 and k.dim() == 4 and v.dim() == 4 and q.shape[0] == k.shape[0] == v.shape[0] == 1
    if packed:
        q, k, v = q[0], k[0], v[0]
    if cap is not None and not cap > 0:
        raise ValueError("cap must be positive and finite")
    CALLS["cqgdn_attend_fwd"] += 1
    out, lse = _lib.ops().attend(q, k, v, limit, first, positions, slopes,
                                 q.shape[-1] ** -0.5 if scale is None else scale, cap or 0.0)
    if packed:
        out, lse = out[None], lse[None]
    return (out, lse) if return_lse else out
