"""The paged cache of the attention layers of a hybrid stack, in 4 or 16 bits, and the attention that reads it.

A serving step of an attention layer, beside ``events.layer_decode_step`` of the GDN layers:

* ``step_pages``  once a step for all layers: pages for the new tokens, slots, positions and row limits;
* ``append``      the layer's new keys, turned by their positions, and values into its cache, and its queries turned
                  (``write``: keys and values as they are);
* ``attend``      the step's query rows over the pages, one new token a request or a prompt's thousands.

Everything is enqueued on the current stream and sized on the host alone, so a step can be captured into
a HIP graph; lengths, tables and pools stay on the device.  No gradient passes through the cache.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, rotary
from .gated_delta_net import CALLS


class KVCache:
    """Keys and values of one layer, ``page`` tokens a page, a power of two from 16 to 65536; D (``head_dim``) is 64,
    128 or 256; ``dtype`` (bf16 or fp16) is that of the rows written, read and attended with.

    In 4 bits ``data`` is uint8 [pages, heads, page * (D + D / 16)]: blocks of 32 neighbouring values of a head share a
    scale, a power of two; a value is a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6 (include/cqgdn.h gives the layout).
    D = 128 takes 136 bytes a token and head for both.  In 16 bits it is ``dtype`` [pages, heads, 2, page, D], keys
    before values: 512 bytes."""

    def __init__(self, data, *, page, head_dim, dtype=torch.bfloat16):
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("a cache holds bf16 or fp16 rows")
        if data.dtype == dtype:
            if data.dim() != 5 or tuple(data.shape[2:]) != (2, page, head_dim):
                raise ValueError("data must be [pages, heads, 2, page, head_dim]")
        elif data.dim() != 3 or data.dtype != torch.uint8 or data.shape[2] != page * (head_dim + head_dim // 16):
            raise ValueError("data must be uint8 [pages, heads, page * (head_dim + head_dim / 16)]")
        self.data, self.page, self.head_dim, self.dtype = data, page, head_dim, dtype

    @classmethod
    def empty(cls, pages, heads, *, page=64, head_dim=128, dtype=torch.bfloat16, bits=4, device="cuda"):
        """A cache of ``pages`` pages (``pages * page`` tokens) that reads as zeros."""
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if page < 16 or page > 65536 or page & (page - 1):
            raise ValueError("page must be a power of two from 16 to 65536")
        if bits not in (4, 16):
            raise ValueError("bits must be 4 or 16")
        data = (torch.zeros(pages, heads, 2, page, head_dim, dtype=dtype, device=device) if bits == 16 else
                torch.zeros(pages, heads, page * (head_dim + head_dim // 16), dtype=torch.uint8, device=device))
        return cls(data, page=page, head_dim=head_dim, dtype=dtype)

    @property
    def bits(self):
        return 4 if self.data.dtype == torch.uint8 else 16

    @property
    def pages(self):
        return self.data.shape[0]

    @property
    def heads(self):
        return self.data.shape[1]


class PageStep(NamedTuple):
    """What ``step_pages`` returns, int32 on the device."""

    starts: torch.Tensor      # [N + 1] first row of each request among the step's rows
    lengths: torch.Tensor     # [N] tokens each request holds after the step
    admitted: torch.Tensor    # [N] 0 where the request's new tokens found no room
    free_count: torch.Tensor  # [1] pages left in the pool
    slots: torch.Tensor       # [tokens] where each row is written, -1: nowhere
    positions: torch.Tensor   # [tokens] position of each row in its request
    visible: torch.Tensor     # [tokens] positions each row sees: itself and those before it


def step_pages(cached, new, tables, free, free_count, *, page, tokens, in_place=False):
    """The pages of a step, from lengths on the device.

    ``cached`` int32 [N]: tokens each request holds; ``new`` int32 [N]: its tokens of this step (0: none;
    negative: it has ended, and its pages return to the pool); ``tables`` int32 [N, columns]: each
    request's pages in order; ``free`` int32 with ``free_count`` int32 [1]: the pool, a stack.  New pages
    are written into ``tables``, returned ones into ``free``.  ``tokens`` is the size of the step's row
    buffers, at least the sum of the new tokens; rows behind them are padding (slot -1, limit 0).

    A request whose new tokens do not fit the pool, its table row or the buffer is not admitted: it keeps
    what it had and its rows get slot -1 and limit 0.  Pages are taken in the requests' order, and behind
    one that the pool cannot serve none that needs pages is admitted.  With ``in_place`` the lengths and
    the pool's count are written back into ``cached`` and ``free_count``."""
    CALLS["cqgdn_step_pages"] += 1
    if not in_place:
        return PageStep(*_lib.ops().step_pages(cached, new, tables, free, free_count, page, tokens))
    starts, admitted, *rows = _lib.ops().step_pages_(cached, new, tables, free, free_count, page, tokens)
    return PageStep(starts, cached, admitted, free_count, *rows)


def write(cache, k, v, slots):
    """Puts the rows k, v [T, heads, D] (of the cache's type, any strides) into the slots (int32 [T],
    page * page size + offset; -1: not written), rounded to the cache's bits.  No slot may be given twice in a call."""
    if k.dtype != cache.dtype or v.dtype != cache.dtype:
        raise ValueError(f"k and v must be {cache.dtype}, as the cache is")
    if cache.bits == 16:
        CALLS["cqgdn_kv16_append"] += 1
        _lib.ops().kv16_append(None, k, v, None, None, None, False, slots, cache.data)
        return
    CALLS["cqgdn_kv4_write"] += 1
    _lib.ops().kv4_write(cache.data, k, v, slots, cache.page)


def append(cache, q, k, v, positions, plan, slots):
    """``rotary.rotate`` of q [T, Hq, D] and k [T, heads, D] by their tokens' positions, and ``write`` of the turned k
    and of v: returns the turned q.  With a 16-bit cache that is one launch, which writes each row once, and gives
    what the two would, bit for bit; with a 4-bit one it is the two.  No gradient passes."""
    if k.dtype != cache.dtype or v.dtype != cache.dtype or q.dtype != cache.dtype:
        raise ValueError(f"q, k and v must be {cache.dtype}, as the cache is")
    positions = rotary.token_positions(positions, plan)
    if cache.bits == 16:
        CALLS["cqgdn_kv16_append"] += 1
        return _lib.ops().kv16_append(q, k, v, positions, plan.turns, plan.axis, plan.adjacent, slots, cache.data)
    with torch.no_grad():
        q, k = rotary.rotate(q, k, positions, plan)
    write(cache, k, v, slots)
    return q


def read(cache, slots):
    """The keys and values that the slots (int32 [T]) hold, [T, heads, D] of the cache's type each; zeros
    for slots outside the cache."""
    if cache.bits == 16:
        if slots.dim() != 1 or slots.dtype != torch.int32:
            raise ValueError("slots must be an int32 vector")
        inside = (slots >= 0) & (slots < cache.pages * cache.page)
        at = torch.where(inside, slots, 0).long()
        rows = cache.data.new_zeros(slots.numel(), cache.heads, 2, cache.head_dim)
        if cache.pages:
            rows = torch.where(inside[:, None, None, None], cache.data[at // cache.page, :, :, at % cache.page], rows)
        return rows[:, :, 0].contiguous(), rows[:, :, 1].contiguous()
    CALLS["cqgdn_kv4_read"] += 1
    return _lib.ops().kv4_read(cache.data, slots, cache.page, cache.head_dim, cache.dtype == torch.float16)


def attend(q, cache, tables, starts, visible, *, window=None, scale=None, cap=None, slopes=None, positions=None,
           max_queries=None, return_lse=False):
    """Attention of the rows q [T, Hq, D] over the cached positions of their requests.

    Rows starts[r] .. starts[r + 1] - 1 (from 0 on) are request r's, whose pages are ``tables[r]``; row t sees the
    first ``visible[t]`` positions, or the last ``window`` of those.  Query head h reads key head
    h // (Hq // heads).  ``scale`` defaults to D^-0.5.  Rows that see nothing, and rows behind
    ``starts[-1]``, are zero.  Positions whose table entry names no page are not seen.  Rows need not be those
    that the step has written: read-only rows take starts and limits of their own.

    Scores, sums and results are held in fp32; each weight is rounded to the cache's type before the product
    with v, which moves a result by up to half a step of the type times sum p |v| / sum p.

    Over a 16-bit cache scores may be capped and biased as in ``attention.attend``: cap tanh(score / cap) with ``cap``, less
    ``slopes[h]`` |positions[t] - j| at position j with ``slopes`` (fp32 [Hq]; ``positions`` int32 [T], default
    visible - 1, where the row's last position is).  A value that is not finite reaches only rows that see it; a row that
    sees only scores of -infinity is NaN.

    ``max_queries`` bounds the rows of one request and sets the launch (default: T; a decode step should
    pass 1): a larger request is still served.  With ``return_lse`` also fp32 [T, Hq]:
    log sum exp(scale q k), -inf for rows that see nothing."""
    if q.dtype != cache.dtype:
        raise ValueError(f"q must be {cache.dtype}, as the cache is")
    if window is not None and window <= 0:
        raise ValueError("window must be positive")
    if q.shape[-1] != cache.head_dim:
        raise ValueError(f"q must be [T, heads, {cache.head_dim}], as the cache is")
    if cap is not None and not cap > 0:
        raise ValueError("cap must be positive and finite")
    scale = cache.head_dim ** -0.5 if scale is None else scale
    max_queries = max(1, q.shape[0]) if max_queries is None else max_queries
    if cache.bits == 16:
        CALLS["cqgdn_kv16_attend"] += 1
        out, lse = _lib.ops().kv16_attend(q, cache.data, tables, starts, visible, positions, slopes, window or 0, scale,
                                          cap or 0.0, max_queries, return_lse)
        return (out, lse) if return_lse else out
    if cap is not None or slopes is not None or positions is not None:
        raise ValueError("capped or biased scores need a 16-bit cache")
    CALLS["cqgdn_kv4_attend"] += 1
    out, lse = _lib.ops().kv4_attend(q, cache.data, tables, starts, visible, cache.page, window or 0, scale, max_queries,
                                     return_lse)
    return (out, lse) if return_lse else out
