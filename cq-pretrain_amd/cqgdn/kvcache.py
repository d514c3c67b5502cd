"""The paged 4-bit cache of the attention layers of a hybrid stack, and the attention that reads it.

A serving step of an attention layer, beside ``events.layer_decode_step`` of the GDN layers:

* ``step_pages``  once a step for all layers: pages for the new tokens, slots, positions and row limits;
* ``write``       the layer's new keys and values into its cache;
* ``attend``      the step's query rows over the pages, one new token a request or a prompt's thousands.

Everything is enqueued on the current stream and sized on the host alone, so a step can be captured into
a HIP graph; lengths, tables and pools stay on the device.  No gradient passes through the cache.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .gated_delta_net import CALLS


class KVCache:
    """Keys and values of one layer in 4 bits: ``data`` uint8 [pages, heads, page * (D + D / 16)].

    Blocks of 32 neighbouring values of a head share a scale, a power of two; a value is a sign and one
    of 0, .5, 1, 1.5, 2, 3, 4, 6 (include/cqgdn.h gives the layout).  ``page`` tokens a page, a power
    of two from 16 to 65536; D (``head_dim``) is 64, 128 or 256; ``dtype`` (bf16 or fp16) is that of
    the rows written, read and attended with.  D = 128 takes 136 bytes a token and head for both."""

    def __init__(self, data, *, page, head_dim, dtype=torch.bfloat16):
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("a 4-bit cache holds bf16 or fp16 rows")
        if data.dim() != 3 or data.dtype != torch.uint8 or data.shape[2] != page * (head_dim + head_dim // 16):
            raise ValueError("data must be uint8 [pages, heads, page * (head_dim + head_dim / 16)]")
        self.data, self.page, self.head_dim, self.dtype = data, page, head_dim, dtype

    @classmethod
    def empty(cls, pages, heads, *, page=64, head_dim=128, dtype=torch.bfloat16, device="cuda"):
        """A cache of ``pages`` pages (``pages * page`` tokens) that reads as zeros."""
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if page < 16 or page > 65536 or page & (page - 1):
            raise ValueError("page must be a power of two from 16 to 65536")
        return cls(torch.zeros(pages, heads, page * (head_dim + head_dim // 16), dtype=torch.uint8, device=device),
                   page=page, head_dim=head_dim, dtype=dtype)

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
    """Rounds the rows k, v [T, heads, D] (of the cache's type, any strides) into the slots (int32 [T],
    page * page size + offset; -1: not written).  No slot may be given twice in a call."""
    if k.dtype != cache.dtype or v.dtype != cache.dtype:
        raise ValueError(f"k and v must be {cache.dtype}, as the cache is")
    CALLS["cqgdn_kv4_write"] += 1
    _lib.ops().kv4_write(cache.data, k, v, slots, cache.page)


def read(cache, slots):
    """The keys and values that the slots (int32 [T]) hold, [T, heads, D] of the cache's type each; zeros
    for slots outside the cache."""
    CALLS["cqgdn_kv4_read"] += 1
    return _lib.ops().kv4_read(cache.data, slots, cache.page, cache.head_dim, cache.dtype == torch.float16)


def attend(q, cache, tables, starts, visible, *, window=None, scale=None, max_queries=None, return_lse=False):
    """Attention of the rows q [T, Hq, D] over the cached positions of their requests.

    Rows starts[r] .. starts[r + 1] - 1 (from 0 on) are request r's, whose pages are ``tables[r]``; row t sees the
    first ``visible[t]`` positions, or the last ``window`` of those.  Query head h reads key head
    h // (Hq // heads).  ``scale`` defaults to D^-0.5.  Rows that see nothing, and rows behind
    ``starts[-1]``, are zero.  Positions whose table entry names no page are not seen.  Rows need not be those
    that the step has written: read-only rows take starts and limits of their own.

    Scores, sums and results are held in fp32; each weight is rounded to the cache's type before the product
    with v, which moves a result by up to half a step of the type times sum p |v| / sum p.

    ``max_queries`` bounds the rows of one request and sets the launch (default: T; a decode step should
    pass 1): a larger request is still served.  With ``return_lse`` also fp32 [T, Hq]:
    log sum exp(scale q k), -inf for rows that see nothing."""
    if q.dtype != cache.dtype:
        raise ValueError(f"q must be {cache.dtype}, as the cache is")
    if window is not None and window <= 0:
        raise ValueError("window must be positive")
    if q.shape[-1] != cache.head_dim:
        raise ValueError(f"q must be [T, heads, {cache.head_dim}], as the cache is")
    CALLS["cqgdn_kv4_attend"] += 1
    out, lse = _lib.ops().kv4_attend(q, cache.data, tables, starts, visible, cache.page, window or 0,
                                     cache.head_dim ** -0.5 if scale is None else scale,
                                     max(1, q.shape[0]) if max_queries is None else max_queries, return_lse)
    return (out, lse) if return_lse else out
