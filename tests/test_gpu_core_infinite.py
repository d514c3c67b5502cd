"""Rows that see keys with scores of -infinity: such keys weigh nothing beside others, and a row that sees no others is NaN
(0 / 0), not zero as one that sees nothing."""

import math

import pytest
import torch

import core_testlib as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def ops(gdn):
    from cqgdn import attention, kvcache

    class Both:
        pass

    Both.attention, Both.kv = attention, kvcache
    return Both


def make(T, S, hq, hk, D, dtype, low):
    """Rows and keys whose first `low` keys have a score of -infinity with every row."""
    g = torch.Generator(device=DEV).manual_seed(T + D)
    q, k, v, dy = (torch.randn(n, h, D, generator=g, device=DEV).to(TYPES[dtype]) for n, h in ((T, hq), (S, hk), (S, hk), (T, hq)))
    q[..., 0] = 1.0
    k[:low, :, 0] = -math.inf
    return q, k, v, dy


def compare(out, lse, q, k, v, first, limit, low, nothing, slopes=None):
    only = ~nothing & (limit.long() <= low)
    assert bool(out[only].isnan().all()) and bool(lse[only].isnan().all()) and bool(only.any())
    assert not bool(out[nothing].any()) and bool((lse[nothing] == -math.inf).all()) and bool(nothing.any())
    rest = ~only & ~nothing
    at = torch.arange(k.shape[0], device=DEV)
    seen = (at >= first[rest][:, None]) & (at < limit[rest][:, None]) & (at >= low)
    finite = k.clone()
    finite[:low, :, 0] = 0
    want, tol = R.attend_ref(q[rest], finite, v, None, limit[rest], scale=q.shape[2] ** -0.5, seen=seen, slopes=slopes)
    R.check(out[rest], want["out"], tol["out"], "out", q.dtype)
    R.check(lse[rest], want["lse"], tol["lse"], "lse", q.dtype)


@pytest.mark.parametrize("S", [150, 2600])  # one part of the keys, and several
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype,bias", [("bf16", False), ("fp16", True)])
def test_packed_rows(ops, dtype, bias, D, S):
    from cqgdn import _lib

    T, hq, hk, low = 90, 4, 2, S * 2 // 3
    assert (_lib.lib().cqgdn_attend_fwd_workspace_size(T, S, hq, hk, D) > 0) == (S > 1000)
    q, k, v, dy = make(T, S, hq, hk, D, dtype, low)
    limit = torch.linspace(1, S, T, device=DEV).int()
    first = (limit // 5).int()
    first[70:] = torch.arange(20, device=DEV).int() * 5
    first[3:90:9] = limit[3:90:9]
    nothing = first >= limit
    slopes = torch.tensor([2.0 ** -8, 0.0, 2.0 ** -7, 2.0 ** -9], device=DEV) if bias else None
    a = q.clone().requires_grad_()
    out, lse = ops.attention.attend(a, k, v, limit, first=first, slopes=slopes, return_lse=True)
    compare(out.detach(), lse.detach(), q, k, v, first, limit, low, nothing, slopes)
    dq, = torch.autograd.grad(out, a, dy)
    only = ~nothing & (limit <= low)
    assert bool(dq[only].isnan().any(-1).all()) and bool(dq[nothing].eq(0).all())


@pytest.mark.parametrize("length", [120, 3000])
@pytest.mark.parametrize("rows", [3, 70])  # the kernels for few and for many rows
@pytest.mark.parametrize("D", [64, 128, 256])
def test_over_the_pages(ops, D, rows, length):
    low, page, hq, hk = length * 2 // 3, 32, 4, 2
    q, k, v, _ = make(rows + 2, length, hq, hk, D, "bf16", low)
    pages = -(-length // page)
    cache = ops.kv.KVCache.empty(pages, hk, page=page, head_dim=D, bits=16, device=DEV)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(length))
    slots = (order[:, None] * page + torch.arange(page)).flatten()[:length].int().to(DEV)
    ops.kv.write(cache, k, v, slots)
    tables = order[None].int().to(DEV)
    visible = torch.cat((torch.linspace(1, length, rows, device=DEV).int(), torch.tensor([0, 9], dtype=torch.int32, device=DEV)))
    starts = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    visible[rows // 2] = 0
    nothing = visible == 0
    nothing[rows:] = True  # behind the last request
    for bound in (rows, 1):
        out, lse = ops.kv.attend(q, cache, tables, starts, visible, max_queries=bound, return_lse=True)
        compare(out, lse, q, k, v, torch.zeros_like(visible), visible, low, nothing)
    # pages that are not there hold no position: a row over them alone sees nothing
    gone = tables.clone()
    gone[:, : low // page + 1] = -1
    out, lse = ops.kv.attend(q, cache, gone, starts, visible, max_queries=rows, return_lse=True)
    away = visible <= (low // page + 1) * page
    assert not bool(out[away].any()) and bool((lse[away] == -math.inf).all())
