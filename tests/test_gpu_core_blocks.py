"""Gradients of keys that rows of many blocks see: the kernels look for those blocks 64 at a time, each of several parts takes
every n-th, and none may be lost or counted twice where one 64 ends."""

import pytest
import torch

import core_testlib as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def attention(gdn):
    from cqgdn import attention

    return attention


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("few", [False, True])
def test_blocks_beyond_the_first_64_and_128(attention, D, few):
    """148 blocks of 64 rows, all of which see most keys, or two in seven some (`few`)."""
    from cqgdn import _lib

    T, S, hq, hk = 4700, 200, 4, 2
    blocks = -(-T * (hq // hk) // 128) * 2
    need = _lib.lib().cqgdn_attend_bwd_workspace_size(T, S, hq, hk, D)
    parts = (need - (blocks * (1536 * hk + 16) + 255) // 256 * 256) // (2 * S * hk * D * 4)
    assert blocks > 128 and parts > 1
    g = torch.Generator(device=DEV).manual_seed(D)
    q, k, v, dy = (torch.randn(n, h, D, generator=g, device=DEV).bfloat16() for n, h in ((T, hq), (S, hk), (S, hk), (T, hq)))
    t = torch.arange(T, device=DEV)
    if few:
        first = torch.where(t // 32 % 7 < 2, t % 150, S).int()
        limit = (first + 1 + t % 45).clamp(max=S).int()
        seen = int((t // 32 % 7 < 2).view(-1)[:: 32].sum())
        assert seen % parts, "parts of unlike numbers of blocks"
    else:
        first, limit = (t % 3).int(), (S - t % 70).int()
        assert blocks % parts, "parts of unlike numbers of blocks"
    a, b, c = (x.clone().requires_grad_() for x in (q, k, v))
    out = attention.attend(a, b, c, limit, first=first)
    row = torch.arange(T * hq // hk, device=DEV).view(T, hq // hk) // 64
    # all blocks, and one at a time, whose loss would go under in the bounds of all
    for block in [None, 0, parts - 1, parts, 62, 63, 64, 65, 127, 128, 129, blocks - 2]:
        y = dy if block is None else torch.where((row == block).repeat(1, hk)[..., None], dy, 0)
        grads = torch.autograd.grad(out, (a, b, c), y, retain_graph=True)
        want, tol = R.attend_ref(q, k, v, first, limit, scale=D ** -0.5, dy=y)
        for name, got in zip(("dq", "dk", "dv"), grads):
            R.check(got, want[name], tol[name], f"{name} of block {block}", q.dtype)
