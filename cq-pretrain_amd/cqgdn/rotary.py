"""Rotary positions with several axes (time, height, width) for the attention layers of a hybrid stack.

``plan`` makes the table of a model's frequencies once; ``rotate`` turns the queries and keys of a call
by their tokens' positions and is differentiable in both.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from decimal import Decimal, localcontext

import torch

from . import _lib
from .gated_delta_net import CALLS

_PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494")


@dataclass(frozen=True)
class RotaryPlan:
    """The frequencies of a model's rotary positions, on the GPU.

    ``turns`` int64 [rotary_dim / 2]: how far a position turns pair i, in units of 2^-64 of a turn, so
    that the angle of any integer position is exact; ``axis`` int32 [rotary_dim / 2]: which of the
    position's axes pair i goes by; ``adjacent``: pair i is (2i, 2i + 1), else (i, i + rotary_dim / 2);
    ``axes``: how many axes the pairs go by (None: not known on the host).
    """

    turns: torch.Tensor
    axis: torch.Tensor
    adjacent: bool = False
    axes: int | None = None


def plan(rotary_dim, *, theta=10000.0, sections=None, mixed=False, adjacent=False, device="cuda"):
    """The plan of frequencies theta^(-2i / rotary_dim), i < rotary_dim / 2.

    ``sections`` gives the number of pairs that each axis turns (time, height, width, ...), one after
    the other; with ``mixed`` the axes take turns over the frequencies, each until its pairs are used
    up.  Without sections there is one axis."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim={rotary_dim} must be positive and even")
    if not theta > 1 or math.isinf(theta):
        raise ValueError(f"theta={theta} must be finite and over 1")
    pairs = rotary_dim // 2
    sections = (pairs,) if sections is None else tuple(int(s) for s in sections)
    if not sections or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError(f"sections={sections} must be counts that sum to rotary_dim / 2 = {pairs}")
    if mixed:
        left, axis = list(sections), []
        while len(axis) < pairs:
            for a, n in enumerate(left):
                if n:
                    axis.append(a)
                    left[a] -= 1
    else:
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    with localcontext() as c:
        c.prec = 50
        step = Decimal(theta) ** (Decimal(-2) / Decimal(rotary_dim))
        turns = [int((step ** i / (2 * _PI) * 2 ** 64).to_integral_value()) for i in range(pairs)]
    return RotaryPlan(torch.tensor(turns, dtype=torch.int64).to(device), torch.tensor(axis, dtype=torch.int32).to(device),
                      bool(adjacent), max(axis) + 1)


def rotate(q, k, positions, plan):
    """q [T, Hq, D] and k [T, Hk, D] (bf16, fp16 or fp32, any strides; or [1, T, H, D]) turned by the
    positions of their tokens: int32 or int64 [axes, T], or [T] (or [1, T]) for text, whose axes are
    alike.  Values of a head behind the plan's rotary_dim pass unchanged.  Computed in fp32, rounded once; differentiable in q and k."""
    packed = q.dim() == 4 and k.dim() == 4 and q.shape[0] == 1 and k.shape[0] == 1
    if packed:
        q, k = q[0], k[0]
    if positions.dim() == 1:
        positions = positions[None]
    if plan.axes is not None and 1 < positions.shape[0] < plan.axes:
        raise ValueError(f"positions have {positions.shape[0]} axes, the plan {plan.axes}")
    CALLS["cqgdn_rotary"] += 1
    q, k = _lib.ops().rotary(q, k, positions, plan.turns, plan.axis, plan.adjacent, False)
    return (q[None], k[None]) if packed else (q, k)
