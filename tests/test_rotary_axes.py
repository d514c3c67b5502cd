"""Positions of fewer axes than a plan goes by: one serves them all (text), others are refused (no launch)."""

import pytest
import torch

from cqgdn import rotary


def _call(plan, positions):
    q = torch.zeros(5, 2, 16)
    return rotary.rotate(q, q[:, :1], positions, plan)


@pytest.mark.parametrize("mixed", [False, True])
def test_positions_of_fewer_axes(mixed):
    three = rotary.plan(16, sections=(2, 3, 3), mixed=mixed, device="cpu")
    assert three.axes == 3 and rotary.plan(16, device="cpu").axes == 1
    assert rotary.plan(16, sections=(4, 4, 0), device="cpu").axes == 2  # no pair goes by the third
    with pytest.raises(ValueError, match="positions have 2 axes, the plan 3"):
        _call(three, torch.zeros(2, 5, dtype=torch.int32))
    for shape in ((5,), (1, 5), (3, 5), (4, 5)):  # as far as the device
        with pytest.raises(ValueError, match="ROCm GPU"):
            _call(three, torch.zeros(shape, dtype=torch.int32))
    by_hand = rotary.RotaryPlan(three.turns, three.axis)
    assert by_hand.axes is None
    with pytest.raises(ValueError, match="ROCm GPU"):
        _call(by_hand, torch.zeros(2, 5, dtype=torch.int32))


@pytest.mark.gpu
def test_one_axis_through_a_plan_of_three(gdn):
    p = rotary.plan(64, sections=(8, 12, 12), device="cuda:0")
    q = torch.randn(7, 2, 64, device="cuda:0")
    pos = torch.arange(7, device="cuda:0")
    y, z = rotary.rotate(q, q, pos, p)
    a, b = rotary.rotate(q, q, pos.expand(3, -1), p)
    assert torch.equal(y, a) and torch.equal(z, b)
