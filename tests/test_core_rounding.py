"""The bounds of rounding_testlib tell apart what the attention's backward pass may round from what it may not: forms with
a mistake planted exceed them, the right ones do not."""

import pytest
import torch

import rounding_testlib as L

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_delta_from_the_rounded_out_shows(dtype, D):
    x = L.inputs([300, 130], 4, 2, D, TYPES[dtype], 64.0, seed=D)
    want, tol = L.expected(*x, terms=1)
    right = L.backward(*x, terms=1)
    wrong = L.backward(*x, terms=1, delta_from_out=True)
    for name in want:
        assert L.excess(right[name], want[name], tol[name]) <= 1, name
        assert L.excess(wrong[name], want[name], tol[name]) > 1.2, name


@pytest.mark.parametrize("D", [64, 128, 256])
def test_one_term_of_dx_shows(D):
    x = L.inputs([63, 5, 2, 40], 4, 2, D, torch.bfloat16, 0.0, seed=D)
    want, tol = L.expected(*x, terms=2)
    right, wrong = L.backward(*x, terms=2), L.backward(*x, terms=1)
    for name in want:
        assert L.excess(right[name], want[name], tol[name]) <= 1, name
        assert L.excess(wrong[name], want[name], tol[name]) > 1.2, name
