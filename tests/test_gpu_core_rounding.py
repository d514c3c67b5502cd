"""What the attention's backward pass rounds, on the GPU: inputs and bounds of rounding_testlib."""

import pytest
import torch

import rounding_testlib as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def attention(gdn):
    from cqgdn import attention

    return attention


def gradients(attention, q, k, v, dy, first, limit):
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    out = attention.attend(q, k, v, limit, first=first, scale=L.scale_of(q.shape[2]))
    dq, dk = torch.autograd.grad(out, (q, k), dy)
    return {"dq": dq, "dk": dk}


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", TYPES)
def test_delta_is_not_that_of_the_rounded_out(attention, dtype, D):
    x = L.inputs([300, 130], 4, 2, D, TYPES[dtype], 64.0, seed=D, device=DEV)
    want, tol = L.expected(*x, terms=1)
    got = gradients(attention, *x)
    for name in want:
        assert L.excess(got[name], want[name], tol[name]) <= 1, name


@pytest.mark.parametrize("D", [64, 128, 256])
def test_dx_has_two_terms_where_a_mask_cuts(attention, D):
    x = L.inputs([63, 5, 2, 40], 4, 2, D, torch.bfloat16, 0.0, seed=D, device=DEV)
    want, tol = L.expected(*x, terms=2)
    got = gradients(attention, *x)
    for name in want:
        assert L.excess(got[name], want[name], tol[name]) <= 1, name
