"""Derivatives of ``rotary.rotate``: that those in forward mode are there and which rows a gradient turns, on tensors
without storage (no launch), and values on the GPU, where a turn's derivative is the turn of the tangents."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from cqgdn import _lib, rotary

DEV = "cuda:0"


@pytest.fixture(scope="module")
def meta():
    """The operator for tensors without storage, for these tests: what its outputs look like."""
    _lib.ops()
    lib = torch.library.Library("cqgdn", "IMPL")
    heads = []  # of each call's q and k

    def rotary(q, k, *a):
        heads.append((q.shape[1], k.shape[1]))
        return torch.empty(q.shape, dtype=q.dtype, device="meta"), torch.empty(k.shape, dtype=k.dtype, device="meta")

    lib.impl("rotary", rotary, "Meta")
    yield heads
    lib._destroy()


def _inputs(device, dtype=torch.float32):
    g = torch.Generator().manual_seed(0)
    p = rotary.plan(32, sections=(4, 6, 6), mixed=True, device="cpu")
    p = rotary.RotaryPlan(p.turns.to(device), p.axis.to(device), p.adjacent)
    q, k, tq, tk = (torch.randn(9, h, 64, generator=g).to(device, dtype) for h in (2, 1, 2, 1))
    return p, q, k, tq, tk, torch.randint(0, 900, (3, 9), generator=g).int().to(device)


def _tangents(f, q, k, tq, tk):
    with fwAD.dual_level():
        y, z = f(q if tq is None else fwAD.make_dual(q, tq), k if tk is None else fwAD.make_dual(k, tk))
        (py, dy), (pz, dz) = fwAD.unpack_dual(y), fwAD.unpack_dual(z)
    return py, pz, dy, dz


@pytest.mark.parametrize("reverse", [(), ("q",), ("k",), ("q", "k")])
def test_tangents_are_there(meta, reverse):
    p, q, k, tq, tk, pos = _inputs("meta")
    q.requires_grad_("q" in reverse)
    k.requires_grad_("k" in reverse)
    for a, b in ((tq, tk), (tq, None), (None, tk)):
        y, z, dy, dz = _tangents(lambda u, v: rotary.rotate(u, v, pos, p), q, k, a, b)
        assert (dy is None) == (a is None) and (dz is None) == (b is None)
        assert (dy is None or dy.shape == q.shape) and (dz is None or dz.shape == k.shape)
        if reverse:
            assert y.requires_grad or z.requires_grad
    calls = []

    def f(u):
        calls.append(1)
        return rotary.rotate(u, k.detach(), pos, p)[0]

    y, dy = torch.func.jvp(f, (q.detach(),), (tq,))
    assert y.shape == dy.shape == q.shape and calls


def test_a_gradient_turns_what_has_one(meta):
    """The output of an input without a gradient needs none, and a backward call turns the gradients that came."""
    p, q, k, _, _, pos = _inputs("meta")
    q.requires_grad_()
    y, z = rotary.rotate(q, k, pos, p)
    assert y.requires_grad and not z.requires_grad
    del meta[:]
    torch.autograd.grad(y, q, torch.empty_like(y))
    assert meta == [(2, 0)]
    y, z = rotary.rotate(k, q, pos, p)
    assert z.requires_grad and not y.requires_grad
    del meta[:]
    torch.autograd.grad(z, q, torch.empty_like(z))
    assert meta == [(0, 2)]
    k.requires_grad_()
    y, z = rotary.rotate(q, k, pos, p)
    del meta[:]
    dq, dk = torch.autograd.grad(y, (q, k), torch.empty_like(y))  # z has no part in it
    assert meta == [(2, 0)] and dq.shape == q.shape and dk.shape == k.shape
    y, z = rotary.rotate(q, k, pos, p)
    del meta[:]
    torch.autograd.grad((y, z), (q, k), (torch.empty_like(y), torch.empty_like(z)))
    assert meta == [(2, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("used", ["y", "z", "yz"])
@pytest.mark.parametrize("wanted", ["q", "k", "qk"])
def test_gradients_of_some_inputs_from_some_outputs(gdn, used, wanted):
    """As with both: a gradient is the same whatever else is asked for, and zeros where nothing comes in."""
    p, q, k, w, v, pos = _inputs(DEV)
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    want = dict(zip("qk", torch.autograd.grad(rotary.rotate(a, b, pos, p), (a, b), (w, v))))
    q.requires_grad_("q" in wanted)
    k.requires_grad_("k" in wanted)
    out = dict(zip("yz", rotary.rotate(q, k, pos, p)))
    assert out["y"].requires_grad == ("q" in wanted) and out["z"].requires_grad == ("k" in wanted)
    pairs = [(out[n], g) for n, g in (("y", w), ("z", v)) if n in used and out[n].requires_grad]
    if not pairs:
        return
    got = torch.autograd.grad([x for x, _ in pairs], [dict(q=q, k=k)[n] for n in wanted], [g for _, g in pairs])
    for n, x in zip(wanted, got):
        assert torch.equal(x, want[n] if dict(q="y", k="z")[n] in used else torch.zeros_like(x))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reverse", [False, True])
def test_tangents_are_turned(gdn, dtype, reverse):
    """The turn of a tangent is computed as the turn of an input is: equal to it."""
    p, q, k, tq, tk, pos = _inputs(DEV, dtype)
    ref = rotary.rotate(q, k, pos, p)
    turned = rotary.rotate(tq, tk, pos, p)
    q.requires_grad_(reverse)
    for a, b in ((tq, tk), (tq, None), (None, tk)):
        y, z, dy, dz = _tangents(lambda u, v: rotary.rotate(u, v, pos, p), q, k, a, b)
        assert torch.equal(y, ref[0]) and torch.equal(z, ref[1])
        assert dy is None if a is None else torch.equal(dy, turned[0])
        assert dz is None if b is None else torch.equal(dz, turned[1])
        if reverse:  # the gradient beside the tangent
            assert torch.equal(torch.autograd.grad(y, q, tq)[0], torch.autograd.grad(rotary.rotate(q, k, pos, p)[0], q, tq)[0])
    y, dy = torch.func.jvp(lambda u: rotary.rotate(u, k, pos, p)[0], (q.detach(),), (tq,))
    assert torch.equal(y, ref[0]) and torch.equal(dy, turned[0])


@pytest.mark.gpu
def test_tangent_of_a_gradient(gdn):
    """Forward over reverse: the gradient is linear in what comes in, and its tangent the turn back of that's."""
    p, q, k, w, tk, pos = _inputs(DEV)
    q.requires_grad_()
    y, _ = rotary.rotate(q, k, pos, p)
    t = torch.randn_like(w)
    with fwAD.dual_level():
        (dq,) = torch.autograd.grad(y, q, fwAD.make_dual(w, t), create_graph=True)
        got = fwAD.unpack_dual(dq).tangent
    (want,) = torch.autograd.grad(rotary.rotate(q, k, pos, p)[0], q, t)
    assert got is not None and torch.equal(got, want)


@pytest.mark.gpu
def test_derivative_against_differences(gdn):
    """The map is linear, so a difference has roundings only.  A turn is off by at most 6 steps of 2^-24 of its pair's
    |a| + |b| <= 2 M (M the largest value) and half a step of a result of at most sqrt(2) M; the sums q +- h t are off
    by half a step of M each and turn into sqrt(2) of that."""
    p, q, k, tq, tk, pos = _inputs(DEV)
    _, _, dy, _ = _tangents(lambda u, v: rotary.rotate(u, v, pos, p), q, k, tq, tk)
    h, u = 0.25, 2 ** -24
    plus, minus = (rotary.rotate(q + x * tq, k, pos, p)[0].double() for x in (h, -h))
    most = float((q.abs() + h * tq.abs()).max())
    bound = 2 * (12 + 2 * 2 ** 0.5) * u * most / (2 * h) + (12 + 2 ** 0.5) * u * float(tq.abs().max())
    assert float(((plus - minus) / (2 * h) - dy.double()).abs().max()) <= bound
