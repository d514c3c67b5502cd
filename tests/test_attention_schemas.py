"""What the attention layers' operators say they write, the tensors that a call changes and no others, and that the
cache's pass no gradient (no launch)."""

import pytest
import torch

from cqgdn import _lib, kvcache

WRITTEN = {
    "rotary": set(),
    "step_pages": {"tables", "free"},
    "step_pages_": {"cached", "tables", "free", "free_count"},
    "kv4_write": {"data"},
    "kv4_read": set(),
    "kv4_attend": set(),
}


@pytest.mark.parametrize("name", WRITTEN)
def test_written_arguments(name):
    schema = getattr(_lib.ops(), name).default._schema
    assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == WRITTEN[name]
    assert all(r.alias_info is None for r in schema.returns)  # outputs of their own
    assert not any(a.name == "in_place" for a in schema.arguments)


@pytest.mark.parametrize("in_place", [False, True])
def test_a_step_in_place_takes_the_operator_that_writes(monkeypatch, in_place):
    i = lambda *x: torch.zeros(*x, dtype=torch.int32)  # noqa: E731
    taken = []

    class Ops:
        def __getattr__(self, name):
            def op(*args):
                taken.append((name, len(args)))
                return tuple(i(1) for _ in range(5 if name == "step_pages_" else 7))
            return op

    monkeypatch.setattr(_lib, "ops", lambda: Ops())
    cached, count = i(2), i(1)
    step = kvcache.step_pages(cached, i(2), i(2, 4), i(8), count, page=16, tokens=5, in_place=in_place)
    assert taken == [("step_pages_" if in_place else "step_pages", 7)]
    assert (step.lengths is cached) == (step.free_count is count) == in_place


def test_no_gradient_passes_through_the_cache():
    """The output of rows that require a gradient does not require one itself, so asking for it fails."""
    _lib.ops()
    lib = torch.library.Library("cqgdn", "IMPL")
    lib.impl("kv4_attend", lambda q, *a: (torch.empty_like(q), torch.empty(0, device="meta")), "Meta")
    try:
        i = lambda *x: torch.zeros(*x, dtype=torch.int32, device="meta")  # noqa: E731
        cache = kvcache.KVCache(torch.empty(3, 2, 16 * 68, dtype=torch.uint8, device="meta"), page=16, head_dim=64)
        q = torch.empty(4, 4, 64, dtype=torch.bfloat16, device="meta", requires_grad=True)
        out = kvcache.attend(q, cache, i(2, 3), i(3), i(4))
        assert not out.requires_grad
        with pytest.raises(RuntimeError, match="does not require grad"):
            out.sum().backward()
    finally:
        lib._destroy()
