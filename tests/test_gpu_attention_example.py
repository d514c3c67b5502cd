"""The example that runs the attention layers' operators together, against the same steps without a cache."""

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = Path(__file__).resolve().parents[1] / "cq-pretrain_amd" / "examples" / "attention_serving.py"


def _example():
    spec = importlib.util.spec_from_file_location("attention_serving", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_serves_and_repeats(gdn):
    ex = _example()
    a, _, _ = ex.serve(layers=2, requests=5, prompt=90, steps=6, width=128)
    b, _, _ = ex.serve(layers=2, requests=5, prompt=90, steps=6, width=128)
    assert a.shape == (5, 128) and bool(torch.isfinite(a.float()).all()) and torch.equal(a, b)


def test_prompt_at_once_and_token_by_token_agree(gdn):
    """A prompt in one step, and the same prompt one token a step, take the same pages and give rows whose
    difference is that of roundings: bf16 projections and weights, u = 2^-8 of a row's size each, some ten of them
    one after another."""
    ex = _example()
    n = 70
    g = torch.Generator().manual_seed(5)
    x = torch.randn(n, 128, generator=g).to("cuda", torch.bfloat16)
    whole, parts = ex.Server(2, 1, n, width=128), ex.Server(2, 1, n, width=128)
    count = lambda k: torch.tensor([k], dtype=torch.int32, device="cuda")  # noqa: E731
    a = whole.step(x, count(n), n)
    b = torch.cat([parts.step(x[i:i + 1], count(1), 1) for i in range(n)])
    assert whole.cached.tolist() == parts.cached.tolist() == [n]
    assert torch.equal(whole.tables, parts.tables) and torch.equal(whole.free_count, parts.free_count)
    size = a.float().square().mean().sqrt()
    assert float((a.float() - b.float()).square().mean().sqrt()) <= 10 * 2 ** -8 * float(size)
