#!/usr/bin/env python3
"""Serves the attention layers of a small stack: prompts admitted together, then decode steps from a HIP graph.

Each layer projects its hidden rows to queries, keys and values, turns them by their positions, rounds keys and
values into its 4-bit pages and attends over those; one ``step_pages`` a step serves all layers, which share block
tables, slots and limits.  Weights and prompts are random.

Usage: python cq-pretrain_amd/examples/attention_serving.py [--layers 4] [--requests 16] [--prompt 500] [--steps 32]
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from cqgdn import kvcache, rotary  # noqa: E402

HEADS, KV_HEADS, D, PAGE = 16, 4, 128, 64


class Layer:
    def __init__(self, width, pages, generator, device):
        def weight(*shape):
            return (torch.randn(*shape, generator=generator) * shape[0] ** -0.5).to(device, torch.bfloat16)

        self.qkv, self.out = weight(width, (HEADS + 2 * KV_HEADS) * D), weight(HEADS * D, width)
        self.cache = kvcache.KVCache.empty(pages, KV_HEADS, page=PAGE, head_dim=D, device=device)

    def __call__(self, x, step, tables, plan, most):
        rows = (x @ self.qkv).unflatten(1, (-1, D))
        q, k = rotary.rotate(rows[:, :HEADS], rows[:, HEADS:HEADS + KV_HEADS], step.positions, plan)
        kvcache.write(self.cache, k, rows[:, HEADS + KV_HEADS:], step.slots)
        y = kvcache.attend(q, self.cache, tables, step.starts, step.visible, max_queries=most)
        return x + y.flatten(1) @ self.out


class Server:
    """``requests`` sequences of up to ``longest`` tokens, their lengths, tables and pool on the device."""

    def __init__(self, layers, requests, longest, width=512, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        columns = -(-longest // PAGE)
        pages = requests * columns
        self.layers = [Layer(width, pages, g, device) for _ in range(layers)]
        self.plan = rotary.plan(D, theta=1e6, device=device)
        self.cached = torch.zeros(requests, dtype=torch.int32, device=device)
        self.tables = torch.full((requests, columns), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_count = torch.tensor([pages], dtype=torch.int32, device=device)

    def step(self, x, new, most):
        """x [tokens, width]: the new tokens' rows, request after request; new int32 [requests] on the device."""
        step = kvcache.step_pages(self.cached, new, self.tables, self.free, self.free_count, page=PAGE, tokens=x.shape[0],
                                  in_place=True)
        for layer in self.layers:
            x = layer(x, step, self.tables, self.plan, most)
        return x


def serve(layers=4, requests=16, prompt=500, steps=32, width=512, seed=0, device="cuda"):
    """The last hidden rows [requests, width], and the seconds that the prompts and the decode steps took."""
    g = torch.Generator().manual_seed(seed + 1)
    lengths = [prompt - (i * 37) % max(1, prompt // 2) for i in range(requests)]
    server = Server(layers, requests, max(lengths) + steps + 1, width, seed, device)
    x = torch.randn(sum(lengths), width, generator=g).to(device, torch.bfloat16)
    new = torch.tensor(lengths, dtype=torch.int32, device=device)
    torch.cuda.synchronize()
    start = time.perf_counter()
    last = server.step(x, new, max(lengths))[new.cumsum(0) - 1].clone()
    torch.cuda.synchronize()
    first = time.perf_counter() - start

    one = torch.ones_like(new)
    feed = last / last.float().square().mean(-1, keepdim=True).sqrt().bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # the first decode step, before the capture
        feed.copy_(server.step(feed, one, 1))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = server.step(feed, one, 1)
        feed.copy_(y / y.float().square().mean(-1, keepdim=True).sqrt().bfloat16())
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(steps - 1):
        graph.replay()
    torch.cuda.synchronize()
    assert server.cached.tolist() == [n + steps for n in lengths]
    return feed, first, time.perf_counter() - start


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    rows, first, rest = serve(a.layers, a.requests, a.prompt, a.steps)
    print(f"{a.requests} prompts of up to {a.prompt} tokens: {first * 1e3:.2f} ms; a decode step: "
          f"{rest / max(a.steps - 1, 1) * 1e6:.1f} us; finite: {bool(torch.isfinite(rows.float()).all())}")


if __name__ == "__main__":
    main()
