"""Decoding that never ends from a cache that does not grow: a decode step captured once and replayed, its page tables built on the GPU.

A toy decoder of a few attention layers (random projections of a hidden state, no feed-forward) reads its streams' prompts in one step and
then replays one captured decode step.  Every replay lays the step out on the device (streams advance, take a page where they enter one and
give back what left the window), stores the new keys and values by slot map and attends over the window and the first positions; the host
only launches.  At the end the memory held is what it was after the first window.

    python examples/endless_stream.py --streams 16 --steps 20000 --window 1024 --first 4
"""
import argparse
import math
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from lastengine_b200.cache import StreamCache
from lastengine_b200.ops import kernels


class Decoder:
    def __init__(self, layers: int, hidden: int, heads: int, kv_heads: int, dim: int, device, seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)
        rand = lambda rows, cols: (torch.randn(rows, cols, generator=g, device=device) / math.sqrt(cols)).to(torch.bfloat16)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.w_in = [rand((heads + 2 * kv_heads) * dim, hidden) for _ in range(layers)]
        self.w_out = [rand(hidden, heads * dim) for _ in range(layers)]
        self.norm = torch.ones(hidden, device=device)

    def step(self, cache: StreamCache, step, x: torch.Tensor) -> None:
        """x [rows, hidden] float: the rows' hidden state, in place."""
        rows, q, k = x.shape[0], self.heads * self.dim, self.kv_heads * self.dim
        h = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
        proj = torch.empty((rows, q + 2 * k), dtype=torch.bfloat16, device=x.device)
        queries = torch.empty((rows, q), dtype=torch.bfloat16, device=x.device)
        out = torch.empty((rows, q), dtype=torch.bfloat16, device=x.device)
        cache.begin(step)
        for layer, (w_in, w_out) in enumerate(zip(self.w_in, self.w_out)):
            kernels.rmsnorm(h, x, self.norm, 1e-5)
            kernels.linear(proj, h, w_in)
            cache.store(layer, step, proj[:, q:q + k], proj[:, q + k:])
            queries.copy_(proj[:, :q])
            cache.attend(layer, step, out, queries, self.heads)
            kernels.linear(x, out, w_out, kernels.ACCUMULATE)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--streams", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--steps", type=int, default=5000)
    ap.add_argument("--window", type=int, default=1024)
    ap.add_argument("--first", type=int, default=4)
    ap.add_argument("--layers", type=int, default=4)
    a = ap.parse_args()
    dev = torch.device("cuda")
    model = Decoder(a.layers, 1024, 16, 4, 64, dev)
    pages = -(-a.first // 64) + -(-a.window // 64) + 1 + -(-a.prompt // 64)
    cache = StreamCache(a.layers, 4, 64, max_seqs=a.streams, max_tokens=64 * pages * a.streams, max_len=a.prompt + a.steps + 8,
                        window=a.window, first=a.first, device=dev)
    slots = [cache.open() for _ in range(a.streams)]

    prompt = cache.plan(a.streams, a.streams * a.prompt, a.prompt, max_kvlen=a.prompt)
    prompt.set(slots, [a.prompt] * a.streams)
    x = torch.randn(a.streams * a.prompt, 1024, device=dev)
    model.step(cache, prompt, x)
    cache.check()

    token = cache.plan(a.streams, a.streams, 1)
    token.set(slots, [1] * a.streams)
    x = x.view(a.streams, a.prompt, 1024)[:, -1].contiguous()      # the last rows' state goes on as the next ones' input
    model.step(cache, token, x)                                    # once outside the graph
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.step(cache, token, x)
        x.mul_(0.5)                                                # (keeps the toy's state bounded)
    held = []
    t0 = time.perf_counter()
    for i in range(a.steps):
        graph.replay()
        if i % max(1, a.steps // 8) == 0:
            held.append(int((cache.pages >= 0).sum()))
    torch.cuda.synchronize()
    dt = time.perf_counter() - t0
    cache.check()
    print(f"{a.streams} streams, {a.layers} layers: {a.steps} steps in {dt:.2f} s, {a.streams * a.steps / dt:.0f} tokens/s; "
          f"each holds {cache.lengths(slots)[0]} positions' count, pages held over time {held}")
    cache.close(slots)
    if int(cache.counts[0]) != cache.free.numel() or not bool(torch.isfinite(x).all()):
        raise SystemExit("pages were lost, or the state is not finite")


if __name__ == "__main__":
    main()
