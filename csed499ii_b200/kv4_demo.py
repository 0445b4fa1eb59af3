"""A small decoder layer that serves requests: 2:4-sparse INT4 projections
around a 4-bit paged key/value cache.

    python -m csed499ii_b200.kv4_demo [--steps 64] [--graph]

Every step is the same five calls whatever the requests do (prompts, single
tokens, requests that end): ``kv4_schedule`` turns the step's token counts into
block tables and slots, the fused projection makes queries, keys and values,
``kv4_append`` writes the cache, ``kv4_attention`` reads it, and the output
projection closes the layer.  Nothing waits for the GPU, so a step of single
tokens can be replayed from a CUDA graph.  Weights and inputs are random.
"""
from __future__ import annotations

import argparse
import time

import torch

from . import Layer_2_4, kv4_append, kv4_attention, kv4_cache, kv4_schedule, kv4_workspace


class _Weight:
    def __init__(self, weight):
        self.weight, self.bias = weight, None


def _projection(k, n, device, generator):
    w = (torch.randn(k, n, device=device, generator=generator) * k**-0.5).half()
    layer = Layer_2_4(k, n, groupsize=128).to(device)
    layer.pack(_Weight(w), (w.view(k // 128, 128, n).abs().amax(1) / 7).half())
    return layer


class CachedAttention:
    """Attention layer of a decoder with its cache and the state of its requests.

    @batch: requests that can run at the same time
    @pages, @page_size: of the cache
    @most: tokens a request can reach
    """

    def __init__(self, hidden, heads, kv_heads, head_dim, batch, pages, page_size=64, most=4096,
                 device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.page_size = heads, kv_heads, head_dim, page_size
        self.qkv = _projection(hidden, (heads + 2 * kv_heads) * head_dim, device, g)
        self.proj = _projection(heads * head_dim, hidden, device, g)
        self.cache = kv4_cache(pages, kv_heads, head_dim, page_size, torch.half, device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.tables = torch.zeros(batch, -(-most // page_size), dtype=torch.int32, device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.count = torch.tensor([pages], dtype=torch.int32, device=device)
        self.workspace = kv4_workspace(device)

    def step(self, x, new_lens, max_new):
        """One step.  ``x``: (rows, hidden), the new tokens of all requests in
        order; ``new_lens``: how many each request adds (-1: it ends).  Returns
        (rows, hidden) and what :func:`kv4_schedule` said."""
        step = kv4_schedule(new_lens, self.lens, self.tables, self.free, self.count, x.shape[0],
                            self.page_size, lens_out=self.lens, free_count_out=self.count)
        q, k, v = self.qkv(x).view(x.shape[0], -1, self.dim).split([self.heads, self.kv_heads, self.kv_heads], 1)
        kv4_append(k, v, self.cache, step.slots)
        y = kv4_attention(q, self.cache, self.tables, step.lens, starts=step.starts, max_new=max_new,
                          workspace=self.workspace)
        return self.proj(y.flatten(1)), step


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=500, help="tokens of the longest prompt")
    ap.add_argument("--graph", action="store_true", help="replay the decoding step from a CUDA graph")
    args = ap.parse_args(argv)
    hidden, heads, kv_heads, dim = 4096, 32, 8, 128
    most = args.prompt + args.steps + 4
    layer = CachedAttention(hidden, heads, kv_heads, dim, args.batch, args.batch * (most // 64 + 1), most=most)
    prompts = torch.randint(1, args.prompt + 1, (args.batch,))
    rows = int(prompts.sum())
    y, step = layer.step(torch.randn(rows, hidden, device="cuda").half(), prompts.int().cuda(), args.prompt)
    assert not step.fate.any()
    one = torch.ones(args.batch, dtype=torch.int32, device="cuda")
    x = y[step.starts[1:].long() - 1].contiguous()

    def decode():
        x.copy_(layer.step(x, one, 1)[0])

    for _ in range(3):  # warm up, and room for what the graph's capture counts as a step
        decode()
    run = decode
    if args.graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            decode()
        run = graph.replay
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(args.steps):
        run()
    torch.cuda.synchronize()
    us = (time.perf_counter() - t0) / args.steps * 1e6
    print(f"{args.batch} requests, {rows} prompt tokens, {int(layer.lens.sum())} in the cache: "
          f"{us:.1f} us a decoding step{' (graph)' if args.graph else ''}, "
          f"{int(layer.count)} pages free")


if __name__ == "__main__":
    main()
