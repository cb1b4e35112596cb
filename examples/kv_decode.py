#!/usr/bin/env python3
"""A decoder layer's attention block with a paged key-value cache that is held at
a budget: QKV projection (W4A16), append, attention of the new tokens, O
projection, and once a row is longer than its budget, eviction by accumulated
attention weight.

    python examples/kv_decode.py [--rows 16] [--prompt 512] [--steps 64] [--budget 384] [--dtype int8]

Sizes are those of a Llama-3-8B-shaped layer (hidden 4096, 32 query heads, 8
key-value heads of 128), weights and activations random.
"""
import argparse
import os
import sys
import time

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sneppx-alg_amd"))

import sneppx_quant  # noqa: E402
import torch  # noqa: E402


class AttentionBlock:
    """QKV, cache, attention and O projection of `rows` sequences.  The lengths
    are known on the host without asking the device: every step adds one token
    to a row, and an eviction leaves min(length, budget)."""

    def __init__(self, lib, rows, capacity, budget, recent, hidden=4096, q_heads=32, kv_heads=8, dim=128,
                 page=16, dtype="bf16", seed=0, device="cuda"):
        self.lib, self.rows, self.budget, self.recent, self.dim = lib, rows, budget, recent, dim
        self.q_heads, self.kv_heads, self.capacity = q_heads, kv_heads, capacity
        g = torch.Generator(device=device).manual_seed(seed)
        self.qkv_w = self._weights(g, (q_heads + 2 * kv_heads) * dim, hidden)
        self.o_w = self._weights(g, hidden, q_heads * dim)
        width = -(-capacity // page)
        self.cache = lib.kv_cache(rows * width, page, kv_heads, dim, dtype, weights=True, positions=True, device=device)
        self.tables = torch.arange(rows * width, dtype=torch.int32, device=device).view(rows, width)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=device)
        self.kept = torch.zeros_like(self.lengths)      # the eviction's lengths
        self.next_pos = torch.zeros_like(self.lengths)
        self.held = [0] * rows                          # what lengths holds
        self.out = torch.empty((rows, q_heads, dim), dtype=torch.bfloat16, device=device)
        self.y = torch.empty((rows, hidden), dtype=torch.bfloat16, device=device)

    def _weights(self, g, N, K):
        w = torch.randn((N, K), device=g.device, generator=g) * 0.02
        qw = torch.empty((N, K // 8), dtype=torch.int32, device=g.device)
        sc = torch.empty((N, K // 128), dtype=torch.int16, device=g.device)
        qz = torch.empty((N, (K // 128 + 7) // 8), dtype=torch.int32, device=g.device)
        self.lib.dev_quantize_w4_awq(w, qw, sc, qz, 128)
        return qw, sc, qz

    def project(self, x):
        """q, k, v [tokens, heads, dim], views of the QKV rows."""
        qw, sc, qz = self.qkv_w
        qkv = torch.empty((x.shape[0], qw.shape[0]), dtype=torch.bfloat16, device=x.device)
        self.lib.qlinear_w4a16(x, qw, sc, qz, None, sc.shape[1], qkv, 128)
        h, kv = self.q_heads, self.kv_heads
        return qkv.unflatten(1, (h + 2 * kv, self.dim)).split((h, kv, kv), 1)

    def _grown(self, counts):
        """The lengths with so many new tokens."""
        held = [n + c for n, c in zip(self.held, counts)]
        if max(held) > self.capacity:
            raise ValueError(f"a row of {max(held)} tokens is beyond the capacity of {self.capacity}")
        return held

    def prompt(self, x, counts):
        """The rows' prompts, one after the other in x [sum(counts), hidden], into
        the cache behind what it holds (their own attention is not part of this
        example, and so not of what an eviction ranks by: a prompt's tokens begin
        with a sum of 0)."""
        self.held = self._grown(counts)
        _, k, v = self.project(x)
        self.starts = torch.tensor([0] + list(counts), dtype=torch.int32).cumsum(0, dtype=torch.int32).to(x.device)
        n = torch.tensor(counts, dtype=torch.int32, device=x.device)
        self.lengths += n
        self.next_pos += n
        self.cache.append(k, v, self.tables, self.lengths, self.next_pos, starts=self.starts)

    def step(self, x):
        """One new token per row, x [rows, hidden]; returns y [rows, hidden]."""
        self.held = self._grown([1] * self.rows)
        longest = max(self.held)
        q, k, v = self.project(x)
        self.lengths += 1
        self.next_pos += 1
        self.cache.append(k, v, self.tables, self.lengths, self.next_pos)
        self.cache.attention(q, self.out, self.tables, self.lengths, longest, accumulate=True)
        qw, sc, qz = self.o_w
        self.lib.qlinear_w4a16(self.out.flatten(1), qw, sc, qz, None, sc.shape[1], self.y, 128)
        if longest > self.budget:
            self.cache.evict(self.tables, self.lengths, self.next_pos, self.kept, longest, self.budget, self.recent)
            self.lengths, self.kept = self.kept, self.lengths
            self.held = [min(n, self.budget) for n in self.held]
        return self.y


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--rows", type=int, default=16)
    p.add_argument("--prompt", type=int, default=512, help="tokens of the longest prompt")
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--budget", type=int, default=384)
    p.add_argument("--dtype", choices=["bf16", "int8"], default="bf16")
    a = p.parse_args()
    lib = sneppx_quant.load()
    block = AttentionBlock(lib, a.rows, max(a.prompt, a.budget) + 1, a.budget, a.budget // 8, dtype=a.dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    counts = [max(1, a.prompt * (i + 1) // a.rows) for i in range(a.rows)]
    block.prompt(torch.randn((sum(counts), 4096), device="cuda", generator=g).to(torch.bfloat16), counts)
    x = torch.randn((a.rows, 4096), device="cuda", generator=g).to(torch.bfloat16)
    for _ in range(4):
        block.step(x)
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(a.steps):
        y = block.step(x)
    torch.cuda.synchronize()
    t = (time.perf_counter() - t) / a.steps
    print(f"{a.rows} rows, {a.dtype} cache held at {a.budget} tokens: {t * 1e6:.1f} us a step, "
          f"lengths {block.lengths.tolist()}, |y| {float(y.float().norm()):.2f}")


if __name__ == "__main__":
    main()
