#!/usr/bin/env python3
"""A decoder layer's attention block in a server: rows come, begin with a common
prompt whose pages they share, decode, and go; pages are taken and given back on
the device.  QKV projection (W4A16), queries and keys normalised and turned to
their positions on the way into the cache, attention that reads the common prompt
once, or attention over the pages that a bound on their logits picks, O projection.

    python examples/kv_serve.py [--rows 16] [--prompt 1024] [--own 128] [--steps 64] [--dtype int8] [--pick 32]

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

I32, BF16 = torch.int32, torch.bfloat16


class ServeBlock:
    """Row 0 holds the common prompt and does not decode; rows 1 .. rows - 1 are
    streams.  The host keeps how long each row is (`held`) and how much of the prompt it
    shares, which it needs for the launches alone: lengths, tables and free pages stay on
    the device."""

    def __init__(self, lib, rows, pages, width, hidden=4096, q_heads=32, kv_heads=8, dim=128, page=16, dtype="bf16",
                 pick=0, seed=0, device="cuda"):
        self.lib, self.rows, self.page, self.pick, self.dim = lib, rows, page, pick, dim
        self.q_heads, self.kv_heads = q_heads, kv_heads
        g = torch.Generator(device=device).manual_seed(seed)
        self.qkv_w = self._weights(g, (q_heads + 2 * kv_heads) * dim, hidden)
        self.o_w = self._weights(g, hidden, q_heads * dim)
        norms = (1.0 + 0.1 * torch.randn(dim, device=device, generator=g) for _ in range(2))
        self.rotary = lib.rotary(dim, base=500000.0, scaling="bands", factor=8.0, original=8192, q_norm=next(norms),
                                 k_norm=next(norms), device=device)
        self.cache = lib.kv_cache(pages, page, kv_heads, dim, dtype, device=device)
        self.free = lib.kv_pages(pages, page, device=device)
        ints = lambda *shape: torch.zeros(shape, dtype=I32, device=device)  # noqa: E731
        self.tables = ints(rows, width) - 1
        self.lengths, self.next_pos, self.granted, self.starts = ints(rows), ints(rows), ints(rows), ints(rows + 1)
        self.held, self.common, self.shared = [0] * rows, 0, [0] * rows
        self._group()
        if pick:
            self.bounds = torch.zeros((pages, kv_heads, 2, dim), dtype=BF16, device=device)
            self.picked, self.picked_lengths = ints(rows, kv_heads, pick), ints(rows)
        self.out = torch.zeros((rows, q_heads, dim), dtype=BF16, device=device)
        self.y = torch.zeros((rows, hidden), dtype=BF16, device=device)

    def _weights(self, g, N, K):
        w = torch.randn((N, K), device=g.device, generator=g) * 0.02
        qw = torch.empty((N, K // 8), dtype=I32, device=g.device)
        sc = torch.empty((N, K // 128), dtype=torch.int16, device=g.device)
        qz = torch.empty((N, (K // 128 + 7) // 8), dtype=I32, device=g.device)
        self.lib.dev_quantize_w4_awq(w, qw, sc, qz, 128)
        return qw, sc, qz

    def project(self, x):
        """q, k, v [tokens, heads, dim], views of the QKV rows."""
        qw, sc, qz = self.qkv_w
        qkv = torch.empty((x.shape[0], qw.shape[0]), dtype=BF16, device=x.device)
        self.lib.qlinear_w4a16(x, qw, sc, qz, None, sc.shape[1], qkv, 128)
        h, kv = self.q_heads, self.kv_heads
        return qkv.unflatten(1, (h + 2 * kv, self.dim)).split((h, kv, kv), 1)

    def extend(self, x, counts):
        """New tokens of the rows, x [sum(counts), hidden]: pages for them, and their keys
        and values into the cache; returns their turned queries.  (A prompt's attention
        among its own tokens is not part of this example.)"""
        self.counts = torch.tensor(counts, dtype=I32).to(x.device)
        slots, positions = (torch.empty(x.shape[0], dtype=I32, device=x.device) for _ in range(2))
        self.free.reserve(self.tables, self.lengths, slots, counts=self.counts, next_pos=self.next_pos,
                          positions=positions, starts=self.starts, granted=self.granted)
        q, k, v = self.project(x)
        self.cache.append_rotated(self.rotary, q, k, v, slots, positions)       # (queries in place)
        self.held = [n + c for n, c in zip(self.held, counts)]
        if self.pick:
            self.cache.key_bounds(self.bounds, self.tables, self.lengths, self.counts, max(counts))
        return q

    def _group(self):
        """Streams next to one another that share as much of the prompt are a group."""
        mine = self.shared
        first = [b for b in range(1, self.rows) if b == 1 or mine[b] != mine[b - 1]]
        self.groups = torch.tensor([b - 1 for b in first] + [self.rows - 1], dtype=I32).to(self.tables.device)
        self.prefix = torch.tensor([mine[b] for b in first], dtype=I32).to(self.tables.device)

    def share(self, rows):
        """Has rows begin with row 0's prompt, as far as it fills pages."""
        self.common = self.held[0] // self.page * self.page
        sources = torch.tensor([0 if b in rows else -1 for b in range(self.rows)], dtype=I32).to(self.tables.device)
        self.free.share(self.tables, self.lengths, sources, torch.full_like(sources, self.common), next_pos=self.next_pos)
        self.held, self.shared = ([self.common if b in rows else n for b, n in enumerate(x)] for x in (self.held, self.shared))
        self._group()

    def end(self, rows):
        """Rows that have ended give their pages back."""
        gone = torch.tensor([b in rows for b in range(self.rows)]).to(self.tables.device)
        for t in (self.lengths, self.next_pos):
            t.masked_fill_(gone, 0)
        self.free.release(self.tables, self.lengths)
        self.held, self.shared = ([0 if b in rows else n for b, n in enumerate(x)] for x in (self.held, self.shared))
        self._group()

    def step(self, x):
        """One new token of each stream, x [rows, hidden] (row 0 is not looked at);
        returns y [rows, hidden]."""
        q = self.extend(x[1:], [0] + [1] * (self.rows - 1))
        longest = max(self.held)
        tables, lengths, out = self.tables[1:], self.lengths[1:], self.out[1:]
        if self.pick:
            self.cache.pick(q, self.bounds, tables, lengths, longest, self.picked[1:], self.picked_lengths[1:], 1, 2)
            self.cache.attention_picked(q, out, self.picked[1:], self.picked_lengths[1:])
        else:
            self.cache.attention_shared(q, out, tables, lengths, longest, self.groups, self.prefix, max(self.shared),
                                        max(n - s for n, s in zip(self.held[1:], self.shared[1:])))
        qw, sc, qz = self.o_w
        self.lib.qlinear_w4a16(self.out.flatten(1), qw, sc, qz, None, sc.shape[1], self.y, 128)
        return self.y


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--rows", type=int, default=16, help="streams")
    p.add_argument("--prompt", type=int, default=1024, help="tokens of the common prompt")
    p.add_argument("--own", type=int, default=128, help="tokens of the longest prompt behind it")
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--dtype", choices=["bf16", "int8"], default="bf16")
    p.add_argument("--pick", type=int, default=0, help="pages that a step attends to (0: all)")
    a = p.parse_args()
    lib, rows, page = sneppx_quant.load(), a.rows + 1, 16
    width = -(-(a.prompt + a.own + a.steps + 5) // page)
    block = ServeBlock(lib, rows, width + a.rows * (-(-(a.own + a.steps + 5) // page) + 1), width, dtype=a.dtype, pick=a.pick)
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = lambda n: torch.randn((n, 4096), device="cuda", generator=g).to(BF16)  # noqa: E731
    block.extend(tokens(a.prompt), [a.prompt] + [0] * a.rows)
    block.share(range(1, rows))
    own = [0] + [max(1, a.own * i // a.rows) for i in range(1, rows)]
    block.extend(tokens(sum(own)), own)
    x = tokens(rows)
    for _ in range(4):
        block.step(x)
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(a.steps):
        y = block.step(x)
    torch.cuda.synchronize()
    t = (time.perf_counter() - t) / a.steps
    used = int((block.free.refs > 0).sum())
    print(f"{a.rows} streams behind {a.prompt} tokens, {a.dtype} cache: {t * 1e6:.1f} us a step, {used} of "
          f"{block.free.pages} pages in use, |y| {float(y.float().norm()):.2f}")


if __name__ == "__main__":
    main()
