"""examples/kv_decode.py: the attention block of a decoder with its cache held
at a budget.  After every step the attention's output, the weights and what the
cache holds are checked against a plain record of the same tokens."""
import os
import sys

import numpy as np
import pytest
import torch

import kv_ref

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
from kv_decode import AttentionBlock  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pool_of(c):
    f = lambda t: None if t is None else t.cpu().double().numpy()     # noqa: E731
    return kv_ref.Pool(f(c.k), f(c.v), f(c.k_scales), f(c.v_scales))


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_decode_steps_at_a_budget(lib, dtype):
    rows, counts, budget, recent, heads, dim = 4, [30, 61, 9, 44], 48, 12, 2, 64
    print(f"[gpu] kv decode example {dtype}", flush=True)
    block = AttentionBlock(lib, rows, 64, budget, recent, hidden=256, q_heads=8, kv_heads=heads, dim=dim, dtype=dtype, seed=3)
    g = torch.Generator(device=DEV).manual_seed(5)
    block.prompt(torch.randn((sum(counts), 256), device=DEV, generator=g).to(torch.bfloat16), counts)
    tables = block.tables.cpu().numpy()
    seen = {}
    for s in range(12):
        x = torch.randn((rows, 256), device=DEV, generator=g).to(torch.bfloat16)
        before = block.lengths.tolist()
        weights = block.cache.weights.cpu().double().numpy()
        y = block.step(x).clone()
        torch.cuda.synchronize()
        q = block.project(x)[0].cpu().double().numpy()
        n = [b + 1 for b in before]
        # what was attended to, and what an eviction moved, are told apart by position
        pos = block.cache.positions.cpu().numpy()
        for b in range(rows):
            held = [tuple(pos[tables[b, t // 16], h, t % 16] for h in range(heads)) for t in range(int(block.lengths[b]))]
            total = counts[b] + s + 1
            assert int(block.next_pos[b]) == total and len(held) == min(n[b], budget)
            for h in range(heads):
                p = [x[h] for x in held]
                assert len(set(p)) == len(p) and set(range(max(0, total - recent), total)) <= set(p)
                if (b, h) in seen:                      # nothing comes back
                    assert set(p) <= seen[b, h] | {total - 1}
                seen[b, h] = set(p)
        if max(n) <= budget:
            want, tol, added, added_tol = kv_ref.attention(pool_of(block.cache), q, tables, n, dim ** -0.5)
            got = block.out.cpu().double().numpy()
            assert (np.abs(got - want) <= tol + 2.0 ** -8 * np.abs(want)).all()
            now = block.cache.weights.cpu().double().numpy()
            # (a slot that the step filled began at 0)
            for b in range(rows):
                weights[tables[b, (n[b] - 1) // 16], :, (n[b] - 1) % 16] = 0
            assert (np.abs(now - weights - added) <= added_tol + 2.0 ** -23 * np.abs(weights)).all()
        assert torch.isfinite(y.float()).all()
    # rows that were over the budget are held at it, and what they hold is attended to
    assert block.lengths.tolist() == [min(c + 12, budget) for c in counts]
    n = block.lengths.tolist()
    q = torch.randn((rows, 8, dim), device=DEV, generator=g).to(torch.bfloat16)
    out = torch.empty((rows, 8, dim), device=DEV)
    block.cache.attention(q, out, block.tables, block.lengths, 64)
    torch.cuda.synchronize()
    want, tol, _, _ = kv_ref.attention(pool_of(block.cache), q.cpu().double().numpy(), tables, n, dim ** -0.5)
    assert (np.abs(out.cpu().double().numpy() - want) <= tol).all()
