"""A pool beyond 4 GB (8 GB of keys and as many values): what stands in its last pages
is written, bounded, picked and attended to as in a small pool of the same rows, bit for
bit; and exact weights with infinite values."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_last_pages_of_a_large_pool(lib, dtype):
    page, heads, dim, rows, width = 64, 4, 128, 3, 6
    pages = (8 << 30) // (page * heads * dim * (1 if dtype == "int8" else 2))
    print(f"[gpu] kv serve in a pool of {pages} pages {dtype}", flush=True)
    small, large = lib.kv_cache(rows * width, page, heads, dim, dtype), lib.kv_cache(pages, page, heads, dim, dtype)
    g = torch.Generator(device=DEV).manual_seed(1)
    t = torch.arange(rows * width, dtype=torch.int32, device=DEV).view(rows, width)
    t[:, :3] = t[0, :3].clone()                        # a common prefix of three pages
    lengths = torch.tensor([200, 384, 300], dtype=torch.int32, device=DEV)
    tokens = rows * width * page
    r = lib.rotary(dim)
    kv = torch.randn((tokens, 2 * heads, dim), device=DEV, generator=g).to(BF)
    pos = torch.arange(tokens, dtype=torch.int32, device=DEV)
    q = torch.randn((rows, 16, dim), device=DEV, generator=g).to(BF)
    groups, prefix = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 3], [192]))
    results = []
    for c, first in ((small, 0), (large, pages - rows * width)):
        tables = t + first
        c.append_rotated(r, None, kv[:, :heads], kv[:, heads:], pos + first * page, pos)
        shared, over = (torch.zeros((rows, 16, dim), device=DEV) for _ in range(2))
        c.attention_shared(q, shared, tables, lengths, 384, groups, prefix, 192, 192)
        bounds = torch.zeros((c.pages, heads, 2, dim), dtype=BF, device=DEV)
        c.key_bounds(bounds, tables, lengths, lengths, 384)
        picked, n = torch.zeros((rows, heads, 3), dtype=torch.int32, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV)
        c.pick(q, bounds, tables, lengths, 384, picked, n)
        c.attention_picked(q, over, picked, n)
        torch.cuda.synchronize()
        last = slice(first, first + rows * width)
        results.append([x.clone() for x in (c.k[last], c.v[last], bounds[last], picked - first, n, shared, over)])
    for a, b in zip(*results):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("out", [BF, torch.float32])
def test_infinite_values_of_exact_weights(lib, out):
    """One token, or equal ones: weights whose lower pieces would be zero."""
    c = lib.kv_cache(8, 16, 1, 64)
    c.k.zero_()
    c.v.fill_(math.inf)
    c.v[..., 1::2] = -math.inf
    c.v[..., 5] = 2.0
    tables = torch.arange(8, dtype=torch.int32, device=DEV).view(2, 4)
    tables[1, :2] = tables[0, :2].clone()
    groups, prefix = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 2], [32]))
    q = torch.ones((2, 4, 64), dtype=BF, device=DEV)
    for lengths in ([1, 1], [32, 32], [33, 40], [64, 64]):
        o = torch.zeros((2, 4, 64), dtype=out, device=DEV)
        c.attention_shared(q, o, tables, torch.tensor(lengths, dtype=torch.int32, device=DEV), 64, groups, prefix, 32, 32)
        o = o.cpu().float()
        assert (o[..., 0::2] == math.inf).all() and (o[..., 1:5:2] == -math.inf).all() and (o[..., 5] == 2.0).all()
