"""SNEPPX_kv_attention over the range of the cache's values: results stay those of
the definition where values come near the largest that bf16 holds."""
import math

import numpy as np
import pytest
import torch

from test_gpu_kv_attention import build, compare

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("n,heads", [(40, 4), (900, 2), (5000, 1)])
def test_weights_of_zero_add_nothing(lib, n, heads, dtype):
    """One token of zeros has all the weight: the result is zero, whatever the values
    whose weights are 2^-512 and less, and so zero in fp32."""
    print(f"[gpu] kv_attention zero weights n={n} {dtype}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, [n], heads, 64, 16, dtype, 40 + n, garbage=False)
    c.k.zero_()
    at = n // 3
    page, off = int(tables[0, at // 16]), at % 16
    c.k[page, :, off] = 64
    if dtype == "int8":
        c.k_scales.fill_(1.0)
        c.v.fill_(100)
    else:
        c.v.fill_(1e30)
    c.v[page, :, off] = 0
    q = torch.ones((1, 2 * heads, 64), dtype=torch.bfloat16, device=DEV)
    out = torch.full((1, 2 * heads, 64), 3.0, device=DEV)
    c.attention(q, out, dtab, dlen, n, 0.125)       # 64 * 64 / 8 = 512 over 0
    torch.cuda.synchronize()
    assert bool((out == 0).all()), float(out.abs().max())


def put(c, ref, tables, b, t, value, scale=None):
    """Sets the value row of a token (int8: its codes and scale), in the cache and in the plain copy."""
    page, off = int(tables[b, t // c.page_size]), t % c.page_size
    x = torch.as_tensor(value)
    if scale is not None:
        c.v_scales[page, :, off] = scale
        ref.vs[page, :, off] = np.float64(np.float32(scale))
        c.v[page, :, off] = x.to(torch.int8).to(DEV)
    else:
        x = x.to(torch.bfloat16)
        c.v[page, :, off] = x.to(DEV)
    ref.v[page, :, off] = c.v[page, :, off].cpu().double().numpy()


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("n,heads", [(40, 4), (900, 2), (5000, 1)])
def test_weights_of_zero_times_the_largest_values(lib, n, heads, dtype):
    """One token has all the weight, the others' logits lie 2^9 and more below it (their
    weights are 2^-512 at most: nothing, whatever they are multiplied by)."""
    print(f"[gpu] kv_attention zero weights, large values n={n} {dtype}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, [n], heads, 64, 16, dtype, 40 + n, garbage=False)
    g = torch.Generator().manual_seed(n)
    c.k.zero_()
    ref.k[:] = 0
    at = n // 3
    page, off = int(tables[0, at // 16]), at % 16
    c.k[page, :, off] = 64
    ref.k[page, :, off] = 64
    for t in range(n):
        if dtype == "int8":
            put(c, ref, tables, 0, t, torch.randint(-100, 100, (heads, 64), generator=g), 1e-2 if t == at else 2e36)
        else:
            v = torch.randn((heads, 64), generator=g)
            put(c, ref, tables, 0, t, v if t == at else torch.where(v < 0, -3e38, 3e38))
    if dtype == "int8":
        c.k_scales.fill_(1.0)
        ref.ks[:] = 1.0
    q = torch.ones((1, 2 * heads, 64), dtype=torch.bfloat16, device=DEV)
    out = torch.empty((1, 2 * heads, 64), device=DEV)
    compare(c, ref, tables, dtab, dlen, [n], q, out, 0.125)       # 64 * 64 / 8 = 512 over 0


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("lengths,heads,accumulate", [([1, 2, 7, 31], 2, False), ([900, 130], 4, True), ([5000], 1, False),
                                                      ([5000, 3], 1, True), ([33000], 1, False)])
@pytest.mark.parametrize("signs", ["alike", "mixed"])
def test_values_near_the_largest(lib, lengths, heads, accumulate, signs, dtype):
    """Every value between 1e38 and 3.3e38: the results are means of them, so finite,
    however many are summed and wherever the largest logit lies."""
    print(f"[gpu] kv_attention values near the largest {lengths} {signs} {dtype}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, lengths, heads, 64, 16, dtype, 70 + heads, weights=accumulate, garbage=False)
    g = torch.Generator().manual_seed(len(lengths))
    v = torch.rand(c.v.shape, generator=g) * 2.3e38 + 1e38
    if signs == "mixed":
        v = torch.where(torch.rand(c.v.shape, generator=g) < 0.5, -v, v)
    if dtype == "int8":
        c.v_scales.fill_(2.6e36)
        ref.vs[:] = np.float64(np.float32(2.6e36))
        c.v.copy_((v / 2.6e36).round().to(torch.int8))
    else:
        c.v.copy_(v.to(torch.bfloat16))
    ref.v[:] = c.v.cpu().double().numpy()
    q = torch.randn((len(lengths), 4 * heads, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).to(torch.bfloat16)
    for o in (torch.float32, torch.bfloat16):
        out = torch.empty(q.shape, dtype=o, device=DEV)
        compare(c, ref, tables, dtab, dlen, lengths, q, out, 1 / math.sqrt(64), accumulate=accumulate)


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("lengths,heads", [([900, 130], 4), ([5000], 1), ([33000], 1)])
def test_values_far_below_one(lib, lengths, heads, dtype):
    """Values of 1e-20: as good in proportion as those near one."""
    print(f"[gpu] kv_attention values far below one {lengths} {dtype}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, lengths, heads, 64, 16, dtype, 90 + heads, garbage=False)
    if dtype == "int8":
        c.v_scales.mul_(1e-20)
        ref.vs[:] = c.v_scales.cpu().double().numpy()
    else:
        c.v.mul_(1e-20)
        ref.v[:] = c.v.cpu().double().numpy()
    q = torch.randn((len(lengths), 4 * heads, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(6)).to(torch.bfloat16)
    out = torch.empty(q.shape, device=DEV)
    compare(c, ref, tables, dtab, dlen, lengths, q, out, 1 / math.sqrt(64))
