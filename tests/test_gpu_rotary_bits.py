"""Sines and cosines of SNEPPX_kv_append_rotated as fp32 holds them, seen in an int8 cache's
scales: of a key whose only element is the first, the scale is max(|cos|, |sin|) * magnitude
/ 127.

Tolerance: the fp64 sine times the magnitude rounded to fp32 (2^-24), products with 1 and 0,
and the division (2^-24): two units of 2^-24; the fp64 angle, a few units of 2^-53 of up to
10^6 radians, adds a thousandth."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("magnitude", [1.0, 1.25, 1.3])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("far", [100, 131072, 1000000])
def test_sines_are_rounded_once(lib, far, interleaved, magnitude):
    tokens, heads, dim = 3000, 4, 128
    rng = np.random.default_rng(far)
    freqs = np.ones(dim // 2)
    freqs[1:4] = rng.uniform(0.01, 1.0, 3)
    pos = rng.integers(0, far, tokens).astype(np.int32)
    r = lib.rotary_from(torch.from_numpy(freqs).to(DEV), dim, interleaved, magnitude)
    k = torch.zeros((tokens, heads, dim), dtype=torch.bfloat16, device=DEV)
    for h in range(heads):                       # (head h: of pair h, the first element)
        k[:, h, 2 * h if interleaved else h] = 1.0
    c = lib.kv_cache(tokens, 1, heads, dim, "int8")
    slots = torch.arange(tokens, dtype=torch.int32, device=DEV)
    c.append_rotated(r, None, k, torch.zeros_like(k), slots, torch.from_numpy(pos).to(DEV))
    torch.cuda.synchronize()
    angle = pos.astype(np.float64)[:, None] * freqs[None, :heads]
    want = np.maximum(np.abs(np.cos(angle)), np.abs(np.sin(angle))) * float(np.float32(magnitude)) / 127
    got = c.k_scales.cpu().double().numpy()[:, :, 0]
    assert (np.abs(got - want) <= 2.002 * 2.0 ** -24 * want).all(), float((np.abs(got - want) / want).max() * 2 ** 24)
