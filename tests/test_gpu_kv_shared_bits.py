"""SNEPPX_kv_attention_shared: weights keep fp32 quality whatever the results' type, so that
a bf16 result is the rounding of a number that fp32 rounding can reach.

Logits here are whole 64ths, exact in fp32, and few, so what is left are the weights'
roundings, each relative: an exponent of up to 2 + 8 + 3 (the logit, the reference above
the maximum, and three for 8 tokens) is below 16 and so rounded by 2^-21, which is 0.35
units of 2^-20; scale * log2(e) by 2^-24 of 1.44 at most, 0.06; the exponential by 2^-23,
0.13.  Numerator and denominator: twice 0.54.  Four products and sums, the reciprocal and
its product: 8 roundings of 2^-24, 0.5; int8 weights times scales 0.06.  In all below 1.75
units of the magnitudes."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bf16(x):
    return torch.from_numpy(x).to(torch.bfloat16).double().numpy()


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("each", [64, 8, 0], ids=["wide", "narrow", "own"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_a_result_is_rounded_once(lib, dim, each, dtype):
    rows, heads, group, prefix, width = 64, 2, 4, 2, 8
    n_groups = rows // each if each else 0
    rng = np.random.default_rng(dim + each)
    lengths = np.array([prefix + 1 + b % 3 for b in range(rows)])
    tables = (np.arange(rows * width).reshape(rows, width) + 2 * rows).astype(np.int32)
    for b in range(rows):
        if each:
            tables[b, :prefix] = 2 * (b // each) + np.arange(prefix)
    pages = rows * width + 2 * rows
    c = lib.kv_cache(pages, 1, heads, dim, dtype)
    logit = rng.integers(-64, 65, (pages, heads))
    c.k.zero_()
    ks = 1.0 if dtype == "bf16" else 1 / 64
    c.k[:, :, 0, 0] = torch.from_numpy(logit / (64 * ks)).to(DEV).to(c.k.dtype)
    v = torch.from_numpy(rng.standard_normal((pages, heads, 1, dim)))
    if dtype == "int8":
        c.k_scales.fill_(ks)
        c.v.copy_((v * 40).clamp(-127, 127).to(torch.int8))
        c.v_scales.copy_(torch.from_numpy(rng.uniform(0.005, 0.025, (pages, heads, 1))))
        vals = c.v.cpu().double().numpy() * c.v_scales.cpu().double().numpy()[..., None]
    else:
        c.v.copy_(v)
        vals = c.v.cpu().double().numpy()
    q = torch.zeros((rows, heads * group, dim), dtype=torch.bfloat16, device=DEV)
    q[..., 0] = torch.from_numpy(rng.choice([1.0, 0.5, -1.0], (rows, heads * group))).to(DEV)
    i32 = lambda x: torch.tensor(np.array(x), dtype=torch.int32, device=DEV)  # noqa: E731
    starts, pre = i32([each * i for i in range(n_groups + 1)]), i32([prefix] * n_groups)
    qn = q[..., 0].cpu().double().numpy()
    want, size = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(rows):
        t = tables[b, : lengths[b]]
        for h in range(heads * group):
            s = qn[b, h] * logit[t, h // group] / 64
            w = np.exp(s - s.max())
            w /= w.sum()
            x = vals[t, h // group, 0]
            want[b, h], size[b, h] = w @ x, w @ np.abs(x)
    tol = 1.75 * 2.0 ** -20 * size + 2.0 ** -23 * np.abs(want)       # (the last for torch's own rounding by way of fp32)
    for o in (torch.float32, torch.bfloat16):
        out = torch.zeros(q.shape, dtype=o, device=DEV)
        c.attention_shared(q, out, i32(tables), i32(lengths), width, starts, pre, prefix, 3, 1.0)
        torch.cuda.synchronize()
        got = out.cpu().double().numpy()
        if o == torch.float32:
            assert (np.abs(got - want) <= tol).all()
        else:
            off = (got < bf16(want - tol)) | (got > bf16(want + tol))
            assert not off.any(), int(off.sum())


@pytest.mark.parametrize("o", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("below", [1, 60, 100, 105, 106, 110, 113])
def test_infinite_values_of_small_weights(lib, below, rows, o):
    """Weights of 2^-113 of the largest are, behind a reference 12 above, 2^-125 in fp32, so
    not zero: an infinite value shows.  (A scale of ln 2 times log2(e) is 1 in fp32: these
    weights are powers of two, all in their first bits.)"""
    c = lib.kv_cache(16 + rows, 1, 1, 64)
    c.k.zero_()
    c.v.fill_(1.0)
    c.k[3, :, :, 0] = -below
    c.v[3] = torch.inf
    c.v[3, :, :, 1::2] = -torch.inf
    tables = torch.arange(16, dtype=torch.int32, device=DEV).repeat(rows, 1)
    tables[:, 8] = 16 + torch.arange(rows, dtype=torch.int32, device=DEV)
    q = torch.zeros((rows, 4, 64), dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 1.0
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for prefix in (8, 0):
        out = torch.zeros(q.shape, dtype=o, device=DEV)
        c.attention_shared(q, out, tables, i32([9] * rows), 16, i32([0, rows]), i32([prefix]), prefix, 9 - prefix,
                           math.log(2.0))
        out = out.float()
        assert (out[..., 0::2] == torch.inf).all() and (out[..., 1::2] == -torch.inf).all()
