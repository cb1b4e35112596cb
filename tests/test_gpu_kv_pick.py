"""SNEPPX_kv_key_bounds, _pick and _attention_picked against plain loops in float64
(serve_ref): bounds and picks equal, attention as in test_gpu_kv_attention.py."""
import math

import numpy as np
import pytest
import torch

import kv_ref
import serve_ref
from test_gpu_kv_attention import build

pytestmark = pytest.mark.gpu
DEV = "cuda"


def keys_of(c):
    k = c.k.float()
    if c.k_scales is not None:
        k = (k * c.k_scales.unsqueeze(-1)).to(torch.bfloat16).float()
    return k.cpu().double().numpy()


def new_bounds(c):
    return torch.full((c.pages, c.kv_heads, 2, c.head_dim), 7.0, dtype=torch.bfloat16, device=DEV)


def renew(c, tables, dtab, dlen, lengths, counts=None, most=1, bounds=None):
    b = new_bounds(c) if bounds is None else bounds
    want = b.cpu().double().numpy()
    c.key_bounds(b, dtab, dlen, None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV), most)
    torch.cuda.synchronize()
    serve_ref.key_bounds(keys_of(c), want, tables, lengths, counts, c.page_size)
    got = b.cpu().double().numpy()
    assert np.array_equal(got, want, equal_nan=True)
    return b, want


BOUNDS = [
    # lengths, heads, dim, page, dtype, counts
    ([1], 1, 128, 16, "bf16", None),
    ([0, 1, 16, 17, 31, 32, 33], 2, 64, 16, "bf16", None),
    ([0, 1, 16, 17, 31, 32, 33], 2, 64, 16, "int8", None),
    ([300, 5, 129], 3, 80, 24, "bf16", [300, 5, 100]),
    ([300, 5, 129], 3, 96, 24, "int8", [1, -3, 1000]),
    ([300, 500], 1, 256, 200, "bf16", [300, 2]),
    ([40, 41], 2, 16, 1, "int8", [7, 0]),
    ([513, 90], 2, 240, 128, "int8", [130, 90]),
]


@pytest.mark.parametrize("case", BOUNDS, ids=str)
def test_bounds(lib, case):
    lengths, heads, dim, page, dtype, counts = case
    print(f"[gpu] kv_key_bounds {case}", flush=True)
    c, _, tables, dtab, dlen = build(lib, lengths, heads, dim, page, dtype, 2 * dim)
    renew(c, tables, dtab, dlen, lengths, counts, 1 if counts is None else max(max(counts), 0))


def test_bounds_of_odd_keys(lib):
    """NaN in one element, infinities, a page that is not there, lengths outside the table."""
    c, _, tables, dtab, dlen = build(lib, [60, 64, 30], 2, 64, 16, "bf16", 3, absent=[(1, 3, -1)])
    c.k[tables[0, 3], 1, 2, 5] = math.nan
    c.k[tables[0, 3], 0, 11, 6] = math.inf
    c.k[tables[0, 2], 0, 0, 6] = -math.inf
    lengths = [60, 64, 1 << 30]
    dlen[2] = 1 << 30
    b, want = renew(c, tables, dtab, dlen, lengths, [60, 64, 2], 64)
    assert np.isnan(want[tables[0, 3], 1, :, 5]).all()


PICKS = [
    # lengths, q heads, kv heads, dim, page, dtype, budget, first, recent
    ([1, 0, 16, 17, 100], 4, 1, 128, 16, "bf16", 4, 1, 1),
    ([1000, 64, 65, 80, 900], 8, 2, 64, 16, "bf16", 5, 1, 2),
    ([1000, 64, 65, 80, 900], 8, 2, 64, 16, "int8", 5, 0, 1),
    ([2000, 777], 32, 8, 128, 64, "bf16", 8, 2, 3),
    ([2000, 777], 28, 4, 80, 24, "bf16", 20, 0, 20),         # all of them the newest
    ([2000, 777], 20, 1, 256, 32, "int8", 7, 6, 1),          # or the first and the newest
    ([3000, 2999], 3, 3, 96, 1, "int8", 1000, 10, 20),       # thousands of pages
    ([5000], 5, 1, 8, 2, "bf16", 1, 0, 1),
    ([333], 2, 2, 240, 128, "bf16", 64, 1, 1),               # a budget beyond the table
]


@pytest.mark.parametrize("case", PICKS, ids=str)
def test_pick(lib, case):
    lengths, hq, heads, dim, page, dtype, budget, first, recent = case
    print(f"[gpu] kv_pick {case}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, lengths, heads, dim, page, dtype, 3 * dim + hq)
    b, bounds = renew(c, tables, dtab, dlen, lengths, lengths, max(lengths))
    q = torch.randn((len(lengths), hq, dim), device=DEV, generator=torch.Generator(device=DEV).manual_seed(hq)).to(torch.bfloat16)
    picked = torch.full((len(lengths), heads, budget), 77, dtype=torch.int32, device=DEV)
    new = torch.zeros(len(lengths), dtype=torch.int32, device=DEV)
    c.pick(q, b, dtab, dlen, max(lengths), picked, new, first, recent)
    torch.cuda.synchronize()
    want, want_len = serve_ref.pick(q.cpu().double().numpy(), bounds, tables, lengths, page, budget, first, recent)
    assert np.array_equal(new.cpu().numpy(), want_len)
    assert np.array_equal(picked.cpu().numpy(), want)
    # attention over them: each head's own table
    for o in (torch.float32, torch.bfloat16):
        out = torch.full(q.shape, 7.0, dtype=o, device=DEV)
        c.attention_picked(q, out, picked, new)
        torch.cuda.synchronize()
        got = out.cpu().double().numpy()
        group = hq // heads
        for h in range(heads):
            one = kv_ref.Pool(*(None if x is None else x[:, h:h + 1] for x in (ref.k, ref.v, ref.ks, ref.vs)))
            hs = slice(h * group, (h + 1) * group)
            w, tol, _, _ = kv_ref.attention(one, q[:, hs].cpu().double().numpy(), want[:, h], want_len, dim ** -0.5)
            if o == torch.bfloat16:
                tol = tol + 2.0 ** -8 * np.abs(w)
            assert (np.abs(got[:, hs] - w) <= tol).all()


def test_ties_go_to_the_earlier_page(lib):
    """Every page the same: the first of them are picked, behind the ones that always are."""
    c, _, tables, dtab, dlen = build(lib, [640, 500], 2, 64, 16, "bf16", 5)
    b = torch.ones((c.pages, 2, 2, 64), dtype=torch.bfloat16, device=DEV)
    q = torch.randn((2, 4, 64), device=DEV).to(torch.bfloat16)
    picked, new = torch.zeros((2, 2, 7), dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    c.pick(q, b, dtab, dlen, 640, picked, new, 0, 2)
    for r, have in ((0, 40), (1, 32)):
        for h in range(2):
            assert picked[r, h].tolist() == [int(x) for x in tables[r, [0, 1, 2, 3, 4, have - 2, have - 1]]]


def test_pages_next_to_the_border(lib):
    """Scores that differ in the last bit of fp32, by one element of 256, are told apart."""
    c, _, tables, dtab, dlen = build(lib, [64 * 16], 1, 256, 16, "bf16", 6)
    b = torch.ones((c.pages, 1, 2, 256), dtype=torch.bfloat16, device=DEV)
    q = torch.ones((1, 1, 256), dtype=torch.bfloat16, device=DEV)
    q[0, 0, 0] = 256.0
    q[0, 0, 255] = 2.0 ** -9
    # sums 511 + x 2^-9: a step of fp32 is 2^-15
    for e in range(64):
        b[int(tables[0, e]), 0, :, 255] = (e % 32) * 2.0 ** -6
    picked, new = torch.zeros((1, 1, 9), dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    c.pick(q, b, dtab, dlen, 1024, picked, new, 0, 1)
    want, _ = serve_ref.pick(q.cpu().double().numpy(), b.cpu().double().numpy(), tables, [1024], 16, 9, 0, 1)
    assert np.array_equal(picked.cpu().numpy(), want)
    # (63 is the newest; then 31, 30 and 62, 29 and 61, 28 and 60, and of 27 and 59 the earlier)
    assert picked[0, 0].tolist() == [int(tables[0, e]) for e in (27, 28, 29, 30, 31, 60, 61, 62, 63)]


def test_pick_of_odd_bounds(lib):
    """NaN and pages that are not there come last, infinite scores in their order; lengths
    outside the table."""
    c, _, tables, dtab, dlen = build(lib, [320, 320], 1, 64, 16, "bf16", 7, absent=[(1, 4, -1), (1, 5, 1 << 30)])
    b = torch.randn((c.pages, 1, 2, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).sort(2)[0].to(torch.bfloat16)
    b[int(tables[0, 3]), 0, :, 9] = math.nan
    b[int(tables[0, 6]), 0, 1, :] = math.inf
    b[int(tables[0, 6]), 0, 0, :] = -math.inf
    q = torch.randn((2, 3, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(torch.bfloat16)
    dlen.copy_(torch.tensor([1 << 30, 320], dtype=torch.int32))
    lengths = [1 << 30, 320]
    for budget in (2, 18, 19):
        picked, new = torch.zeros((2, 1, budget), dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
        c.pick(q, b, dtab, dlen, 320, picked, new, 0, 1)
        want, want_len = serve_ref.pick(q.cpu().double().numpy(), b.cpu().double().numpy(), tables, lengths, 16, budget, 0, 1, 320)
        assert np.array_equal(picked.cpu().numpy(), want) and np.array_equal(new.cpu().numpy(), want_len)


def test_weights_of_picked_pages(lib):
    """accumulate adds to the tokens that a head attended to, and to no others."""
    lengths = [600, 90]
    c, ref, tables, dtab, dlen = build(lib, lengths, 2, 64, 16, "bf16", 8, weights=True)
    b, bounds = renew(c, tables, dtab, dlen, lengths, lengths, 600)
    q = torch.randn((2, 8, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).to(torch.bfloat16)
    picked, new = torch.zeros((2, 2, 9), dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    c.pick(q, b, dtab, dlen, 600, picked, new)
    before = c.weights.cpu().double().numpy()
    out = torch.zeros((2, 8, 64), device=DEV)
    c.attention_picked(q, out, picked, new, accumulate=True)
    torch.cuda.synchronize()
    diff = c.weights.cpu().double().numpy() - before
    for h in range(2):
        one = kv_ref.Pool(ref.k[:, h:h + 1], ref.v[:, h:h + 1])
        _, _, added, tol = kv_ref.attention(one, q[:, 4 * h:4 * h + 4].cpu().double().numpy(), picked[:, h].cpu().numpy(),
                                            new.tolist(), 0.125)
        assert (np.abs(diff[:, h] - added[:, 0]) <= tol[:, 0] + 2.0 ** -23 * np.abs(before[:, h])).all()
