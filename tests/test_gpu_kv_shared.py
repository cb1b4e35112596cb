"""SNEPPX_kv_attention_shared against the definition in float64 (kv_ref.attention over
every row's whole table).

Tolerances: kv_ref's bound of fp32 rounding.  Its reference point for weights is a
whole number up to 8 + log2(max_length) above the largest logit, so an exponent of up
to that size is rounded once more: 2^-19 at 64, of a weight, which is 32 units of
2^-24.  A bf16 result adds 2^-8 of itself, and weights cut to two bf16 pieces: each
is low by up to 2^-16 of itself, so a sum of them by up to 2^-15 of its magnitudes."""
import math

import numpy as np
import pytest
import torch

import kv_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def build(lib, groups, loose, heads, dim, page, dtype, seed, std=1.0):
    """groups: [(prefix tokens, [own tokens of each row])], then rows of no group.
    Whole pages of a prefix are shared, the rest of it is in every row's own page.
    What no row uses holds NaN."""
    rng = np.random.default_rng(seed)
    lengths, starts, prefix, lists, parents = [], [0], [], [], []
    for n, mine in groups:
        parents += [len(lengths)] * len(mine)
        lengths += [max(0, n + m) for m in mine]
        starts.append(len(lengths))
        prefix.append(n)
        lists += [n // page] * len(mine)
    parents += [None] * len(loose)
    lengths += loose
    lists += [0] * len(loose)
    rows, width = len(lengths), max(1, -(-max(lengths) // page))
    need = sum(-(-n // page) for n in lengths) + 3 + sum(n // page for n, _ in groups)
    perm = rng.permutation(need)
    tables = -np.ones((rows, width), np.int32)
    at = 0
    for b in range(rows):
        n, have = -(-lengths[b] // page), 0
        if parents[b] is not None:
            a = parents[b]
            if a == b:
                have = max(n, lists[b])
                have = min(have, width)
                tables[b, :have] = perm[at:at + have]
                at += have
            else:
                have = lists[b]
                tables[b, :have] = tables[a, :have]
        if n > have:
            tables[b, have:n] = perm[at:at + n - have]
            at += n - have
    pages = need
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((pages, heads, page, dim), generator=g) * std for _ in range(2))
    used = np.zeros((pages, page), bool)
    for b in range(rows):
        t = np.arange(lengths[b])
        used[tables[b, t // page], t % page] = True
        if parents[b] is not None and lists[b] * page < groups[starts_of(starts, b)][0]:
            # the same tokens in the row's own copy of the prefix's last page
            n = groups[starts_of(starts, b)][0]
            for t in range(lists[b] * page, min(n, lengths[b])):
                src, dst = tables[parents[b], t // page], tables[b, t // page]
                k[dst, :, t % page], v[dst, :, t % page] = k[src, :, t % page], v[src, :, t % page]
    # (pages that a first row shorter than the prefix names behind its end are other rows')
    for (n, mine), r0 in zip(groups, starts):
        if mine:
            t = np.arange(min(n, width * page))
            t = t[tables[r0, t // page] >= 0]
            used[tables[r0, t // page], t % page] = True
    c = lib.kv_cache(pages, page, heads, dim, dtype)
    ks = vs = None
    dead = torch.from_numpy(~used)[:, None, :].expand(pages, heads, page)
    if dtype == "int8":
        ks, vs = (torch.rand((pages, heads, page), generator=g) * 0.02 + 0.005 for _ in range(2))
        k, v = ((x * 40).round().clamp(-128, 127) for x in (k, v))
        for b in range(rows):
            if parents[b] is not None:
                n = groups[starts_of(starts, b)][0]
                for t in range(lists[b] * page, min(n, lengths[b])):
                    src, dst = tables[parents[b], t // page], tables[b, t // page]
                    ks[dst, :, t % page], vs[dst, :, t % page] = ks[src, :, t % page], vs[src, :, t % page]
        for s in (ks, vs):
            s[dead] = math.nan
        c.k_scales.copy_(ks)
        c.v_scales.copy_(vs)
        k, v = k.to(torch.int8), v.to(torch.int8)
    else:
        k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        k[dead], v[dead] = math.nan, math.inf
    c.k.copy_(k)
    c.v.copy_(v)
    ref = kv_ref.Pool(k.double().numpy(), v.double().numpy(), None if ks is None else ks.double().numpy(),
                      None if vs is None else vs.double().numpy())
    i32 = lambda x: torch.tensor(np.array(x), dtype=torch.int32, device=DEV)  # noqa: E731
    return c, ref, tables, lengths, i32(tables), i32(lengths), i32(starts), i32(prefix)


def starts_of(starts, b):
    return next(i for i in range(len(starts) - 1) if starts[i] <= b < starts[i + 1])


def check(c, ref, tables, lengths, dev, q, o, scale, most=None, max_prefix=None, max_own=None):
    dtab, dlen, starts, prefix = dev
    out = torch.full(q.shape, 7.0, dtype=torch.float32 if o == "f32" else torch.bfloat16, device=DEV)
    top = most if most is not None else dtab.shape[1] * c.page_size
    c.attention_shared(q, out, dtab, dlen, top, starts, prefix, max(prefix.tolist(), default=0) if max_prefix is None else max_prefix,
                       max(lengths) if max_own is None else max_own, scale)
    torch.cuda.synchronize()
    want, tol, _, _ = kv_ref.attention(ref, q.cpu().double().numpy(), tables, lengths, scale, most)
    size, _, _, _ = kv_ref.attention(kv_ref.Pool(ref.k, np.abs(ref.v), ref.ks, ref.vs), q.cpu().double().numpy(), tables,
                                     lengths, scale, most)
    tol = tol + 64 * 2.0 ** -24 * size
    got = out.cpu().double().numpy()
    if o == "bf16":
        tol = tol + 2.0 ** -8 * np.abs(want) + 2.0 ** -15 * size
    # (a row that is said to be longer than it was written attends to what its page holds)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isfinite(got), fine)
    assert (np.abs(got - want) <= tol)[fine].all(), float((np.abs(got - want) / np.maximum(tol, 1e-38))[fine].max())
    return out


CASES = [
    # groups, rows of none, q heads, kv heads, dim, page, dtype, out
    ([(64, [1, 2])], [], 4, 1, 128, 16, "bf16", "f32"),
    ([(64, [0, 0, 0])], [], 4, 2, 64, 16, "bf16", "f32"),                # nothing behind the prefix
    ([(0, [5, 6])], [3], 4, 2, 64, 16, "bf16", "f32"),                   # no prefix
    ([], [3, 0, 70], 4, 2, 64, 16, "bf16", "f32"),                       # no groups
    ([(48, [1] * 5), (160, [30, 0, 7]), (16, [300])], [0, 1, 129], 8, 2, 128, 16, "bf16", "f32"),
    ([(48, [1] * 5), (160, [30, 0, 7]), (16, [300])], [0, 1, 129], 8, 2, 128, 16, "int8", "f32"),
    ([(1000, [3, 64, 65, 100])], [], 32, 8, 128, 16, "bf16", "bf16"),    # a prefix that ends inside a page
    ([(1000, [3, 64, 65, 100])], [], 32, 8, 128, 64, "int8", "bf16"),
    ([(500, [-100, 20, -500, -1])], [], 8, 2, 64, 16, "bf16", "f32"),    # rows shorter than the prefix
    ([(640, list(range(40)))], [], 8, 2, 128, 32, "bf16", "f32"),        # two tiles of queries, one part full
    ([(640, list(range(33)))], [], 16, 4, 128, 32, "bf16", "bf16"),
    ([(320, list(range(16)))], [], 8, 1, 256, 16, "bf16", "f32"),        # 128 queries
    ([(320, list(range(9)))], [], 8, 1, 256, 16, "int8", "f32"),         # 72
    ([(320, list(range(8)))], [], 8, 1, 80, 24, "bf16", "f32"),          # 64
    ([(320, [4, 9])], [2], 300, 2, 64, 16, "bf16", "f32"),               # more query heads than a tile has
    ([(100, [1, 2]), (130, [3])], [], 14, 2, 96, 1, "bf16", "f32"),
    ([(100, [1, 2]), (130, [3])], [], 3, 3, 8, 5, "bf16", "f32"),
    ([(100, [1, 2]), (130, [3])], [], 6, 3, 16, 128, "int8", "f32"),
    ([(32, [1, 2])] * 70, [5], 4, 1, 64, 16, "bf16", "f32"),             # more groups than a wave has lanes
    ([(320, list(range(17)))], [], 8, 1, 96, 16, "bf16", "f32"),         # heads between 64 and 128, 136 queries
    ([(320, list(range(17)))], [], 8, 1, 80, 16, "int8", "bf16"),
    ([(200, [3, 0, 90])], [4], 8, 2, 72, 16, "bf16", "f32"),
    ([(5000, [10, 20, 30])], [], 8, 2, 64, 16, "bf16", "f32"),           # many spans
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}g-{sum(len(m) for _, m in c[0])}+{len(c[1])}-{c[2]}-{c[3]}-{c[4]}-p{c[5]}-{c[6]}-{c[7]}")
def test_shared(lib, case):
    groups, loose, hq, heads, dim, page, dtype, o = case
    print(f"[gpu] kv_attention_shared {case}", flush=True)
    c, ref, tables, lengths, *dev = build(lib, groups, loose, heads, dim, page, dtype, 3 * dim + hq)
    g = torch.Generator(device=DEV).manual_seed(hq)
    q = torch.randn((len(lengths), hq, dim), device=DEV, generator=g).to(torch.bfloat16)
    check(c, ref, tables, lengths, dev, q, o, 1 / math.sqrt(dim))


@pytest.mark.parametrize("max_prefix,max_own", [(0, 0), (1, 1), (1 << 20, 1 << 20), (640, 0), (0, 640)])
def test_sizes_of_the_launch_are_hints(lib, max_prefix, max_own):
    c, ref, tables, lengths, *dev = build(lib, [(640, [3, 200, 0]), (90, [1])], [300], 2, 64, 16, "bf16", 5)
    q = torch.randn((len(lengths), 8, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(torch.bfloat16)
    check(c, ref, tables, lengths, dev, q, "f32", 0.125, max_prefix=max_prefix, max_own=max_own)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales_and_strided_rows(lib, scale):
    c, ref, tables, lengths, *dev = build(lib, [(200, [3, 20, 0])], [40], 2, 64, 16, "bf16", 6)
    wide = torch.randn((len(lengths), 12 * 64 + 3), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).to(torch.bfloat16)
    q = wide[:, 3: 3 + 8 * 64].unflatten(1, (8, 64))
    check(c, ref, tables, lengths, dev, q, "f32", scale)


def test_max_length_cuts(lib):
    c, ref, tables, lengths, *dev = build(lib, [(200, [30, 200])], [90], 2, 64, 16, "bf16", 8)
    q = torch.randn((len(lengths), 4, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).to(torch.bfloat16)
    for most in (0, 1, 100, 200, 230, 1 << 40):
        if most == 0:
            out = torch.full(q.shape, 7.0, device=DEV)
            c.attention_shared(q, out, dev[0], dev[1], 0, dev[2], dev[3], 200, 200)
            assert (out == 0).all()
        else:
            check(c, ref, tables, lengths, dev, q, "f32", 0.125, most=most)


def test_large_logits_and_values(lib):
    """Logits of hundreds and values near the largest of bf16: finite, and the softmax's."""
    c, ref, tables, lengths, *dev = build(lib, [(300, [3, 70])], [40], 1, 64, 16, "bf16", 9)
    finite = torch.isfinite(c.v)
    c.v.copy_(torch.where(finite, c.v.sign() * 3e38, c.v.float()).to(torch.bfloat16))
    ref.v = c.v.cpu().double().numpy()
    q = torch.randn((len(lengths), 4, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)).to(torch.bfloat16)
    with np.errstate(over="ignore"):
        check(c, ref, tables, lengths, dev, q * 0, "f32", 1.0)
    c.v.copy_(torch.where(finite, torch.randn_like(c.v.float()), c.v.float()).to(torch.bfloat16))
    ref.v = c.v.cpu().double().numpy()
    # (a logit's rounding of up to 2^-24 of its magnitudes is in kv_ref's bound)
    check(c, ref, tables, lengths, dev, q * 30, "f32", 1.0)


def test_absent_pages_and_odd_lengths(lib):
    c, ref, tables, lengths, dtab, dlen, starts, prefix = build(lib, [(200, [30, 50])], [90], 2, 64, 16, "bf16", 10)
    for b, e, x in ((0, 2, -1), (1, 2, -1), (1, 13, 1 << 30), (2, 0, -5), (2, 1, -5)):
        tables[b, e] = x
    dtab.copy_(torch.from_numpy(tables))
    dlen[2] = lengths[2] = 1 << 30
    q = torch.randn((3, 4, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).to(torch.bfloat16)
    check(c, ref, tables, lengths, (dtab, dlen, starts, prefix), q, "f32", 0.125, max_own=300)
    dlen.copy_(torch.tensor([-4, 0, -1 << 31], dtype=torch.int32))
    out = torch.full(q.shape, 7.0, device=DEV)
    c.attention_shared(q, out, dtab, dlen, 500, starts, prefix, 200, 100)
    assert (out == 0).all()


def test_infinite_and_nan_logits(lib):
    """A row whose every logit is -inf gives NaN, as the formula; one NaN key makes its
    rows NaN and no others; an infinite value with weight shows."""
    c, ref, tables, lengths, *dev = build(lib, [(128, [20, 30])], [40], 1, 64, 16, "bf16", 11)
    q = torch.ones((3, 2, 64), device=DEV).to(torch.bfloat16)
    own = lambda b, t: (int(tables[b, t // 16]), 0, t % 16)  # noqa: E731
    for t in range(40):
        c.k[own(2, t)] = -math.inf
    c.k[own(1, 130)] = math.nan
    c.v[own(0, 5)][7] = math.inf
    out = torch.zeros((3, 2, 64), device=DEV)
    c.attention_shared(q, out, *dev[:2], 200, *dev[2:], 128, 40)
    o = out.cpu()
    assert torch.isnan(o[2]).all() and torch.isnan(o[1]).all()
    assert (o[0, :, 7] == math.inf).all()
    o[0, :, 7] = 0
    assert torch.isfinite(o[0]).all()


@pytest.mark.parametrize("own", [[-100, 20, -1], [-1, -200, -500], [-500, 0, 3]])
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_rows_shorter_than_their_prefix(lib, own, dtype):
    """Entries behind a short row's end name no page: the prefix is read by the table of a
    row that has it, and by none if none has."""
    c, ref, tables, lengths, *dev = build(lib, [(500, own)], [70], 2, 64, 16, dtype, 12)
    for b, n in enumerate(lengths):
        tables[b, -(-n // 16):] = -1
    dev[0].copy_(torch.from_numpy(tables))
    q = torch.randn((4, 8, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(6)).to(torch.bfloat16)
    check(c, ref, tables, lengths, dev, q, "f32", 0.125)
    check(c, ref, tables, lengths, dev, q, "bf16", 0.125, max_own=1)
