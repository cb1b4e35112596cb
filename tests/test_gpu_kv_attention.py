"""SNEPPX_kv_attention against the definition in float64 (kv_ref.attention).

Tolerances: kv_ref's bound of what fp32 rounding of the products, sums and
exponentials can move a result by; a bf16 result adds 2^-8 of itself (its unit
in the last place; the rounding is half of that)."""
import math

import numpy as np
import pytest
import torch

import kv_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def build(lib, lengths, heads, dim, page, dtype, seed, absent=(), spare=3, weights=False, std=1.0, garbage=True):
    """A cache with random rows in random pages; what no row uses holds NaN."""
    rng = np.random.default_rng(seed)
    width = max(1, -(-max(max(lengths), 1) // page))
    rows = len(lengths)
    pages = rows * width + spare
    tables = rng.permutation(pages)[: rows * width].reshape(rows, width).astype(np.int32)
    used = np.zeros((pages, 1, page, 1), bool)
    for b, n in enumerate(lengths):
        for t in range(max(n, 0)):
            used[tables[b, t // page], 0, t % page] = True
    for b, e, value in absent:
        used[tables[b, e]] = False
        tables[b, e] = value
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((pages, heads, page, dim), generator=g) * std for _ in range(2))
    c = lib.kv_cache(pages, page, heads, dim, dtype, weights=weights)
    ks = vs = None
    if dtype == "int8":
        ks, vs = (torch.rand((pages, heads, page), generator=g) * 0.02 + 0.005 for _ in range(2))
        k, v = (torch.randint(-128, 128, k.shape, generator=g).float() for _ in range(2))
        if garbage:
            for s in (ks, vs):
                s[torch.from_numpy(~used[..., 0]).expand_as(s)] = math.nan
        c.k_scales.copy_(ks)
        c.v_scales.copy_(vs)
        k, v = k.to(torch.int8), v.to(torch.int8)
    else:
        k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        if garbage:
            for x, bad in ((k, math.nan), (v, math.inf)):
                x[torch.from_numpy(~used).expand_as(x)] = bad
    c.k.copy_(k)
    c.v.copy_(v)
    if weights:
        c.weights.copy_(torch.rand(c.weights.shape, generator=g))
    ref = kv_ref.Pool(k.double().numpy(), v.double().numpy(), None if ks is None else ks.double().numpy(),
                      None if vs is None else vs.double().numpy())
    return c, ref, tables, torch.from_numpy(tables).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)


def compare(c, ref, tables, dtab, dlen, lengths, q, out, scale, most=None, accumulate=False, stream=None):
    before = c.weights.cpu().double().numpy() if accumulate else None
    top = most if most is not None else dtab.shape[1] * c.page_size
    c.attention(q, out, dtab, dlen, top, scale, accumulate=accumulate, stream=stream)
    torch.cuda.synchronize()
    want, tol, added, added_tol = kv_ref.attention(ref, q.cpu().double().numpy(), tables, lengths, scale, most)
    got = out.cpu().double().numpy()
    if out.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * np.abs(want)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / np.maximum(tol, 1e-38)).max())
    if accumulate:
        w = c.weights.cpu().double().numpy()
        t = added_tol + 2.0 ** -23 * np.abs(before)
        assert (np.abs(w - before - added) <= t).all(), float((np.abs(w - before - added) / np.maximum(t, 1e-38)).max())


CASES = [
    # lengths, q_heads, kv_heads, dim, page, dtype, out
    ([1], 4, 1, 128, 16, "bf16", "bf16"),
    ([0], 4, 1, 128, 16, "bf16", "f32"),
    ([0, 1, 2, 31, 32, 33, 63, 64, 65], 8, 2, 128, 16, "bf16", "f32"),
    ([127, 128, 129, 255, 256, 257], 8, 2, 128, 16, "int8", "f32"),
    ([511, 512, 513, 1000], 8, 8, 64, 32, "bf16", "f32"),
    ([2049, 3, 777], 32, 8, 128, 16, "bf16", "bf16"),
    ([2049, 3, 777], 32, 8, 128, 16, "int8", "bf16"),
    ([5000], 4, 1, 128, 64, "bf16", "f32"),
    ([5000], 4, 1, 128, 64, "int8", "f32"),
    ([300, 301], 7, 1, 80, 24, "bf16", "f32"),
    ([300, 301], 16, 1, 96, 1, "int8", "f32"),
    ([97, 500], 20, 1, 256, 3, "bf16", "f32"),
    ([97, 500], 33, 1, 64, 512, "int8", "f32"),
    ([97, 500], 64, 2, 128, 48, "bf16", "bf16"),
    ([200, 33], 3, 3, 8, 16, "bf16", "f32"),
    ([200, 33], 3, 3, 16, 16, "int8", "f32"),
    ([200, 33], 6, 3, 200, 5, "bf16", "f32"),
    ([150, 149], 12, 12, 240, 16, "int8", "f32"),
    ([40] * 70, 2, 2, 32, 8, "bf16", "f32"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{max(c[0])}x{len(c[0])}-{c[1]}-{c[2]}-{c[3]}-p{c[4]}-{c[5]}-{c[6]}")
@pytest.mark.parametrize("accumulate", [False, True])
def test_attention(lib, case, accumulate):
    lengths, hq, heads, dim, page, dtype, o = case
    print(f"[gpu] kv_attention {case} accumulate={accumulate}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, lengths, heads, dim, page, dtype, 7 * dim + hq, weights=accumulate)
    g = torch.Generator(device=DEV).manual_seed(hq)
    q = torch.randn((len(lengths), hq, dim), device=DEV, generator=g).to(torch.bfloat16)
    out = torch.full((len(lengths), hq, dim), 7.0, dtype=torch.float32 if o == "f32" else torch.bfloat16, device=DEV)
    compare(c, ref, tables, dtab, dlen, lengths, q, out, 1 / math.sqrt(dim), accumulate=accumulate)


@pytest.mark.parametrize("lengths,heads,dim,dtype", [
    ([3000, 0, 1, 2500, 1200, 700, 4000], 64, 16, "bf16"),       # shares of several steps that go across rows
    ([128] * 40 + [0] * 30 + list(range(0, 400, 5)), 32, 8, "bf16"),      # 150 rows, many of one step or none
    ([513, 0, 77, 1024, 300] * 30, 64, 16, "int8"),
    ([20000], 1, 16, "int8"),                                    # more shares of a row than a wave has lanes
    ([40001, 300], 1, 16, "bf16"),                               # and as many as a row may have
    ([1] * 300, 2, 32, "bf16"),
    (list(range(300)), 32, 8, "bf16"),                           # a share of many whole rows
])
def test_division_of_rows(lib, lengths, heads, dim, dtype):
    """How rows are cut depends on all their lengths: shares of whole steps that
    end and begin within rows, or rows that begin shares."""
    print(f"[gpu] kv_attention division of {len(lengths)} rows {heads} {dim} {dtype}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, lengths, heads, dim, 64, dtype, 50 + dim, weights=True)
    g = torch.Generator(device=DEV).manual_seed(heads)
    q = torch.randn((len(lengths), heads, dim), device=DEV, generator=g).to(torch.bfloat16)
    out = torch.full((len(lengths), heads, dim), 7.0, device=DEV)
    compare(c, ref, tables, dtab, dlen, lengths, q, out, 1 / math.sqrt(dim))
    # the same with the weights added
    both = torch.full_like(out, 5.0)
    compare(c, ref, tables, dtab, dlen, lengths, q, both, 1 / math.sqrt(dim), accumulate=True)
    assert torch.equal(both.view(torch.int32), out.view(torch.int32))
    # the same through the second launch (as recorded calls join), bit for bit
    st = torch.cuda.Stream()
    again = torch.full_like(out, 5.0)
    torch.cuda.synchronize()
    rec = lib.capture(lambda: c.attention(q, again, dtab, dlen, dtab.shape[1] * 64, 1 / math.sqrt(dim),
                                          stream=st.cuda_stream), stream=st.cuda_stream)
    lib.graph_launch(rec, stream=st.cuda_stream)
    st.synchronize()
    assert torch.equal(again.view(torch.int32), out.view(torch.int32))
    lib.graph_destroy(rec)
    lib.fn["SNEPPX_qlinear_release_workspaces"](st.cuda_stream)


@pytest.mark.parametrize("lengths,heads,dim,dtype", [
    ([2500, 2500], 64, 16, "bf16"),              # 8 shares of 5 steps: four for each row
    ([2304, 2176, 0], 64, 16, "int8"),           # one more row than fits
    ([1990] * 4, 64, 24, "bf16"),
    ([7000, 6700], 64, 16, "int8"),
    ([3000, 900, 2100], 33, 8, "bf16"),
    ([653] * 5, 32, 256, "bf16"),                # one workgroup to a CU: across rows from three steps a share on
    ([500, 20, 0, 333, 480, 77, 129], 32, 256, "bf16"),
])
def test_division_of_rows_in_as_many_shares(lib, lengths, heads, dim, dtype):
    """Long shares: rows begin them where no more are needed for it."""
    test_division_of_rows(lib, lengths, heads, dim, dtype)


def test_calls_of_many_divisions_in_turn(lib):
    """One stream's scratch and counters serve calls of every size in turn."""
    print("[gpu] kv_attention sizes in turn", flush=True)
    cases = [([700, 30], 8, 64, "bf16"), ([5], 1, 128, "int8"), ([2000, 0, 900, 1], 4, 256, "bf16"), ([300] * 9, 16, 32, "int8")]
    made = []
    for i, (lengths, heads, dim, dtype) in enumerate(cases):
        c, ref, tables, dtab, dlen = build(lib, lengths, heads, dim, 16, dtype, 60 + i)
        g = torch.Generator(device=DEV).manual_seed(i)
        q = torch.randn((len(lengths), 2 * heads, dim), device=DEV, generator=g).to(torch.bfloat16)
        made.append((c, ref, tables, dtab, dlen, lengths, q, torch.empty(q.shape, device=DEV), 1 / math.sqrt(dim)))
    for m in made + made[::-1]:
        compare(*m)


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("page,absent", [(16, [(0, 0, -1), (0, 7, 1 << 30), (1, 3, -5), (2, 0, -1)]), (3, [(0, 40, -1)]),
                                         (64, [(0, 4, -1), (1, 0, 999999)])])
def test_absent_pages(lib, dtype, page, absent):
    """Tokens of pages that are not there have no weight; row 2 has none."""
    lengths = [400, 300, 10]
    print(f"[gpu] kv_attention absent pages page={page} {dtype}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, lengths, 2, 64, page, dtype, page, absent=absent, weights=True)
    q = torch.randn((3, 8, 64), device=DEV).to(torch.bfloat16)
    out = torch.empty((3, 8, 64), device=DEV)
    compare(c, ref, tables, dtab, dlen, lengths, q, out, 0.125, accumulate=True)
    if page == 16:
        assert bool((out[2] == 0).all())


@pytest.mark.parametrize("most", [1, 100, 128, 333])
def test_lengths_beyond_what_is_there(lib, most):
    """Lengths above max_length or the table count as that, negative ones as 0."""
    lengths = [333, 5, 200]
    print(f"[gpu] kv_attention max_length={most}", flush=True)
    c, ref, tables, dtab, _ = build(lib, lengths, 2, 128, 16, "bf16", 5, garbage=False)
    said = [1 << 30, -7, 200]
    dlen = torch.tensor(said, dtype=torch.int32, device=DEV)
    q = torch.randn((3, 8, 128), device=DEV).to(torch.bfloat16)
    out = torch.empty((3, 8, 128), device=DEV)
    compare(c, ref, tables, dtab, dlen, said, q, out, 0.1, most=most)
    assert bool((out[1] == 0).all())


@pytest.mark.parametrize("shift", [0, 1, 4])
@pytest.mark.parametrize("o", ["f32", "bf16"])
def test_strided_rows(lib, shift, o):
    """Slices of wider rows, at offsets that leave them unaligned."""
    lengths, hq, dim = [70, 200], 8, 80
    print(f"[gpu] kv_attention strided rows shift={shift} {o}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, lengths, 2, dim, 16, "bf16", 11)
    wide = torch.randn((2, hq * dim + 13 + shift), device=DEV).to(torch.bfloat16)
    q = wide[:, shift:shift + hq * dim].unflatten(1, (hq, dim))
    dst = torch.full((2, hq * dim + 9), 3.0, dtype=torch.float32 if o == "f32" else torch.bfloat16, device=DEV)
    out = dst[:, shift:shift + hq * dim].unflatten(1, (hq, dim))
    compare(c, ref, tables, dtab, dlen, lengths, q, out, 1 / math.sqrt(dim))
    rest = torch.cat([dst[:, :shift], dst[:, shift + hq * dim:]], 1)
    assert bool((rest == 3.0).all())


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_sharp_and_growing_logits(lib, dtype):
    """Logits in the thousands, and rows whose maximum grows along the length."""
    lengths = [900, 900]
    print(f"[gpu] kv_attention sharp logits {dtype}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, lengths, 1, 64, 16, dtype, 21, garbage=False)
    ramp = np.linspace(0.01, 30, 900)
    for b in range(2):
        for t in range(900):
            f = ramp[t] if b == 0 else ramp[899 - t]
            if dtype == "int8":
                s = np.float32(ref.ks[tables[b, t // 16], 0, t % 16] * f)
                c.k_scales[int(tables[b, t // 16]), 0, t % 16] = float(s)
                ref.ks[tables[b, t // 16], 0, t % 16] = s
            else:
                x = (c.k[int(tables[b, t // 16]), 0, t % 16].float() * f).to(torch.bfloat16)
                c.k[int(tables[b, t // 16]), 0, t % 16] = x
                ref.k[tables[b, t // 16], 0, t % 16] = x.cpu().double().numpy()
    q = torch.randn((2, 4, 64), device=DEV).to(torch.bfloat16)
    out = torch.empty((2, 4, 64), device=DEV)
    for scale in (0.125, 4.0, -1.0, 0.0):
        compare(c, ref, tables, dtab, dlen, lengths, q, out, scale)


def test_nonfinite_values_are_the_rows_own(lib):
    """An infinite or NaN value in one row's tokens reaches that row's results as
    the softmax has it, and no other row's."""
    lengths = [100, 100, 100, 100]
    print("[gpu] kv_attention nonfinite values", flush=True)
    c, ref, tables, dtab, dlen = build(lib, lengths, 1, 64, 16, "bf16", 33)
    q = torch.randn((4, 4, 64), device=DEV).to(torch.bfloat16)
    c.v[int(tables[0, 2]), 0, 3, 5] = math.inf           # an infinite value: infinite in its column alone
    c.k[int(tables[1, 6]), 0, 2, 0] = math.nan           # a NaN key: its row is NaN
    c.k[int(tables[2, 1]), 0, 0, 0] = math.inf           # an infinite key: weight 0, or NaN with a positive query
    out = torch.empty((4, 4, 64), device=DEV)
    c.attention(q, out, dtab, dlen, 112)
    torch.cuda.synchronize()
    o = out.cpu()
    assert bool((o[0, :, 5] == math.inf).all()) and bool(torch.isfinite(o[0, :, :5]).all() & torch.isfinite(o[0, :, 6:]).all())
    assert bool(torch.isnan(o[1]).all())
    up = q[2, :, 0].cpu().float() > 0
    assert bool(torch.isnan(o[2][up]).all()) and bool(torch.isfinite(o[2][~up]).all())
    assert bool(torch.isfinite(o[3]).all())


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("n", [1, 2, 100])
def test_infinite_values_with_short_weights(lib, n, dtype):
    """Equal weights, which as powers of two have few significant bits: an infinite
    value (int8: an infinite scale) times any part of them is infinite."""
    print(f"[gpu] kv_attention infinite values n={n} {dtype}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, [n], 1, 64, 16, dtype, 37, garbage=False)
    c.k.zero_()
    page, off = int(tables[0, (n - 1) // 16]), (n - 1) % 16
    if dtype == "int8":
        c.v[page, 0, off] = 1
        c.v[page, 0, off, 7] = -1
        c.v_scales[page, 0, off] = math.inf
    else:
        c.v[page, 0, off, 5] = math.inf
        c.v[page, 0, off, 7] = -math.inf
    out = torch.empty((1, 4, 64), device=DEV)
    c.attention(torch.ones((1, 4, 64), dtype=torch.bfloat16, device=DEV), out, dtab, dlen, 112)
    torch.cuda.synchronize()
    o = out.cpu()
    assert bool((o[0, :, 5] == math.inf).all()) and bool((o[0, :, 7] == -math.inf).all())
    rest = torch.tensor([d for d in range(64) if d not in (5, 7)])
    assert bool(torch.isfinite(o[0][:, rest]).all() if dtype == "bf16" else (o[0][:, rest] == math.inf).all())


def test_all_logits_minus_infinity(lib):
    """Tokens are there and every logit is -inf: 0 / 0, as the softmax has it; a
    row without tokens beside it stays zero."""
    print("[gpu] kv_attention all -inf", flush=True)
    c, ref, tables, dtab, dlen = build(lib, [300, 0], 1, 64, 16, "bf16", 34, garbage=False)
    c.k.fill_(1.0)
    c.k[..., 0] = -math.inf
    q = torch.ones((2, 4, 64), dtype=torch.bfloat16, device=DEV)
    out = torch.empty((2, 4, 64), device=DEV)
    c.attention(q, out, dtab, dlen, 304)
    torch.cuda.synchronize()
    assert bool(torch.isnan(out[0]).all()) and bool((out[1] == 0).all())
    # one finite logit among them takes all the weight
    c.k[int(tables[0, 5]), 0, 4, 0] = 0.0
    c.attention(q, out, dtab, dlen, 304)
    torch.cuda.synchronize()
    assert bool(torch.equal(out[0], c.v[int(tables[0, 5]), 0, 4].float().expand(4, -1)))


def test_shared_pages_and_repeatability(lib):
    """Rows that share pages; two calls give the same bits."""
    print("[gpu] kv_attention shared pages", flush=True)
    c, ref, tables, dtab, dlen = build(lib, [700, 700, 650], 2, 128, 16, "bf16", 35)
    tables[1] = tables[0]
    tables[2, :30] = tables[0, :30]
    dtab = torch.from_numpy(tables).to(DEV)
    lengths = [700, 650, 480]
    dlen = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = torch.randn((3, 8, 128), device=DEV).to(torch.bfloat16)
    out, again = torch.empty((3, 8, 128), device=DEV), torch.empty((3, 8, 128), device=DEV)
    compare(c, ref, tables, dtab, dlen, lengths, q, out, 0.08)
    c.attention(q, again, dtab, dlen, 704, 0.08)
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int32), again.view(torch.int32))


def test_offsets_beyond_32_bits(lib):
    """Pages beyond 4 GiB of the pool (9 GiB each of k and v)."""
    print("[gpu] kv_attention pool of 9 GiB", flush=True)
    heads, dim, page = 8, 128, 64
    pages = (9 << 30) // (heads * dim * page * 2)
    c = lib.kv_cache(pages, page, heads, dim, weights=True)
    n, width = 500, 8
    for first in (pages - width, pages // 2):
        tab = torch.arange(first, first + width, dtype=torch.int32, device=DEV).view(1, width)
        g = torch.Generator(device=DEV).manual_seed(first)
        kk, vv = (torch.randn((width, heads, page, dim), device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
        c.k[first:first + width], c.v[first:first + width] = kk, vv
        q = torch.randn((1, 32, dim), device=DEV, generator=g).to(torch.bfloat16)
        out = torch.empty((1, 32, dim), device=DEV)
        c.attention(q, out, tab, torch.tensor([n], dtype=torch.int32, device=DEV), 512, 0.09, accumulate=True)
        torch.cuda.synchronize()
        ref = kv_ref.Pool(kk.cpu().double().numpy(), vv.cpu().double().numpy())
        want, tol, added, added_tol = kv_ref.attention(ref, q.cpu().double().numpy(),
                                                       np.arange(width, dtype=np.int32)[None], [n], 0.09)
        assert (np.abs(out.cpu().double().numpy() - want) <= tol).all()
        got = c.weights[first:first + width].cpu().double().numpy()
        assert (np.abs(got - added) <= added_tol).all()
    assert float(c.weights[: pages // 2].abs().max()) == 0.0


def test_on_another_stream_and_in_a_graph(lib):
    """A stream of the caller's, eager and recorded; replays equal the eager call."""
    print("[gpu] kv_attention stream and graph", flush=True)
    c, ref, tables, dtab, dlen = build(lib, [3000, 17, 1200, 0], 2, 128, 16, "bf16", 36)
    q = torch.randn((4, 8, 128), device=DEV).to(torch.bfloat16)
    eager = torch.empty((4, 8, 128), device=DEV)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        c.attention(q, eager, dtab, dlen, 3008)
    st.synchronize()
    out = torch.zeros_like(eager)
    torch.cuda.synchronize()
    g = lib.capture(lambda: c.attention(q, out, dtab, dlen, 3008, stream=st.cuda_stream), stream=st.cuda_stream)
    for i in range(4):
        out.fill_(float(i))
        torch.cuda.synchronize()
        lib.graph_launch(g, stream=st.cuda_stream)
        st.synchronize()
        assert torch.equal(out.view(torch.int32), eager.view(torch.int32)), i
        c.attention(q, torch.empty_like(out), dtab, dlen, 3008)          # the program's own work between replays
        torch.cuda.synchronize()
    lib.graph_destroy(g)
    lib.fn["SNEPPX_qlinear_release_workspaces"](st.cuda_stream)
