"""SNEPPX_kv_append and SNEPPX_kv_evict against plain implementations
(kv_ref): rows are copied, quantized by the oracle's per-row rule, or moved, so
everything is compared bit for bit."""
import math

import numpy as np
import pytest
import torch

import kv_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bits(t):
    t = t.cpu()
    return t.view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()]).numpy()


def bf16_of(x):
    return torch.from_numpy(x).to(torch.bfloat16)


def new_cache(lib, pages, page, heads, dim, dtype):
    c = lib.kv_cache(pages, page, heads, dim, dtype, weights=True, positions=True)
    c.k.fill_(11)
    c.v.fill_(13)
    c.weights.fill_(5.0)
    c.positions.fill_(-9)
    if c.k_scales is not None:
        c.k_scales.fill_(2.0)
        c.v_scales.fill_(3.0)
    return c


APPENDS = [
    # new tokens per row, lengths with them, heads, dim, page
    ([1, 1, 1], [1, 17, 40], 8, 128, 16),
    ([1], [5], 1, 64, 3),
    ([0, 5, 1, 33, 0, 2], [3, 5, 9, 50, 0, 200], 2, 80, 16),
    ([300, 7], [300, 1000], 4, 256, 64),
    ([3, 4], [2, 90], 2, 16, 1),                 # more new tokens than slots: the first ones have none
    ([1] * 130, list(range(1, 131)), 3, 96, 24),
    ([17, 3], [400, 4], 5, 240, 7),
]


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("stored", [False, True])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{sum(c[0])}t{len(c[0])}r-{c[2]}-{c[3]}-p{c[4]}")
def test_append(lib, oracle, case, stored, dtype):
    counts, lengths, heads, dim, page = case
    print(f"[gpu] kv_append {case[1:]} {dtype} stored={stored}", flush=True)
    rng = np.random.default_rng(dim + len(counts))
    rows, tokens = len(counts), sum(counts)
    width = -(-max(lengths) // page)
    pages = rows * width + 2
    tables = rng.permutation(pages)[: rows * width].reshape(rows, width).astype(np.int32)
    if rows > 2:
        tables[2, 0] = -1                        # a page that is not there
    c = new_cache(lib, pages, page, heads, dim, dtype)
    wide = rng.normal(0, 1, (tokens, 2 * heads * dim + 8)).astype(np.float32)
    wide[0, : heads * dim] = 0.0
    if tokens > 3:
        wide[3, : heads * dim] *= 1e-39          # below the smallest normal scale
    wide = bf16_of(wide)
    dw = wide.to(DEV)
    k, v = (dw[:, i * heads * dim:(i + 1) * heads * dim].unflatten(1, (heads, dim)) for i in (0, 1))
    starts = np.cumsum([0] + counts).astype(np.int32)
    next_pos = np.array(lengths, np.int32) + 100
    ks, vs = (torch.full((tokens, heads, dim), 4.0, dtype=torch.bfloat16, device=DEV) if stored else None for _ in range(2))
    want = {n: getattr(c, n).cpu().clone() for n in ("k", "v", "weights", "positions")}
    scales = {n: getattr(c, n).cpu().clone() for n in ("k_scales", "v_scales")} if dtype == "int8" else {}
    use = None if counts == [1] * rows and tokens == rows else torch.from_numpy(starts).to(DEV)
    c.append(k, v, torch.from_numpy(tables).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV),
             torch.from_numpy(next_pos).to(DEV), starts=use, k_stored=ks, v_stored=vs)
    torch.cuda.synchronize()
    ws = [torch.full((tokens, heads, dim), 4.0, dtype=torch.bfloat16) for _ in range(2)]
    for t, b, slot, pos in kv_ref.append_slots(starts, lengths, next_pos, tokens):
        if slot < 0:
            continue
        pg, off = int(tables[b, slot // page]), slot % page
        if not 0 <= pg < pages:
            continue
        want["weights"][pg, :, off] = 0.0
        want["positions"][pg, :, off] = pos
        for i, n in enumerate("kv"):
            x = wide[t, i * heads * dim:(i + 1) * heads * dim].view(heads, dim)
            if dtype == "int8":
                _, codes, s = oracle.quantize_int8_channel(x.float().numpy())
                want[n][pg, :, off] = torch.from_numpy(codes)
                scales[n + "_scales"][pg, :, off] = torch.from_numpy(s)
                x = (torch.from_numpy(codes).float() * torch.from_numpy(s)[:, None]).to(torch.bfloat16)
            else:
                want[n][pg, :, off] = x
            ws[i][t] = x
    for n, w in {**want, **scales}.items():
        assert np.array_equal(bits(getattr(c, n)), bits(w)), n
    if stored:
        assert np.array_equal(bits(ks), bits(ws[0])) and np.array_equal(bits(vs), bits(ws[1]))


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("shift", [1, 4, 5])
def test_append_from_unaligned_rows(lib, oracle, shift, dtype):
    print(f"[gpu] kv_append unaligned shift={shift} {dtype}", flush=True)
    heads, dim, page = 2, 64, 16
    c = new_cache(lib, 8, page, heads, dim, dtype)
    wide = bf16_of(np.random.default_rng(shift).normal(0, 1, (3, heads * dim + 11)).astype(np.float32))
    x = wide.to(DEV)[:, shift:shift + heads * dim].unflatten(1, (heads, dim))
    tab = torch.tensor([[4], [2], [7]], dtype=torch.int32, device=DEV)
    c.append(x, x, tab, torch.tensor([3, 16, 1], dtype=torch.int32, device=DEV), torch.tensor([3, 16, 1], dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    for b, (pg, off) in enumerate(((4, 2), (2, 15), (7, 0))):
        row = wide[b, shift:shift + heads * dim].view(heads, dim)
        for pool, scales in ((c.k, c.k_scales), (c.v, c.v_scales)):
            got = pool[pg, :, off].cpu()
            if dtype == "int8":
                _, codes, s = oracle.quantize_int8_channel(row.float().numpy())
                assert np.array_equal(got.numpy(), codes) and np.array_equal(scales[pg, :, off].cpu().numpy(), s)
            else:
                assert np.array_equal(bits(got), bits(row))


def test_append_int8_of_nonfinite_rows(lib, oracle):
    """Infinities and NaN quantize as the reference's rule has them."""
    print("[gpu] kv_append nonfinite rows", flush=True)
    x = np.random.default_rng(3).normal(0, 1, (4, 32)).astype(np.float32)
    x[0, 3], x[1, 4], x[2, 5], x[2, 6] = math.inf, math.nan, -math.inf, math.nan
    c = new_cache(lib, 1, 4, 4, 32, "int8")
    b = bf16_of(x)
    t = b.to(DEV).view(1, 4, 32)
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    c.append(t, t, torch.zeros((1, 1), dtype=torch.int32, device=DEV), one, one)
    torch.cuda.synchronize()
    _, codes, s = oracle.quantize_int8_channel(b.float().numpy())
    assert np.array_equal(c.k[0, :, 0].cpu().numpy(), codes)
    assert np.array_equal(bits(c.k_scales[0, :, 0]), s.view(np.int32))


# ------------------------------------------------------------------- evict
def cut(lib, lengths, heads, dim, page, dtype, budget, recent, weights, seed=0, positions=None, absent=(), most=None,
        give_new=True):
    """One eviction checked against kv_ref.evict; weights(rng, shape) fills the plane."""
    rng = np.random.default_rng(seed)
    rows = len(lengths)
    width = max(1, -(-max(max(lengths), 1) // page))
    pages = rows * width + 2
    tables = rng.permutation(pages)[: rows * width].reshape(rows, width).astype(np.int32)
    c = lib.kv_cache(pages, page, heads, dim, dtype, weights=True, positions=True)
    for pool in (c.k, c.v):
        raw = torch.from_numpy(rng.integers(0, 256, pool.numel() * pool.element_size(), dtype=np.uint8))
        pool.view(torch.uint8).view(-1).copy_(raw)
    w = weights(rng, (pages, heads, page)).astype(np.float32)
    pos = np.zeros((pages, heads, page), np.int32)
    next_pos = np.array(lengths, np.int32) + 50
    for b, n in enumerate(lengths):
        for t in range(n):
            pos[tables[b, t // page], :, t % page] = 50 + t
    if positions is not None:
        pos = positions(rng, pos, tables)
    for b, e, value in absent:
        tables[b, e] = value
    c.weights.copy_(torch.from_numpy(w))
    c.positions.copy_(torch.from_numpy(pos))
    planes = [c.k.cpu().view(torch.uint8).numpy().copy(), c.v.cpu().view(torch.uint8).numpy().copy(), w.view(np.int32).copy(), pos.copy()]
    if dtype == "int8":
        for s in (c.k_scales, c.v_scales):
            s.copy_(torch.from_numpy(rng.random(s.shape, np.float32)))
            planes.append(bits(s).copy())
    ref = kv_ref.Pool(np.zeros((pages, heads, page, 1)), None, weights=w.copy(), positions=pos.copy())
    new = torch.full((rows,), -3, dtype=torch.int32, device=DEV)
    top = most if most is not None else width * page
    dlen = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    c.evict(torch.from_numpy(tables).to(DEV), dlen, torch.from_numpy(next_pos).to(DEV), new if give_new else None, top,
            budget, recent)
    torch.cuda.synchronize()
    want = kv_ref.evict(ref, planes, tables, lengths, next_pos, budget, recent, most)
    got = [c.k.cpu().view(torch.uint8).numpy(), c.v.cpu().view(torch.uint8).numpy(), bits(c.weights), bits(c.positions)]
    if dtype == "int8":
        got += [bits(c.k_scales), bits(c.v_scales)]
    for name, g, x in zip(("k", "v", "weights", "positions", "k_scales", "v_scales"), got, planes):
        assert np.array_equal(g, x), name
    if give_new:
        assert np.array_equal(new.cpu().numpy(), want)
    assert dlen.tolist() == lengths


def uniform(rng, shape):
    return rng.random(shape) ** 6 * 30


def few_values(rng, shape):
    return rng.integers(0, 3, shape)


def all_alike(rng, shape):
    return np.full(shape, 0.25)


def odd_numbers(rng, shape):
    """NaN, infinities, negative numbers, both zeros, subnormals."""
    return rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-42, -1e-42, 1.0, -1.0, 3e38], np.float32), shape)


@pytest.mark.parametrize("weights", [uniform, few_values, all_alike, odd_numbers])
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("lengths,budget,recent", [
    ([65, 64, 63, 0, 1], 64, 16),                # one too many, none too many
    ([300, 129, 1], 100, 10),
    ([300, 129, 2], 1, 0),                       # everything but one
    ([300, 299], 150, 150),                      # the newest alone
    ([1500, 1025, 1024, 1023], 700, 33),
])
def test_evict(lib, lengths, budget, recent, dtype, weights):
    print(f"[gpu] kv_evict {lengths} {budget} {recent} {dtype} {weights.__name__}", flush=True)
    cut(lib, lengths, 2, 32, 16, dtype, budget, recent, weights, seed=budget)


@pytest.mark.parametrize("heads,dim,page,dtype", [(1, 8, 1, "bf16"), (8, 128, 64, "bf16"), (3, 256, 5, "bf16"),
                                                  (5, 256, 24, "int8"), (12, 80, 48, "int8")])
def test_evict_layouts(lib, heads, dim, page, dtype):
    print(f"[gpu] kv_evict layout {heads} {dim} {page} {dtype}", flush=True)
    cut(lib, [211, 64, 140], heads, dim, page, dtype, 77, 20, uniform, seed=dim)


@pytest.mark.parametrize("length,budget", [(4097, 4096), (8200, 4000), (33000, 20000), (40000, 39999), (70001, 300)])
def test_evict_long(lib, length, budget):
    print(f"[gpu] kv_evict long {length} {budget}", flush=True)
    cut(lib, [length], 2, 16, 64, "bf16", budget, budget // 9, uniform, seed=length)


@pytest.mark.parametrize("weights", [uniform, few_values, all_alike, odd_numbers])
@pytest.mark.parametrize("lengths,budget,recent,page", [
    ([20000, 8200, 0, 4097], 4096, 300, 64),     # the budget ends a chunk of 4096 slots
    ([17000, 16999, 16384], 16998, 0, 24),       # one or two too many
    ([20481, 20480], 8193, 8193, 5),             # the newest alone
    ([16385, 3], 1, 1, 7),
])
def test_evict_long_rows_by_weights(lib, lengths, budget, recent, page, weights):
    """Rows that several workgroups cut: many keys alike, ties in several chunks."""
    print(f"[gpu] kv_evict long rows {lengths} {budget} {recent} {page} {weights.__name__}", flush=True)
    cut(lib, lengths, 2, 16, page, "int8", budget, recent, weights, seed=budget + page)


@pytest.mark.parametrize("weights", [uniform, few_values])
@pytest.mark.parametrize("lengths,heads,budget", [([17000], 130, 8192), ([16900, 16385], 130, 16384), ([17000], 260, 6000)])
def test_evict_long_rows_of_many_heads(lib, lengths, heads, budget, weights):
    """Workgroups that have more slots each where rows and heads are many."""
    print(f"[gpu] kv_evict long rows of many heads {lengths} {heads} {budget} {weights.__name__}", flush=True)
    cut(lib, lengths, heads, 8, 64, "bf16", budget, 99, weights, seed=heads)


@pytest.mark.parametrize("weights", [uniform, few_values, all_alike, odd_numbers])
@pytest.mark.parametrize("lengths,heads,budget,page", [
    ([2, 1, 0], 3, 1, 16),
    ([600, 599, 3], 3, 599, 24),
    ([17001, 17000, 400], 2, 17000, 64),
    ([40001], 2, 40000, 7),
])
def test_evict_one_token_too_many(lib, lengths, heads, budget, page, weights):
    print(f"[gpu] kv_evict one too many {lengths} {heads} {budget} {page} {weights.__name__}", flush=True)
    cut(lib, lengths, heads, 16, page, "int8", budget, budget // 8, weights, seed=budget, most=budget + 1)


def test_evict_one_token_too_many_of_many_heads(lib):
    """Longer chunks, absent pages, all tokens recent."""
    print("[gpu] kv_evict one too many, many heads", flush=True)
    cut(lib, [17001, 16900], 150, 8, 64, "bf16", 17000, 1, few_values, seed=3, most=17001)
    cut(lib, [17001, 17001], 2, 8, 64, "bf16", 17000, 0, uniform, seed=4, most=17001, absent=[(1, 100, -1)])
    cut(lib, [17001, 17001], 2, 8, 64, "bf16", 17000, 17000, uniform, seed=4, most=17001,
        positions=lambda rng, pos, tables: np.full_like(pos, 10 ** 6))


@pytest.mark.parametrize("length,budget,page", [(8193, 4096, 1), (9000, 8999, 3), (8200, 4100, 7), (8192, 8000, 2)])
def test_evict_long_rows_in_small_pages(lib, length, budget, page):
    print(f"[gpu] kv_evict small pages {length} {budget} {page}", flush=True)
    cut(lib, [length, length - 200], 3, 16, page, "int8", budget, budget // 9, few_values, seed=length)


def test_evict_long_rows_with_absent_pages(lib):
    print("[gpu] kv_evict long rows, absent pages", flush=True)
    cut(lib, [20000, 18000, 17000], 2, 16, 64, "bf16", 9000, 100, uniform, seed=8, absent=[(0, 200, -1), (2, 0, 1 << 29)])
    cut(lib, [20000, 18000, 17000], 2, 16, 64, "bf16", 9000, 100, few_values, seed=8, most=17500)


def test_evict_after_an_eviction(lib):
    """Positions in any order, and more recent ones than the budget holds."""
    print("[gpu] kv_evict positions", flush=True)

    def shuffled(rng, pos, tables):
        for h in range(pos.shape[1]):
            pos[:, h] = rng.permutation(pos[:, h].ravel()).reshape(pos[:, h].shape)
        return pos

    def newest(rng, pos, tables):
        return np.full_like(pos, 10 ** 6)

    for how in (shuffled, newest):
        cut(lib, [200, 150], 3, 16, 16, "bf16", 80, 30, uniform, seed=2, positions=how)
    cut(lib, [200, 150], 3, 16, 16, "bf16", 80, 30, all_alike, seed=2, positions=newest)


def test_evict_leaves_rows_with_absent_pages(lib):
    print("[gpu] kv_evict absent pages", flush=True)
    cut(lib, [200, 150, 90], 2, 16, 16, "bf16", 80, 30, uniform, seed=4, absent=[(0, 12, -1), (2, 5, 1 << 29)])


def test_evict_up_to_max_length(lib):
    print("[gpu] kv_evict max_length", flush=True)
    cut(lib, [200, 150, 90], 2, 16, 16, "bf16", 80, 30, uniform, seed=6, most=130)
    cut(lib, [200, 150, 90], 2, 16, 16, "bf16", 80, 30, uniform, seed=6, most=80)
    cut(lib, [200, 150, 90], 2, 16, 16, "bf16", 80, 30, uniform, seed=6, give_new=False)


def test_evict_in_a_graph(lib):
    """Recorded: replays on restored planes move the same rows each time."""
    print("[gpu] kv_evict graph", flush=True)
    rows, L, budget = 3, 500, 300
    c = lib.kv_cache(rows * 32, 16, 2, 64, weights=True, positions=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    tab = torch.randperm(rows * 32, device=DEV, generator=g).to(torch.int32).view(rows, 32)
    planes = (c.k, c.v, c.weights, c.positions)
    for t in planes[:3]:
        t.copy_(torch.rand(t.shape, device=DEV, generator=g))
    dlen = torch.full((rows,), L, dtype=torch.int32, device=DEV)
    nxt = dlen + 5
    new = torch.zeros_like(dlen)
    before = [t.clone() for t in planes]
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    call = lambda: c.evict(tab, dlen, nxt, new, L, budget, 40, stream=st.cuda_stream)   # noqa: E731
    call()
    st.synchronize()
    want = [t.clone() for t in planes]
    rec = lib.capture(call, stream=st.cuda_stream)
    for i in range(3):
        for t, x in zip(planes, before):
            t.copy_(x)
        new.zero_()
        torch.cuda.synchronize()
        lib.graph_launch(rec, stream=st.cuda_stream)
        st.synchronize()
        for t, x in zip(planes, want):
            assert np.array_equal(bits(t), bits(x)), i
        assert new.tolist() == [budget] * rows
    lib.graph_destroy(rec)
    lib.fn["SNEPPX_qlinear_release_workspaces"](st.cuda_stream)


@pytest.mark.parametrize("budget", [9000, 17000])
def test_evict_long_rows_in_a_graph(lib, budget):
    """Rows that several workgroups cut, and one token too many of them, recorded:
    the lengths are those of each replay."""
    print(f"[gpu] kv_evict long rows graph {budget}", flush=True)
    rows, L, wide = 2, 17001, 266
    c = lib.kv_cache(rows * wide, 64, 2, 16, weights=True, positions=True)
    g = torch.Generator(device=DEV).manual_seed(2)
    tab = torch.randperm(rows * wide, device=DEV, generator=g).to(torch.int32).view(rows, wide)
    planes = (c.k, c.v, c.weights, c.positions)
    for t in planes[:3]:
        t.copy_(torch.rand(t.shape, device=DEV, generator=g))
    dlen = torch.full((rows,), L, dtype=torch.int32, device=DEV)
    new = torch.zeros_like(dlen)
    before = [t.clone() for t in planes]
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    call = lambda: c.evict(tab, dlen, dlen, new, L, budget, 40, stream=st.cuda_stream)   # noqa: E731
    rec = lib.capture(call, stream=st.cuda_stream)
    for i, lengths in enumerate(([L, L], [budget, L], [L, 300], [L, L])):
        dlen.copy_(torch.tensor(lengths, dtype=torch.int32))
        results = []
        for run in (call, lambda: lib.graph_launch(rec, stream=st.cuda_stream)):
            for t, x in zip(planes, before):
                t.copy_(x)
            new.zero_()
            torch.cuda.synchronize()
            run()
            st.synchronize()
            results.append([bits(t).copy() for t in planes] + [new.cpu().numpy().copy()])
        for x, y in zip(*results):
            assert np.array_equal(x, y), i
        assert results[1][-1].tolist() == [min(n, budget) for n in lengths]
    lib.graph_destroy(rec)
    lib.fn["SNEPPX_qlinear_release_workspaces"](st.cuda_stream)
