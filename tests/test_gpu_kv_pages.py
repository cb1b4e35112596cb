"""SNEPPX_kv_reserve, _release and _share against plain loops (serve_ref): whole
numbers, equal everywhere."""
import numpy as np
import pytest
import torch

import serve_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def state(rng, rows, width, page, pages, used, fill=0.6):
    """Rows that hold random pages up to their lengths, some of them shared, and pages
    that nobody here holds."""
    lengths = (rng.random(rows) * fill * width * page).astype(np.int32)
    tables = -np.ones((rows, width), np.int32)
    perm = rng.permutation(pages)
    at = 0
    for b in range(rows):
        n = -(-int(lengths[b]) // page)
        n = min(n, max(0, int(pages * (1 - used)) - at))
        lengths[b] = min(lengths[b], n * page)
        tables[b, :n] = perm[at:at + n]
        at += n
    refs = np.zeros(pages, np.int32)
    np.add.at(refs, tables[tables >= 0], 1)
    refs[perm[pages - int(pages * used):]] += 1
    return refs, tables, lengths, (lengths + rng.integers(0, 50, rows)).astype(np.int32)


def dev(*xs):
    return [None if x is None else torch.from_numpy(np.array(x)).to(DEV) for x in xs]


def run(lib, refs, page, tables, lengths, next_pos, counts, tokens, positions=True):
    d_refs, d_tab, d_len, d_pos, d_cnt = dev(refs, tables, lengths, next_pos, counts)
    slots = torch.full((tokens,), 77, dtype=torch.int32, device=DEV)
    pos = torch.full((tokens,), 77, dtype=torch.int32, device=DEV) if positions else None
    p = lib.kv_pages_from(d_refs, page)
    starts, granted = p.reserve(d_tab, d_len, slots, counts=d_cnt, next_pos=d_pos, positions=pos)
    torch.cuda.synchronize()
    w = [None if x is None else np.array(x, np.int64) for x in (refs, tables, lengths, next_pos)]
    want = serve_ref.reserve(w[0], page, w[1], w[2], w[3], counts, tokens)
    for got, ref, name in zip((d_refs, d_tab, d_len, d_pos, starts, granted, slots, pos), (*w, *want),
                              ("refs", "tables", "lengths", "next_pos", "starts", "granted", "slots", "positions")):
        if got is not None:
            assert np.array_equal(got.cpu().numpy(), ref), name
    return granted.cpu().numpy(), w


CASES = [
    # rows, width, page, pages, share of the pool that others hold, most new tokens
    (1, 4, 16, 8, 0.0, 1),
    (1, 1, 1, 1, 0.0, 1),
    (3, 8, 16, 40, 0.3, 20),
    (64, 40, 16, 3000, 0.2, 1),
    (64, 40, 16, 1700, 0.2, 300),          # too few pages for all
    (200, 9, 3, 2500, 0.5, 9),
    (1024, 6, 2, 9000, 0.1, 4),
    (1025, 6, 2, 9000, 0.1, 4),            # more rows than a turn has
    (2500, 5, 4, 9000, 0.3, 7),            # and pages that run out in a later one
    (5, 3000, 1, 30000, 0.2, 1500),        # rows of many pages
    (3, 9000, 1, 50000, 0.9, 3000),        # few free among many
    (40, 300, 16, 100000, 0.0, 2000),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("seed", [0, 1])
def test_reserve(lib, case, seed):
    print(f"[gpu] kv_reserve {case} seed {seed}", flush=True)
    rows, width, page, pages, used, most = case
    rng = np.random.default_rng(seed + 10 * rows)
    refs, tables, lengths, nxt = state(rng, rows, width, page, pages, used)
    counts = None if most == 1 else rng.integers(0, most + 1, rows).astype(np.int32)
    total = rows if counts is None else int(counts.sum())
    granted, w = run(lib, refs, page, tables, lengths, nxt if seed else None, counts, total + 5, positions=seed == 0)
    # every page is held as often as refs says, and no page by two rows
    held = np.bincount(w[1][w[1] >= 0], minlength=pages)
    assert held.max(initial=0) <= 1
    if case[3] == 1700:
        assert (granted == 0).any() and (granted > 0).any()


@pytest.mark.parametrize("tokens", [0, 3, 5000])
def test_tokens_short_and_long(lib, tokens):
    """slots for fewer tokens than there are, and for many more."""
    rng = np.random.default_rng(4)
    refs, tables, lengths, nxt = state(rng, 9, 20, 4, 200, 0.1)
    run(lib, refs, 4, tables, lengths, nxt, np.arange(9, dtype=np.int32), tokens)


def test_odd_values(lib):
    """Lengths and counts outside their range, entries that name no page or one already,
    a row without room, counts of the largest number."""
    refs = np.array([1, 0, 0, 1, 0, 0, 0, 1], np.int32)
    tables = np.array([[0, -1, -1], [3, 99, -7], [7, -1, 5], [-1, -1, -1], [-1, 2 ** 31 - 1, -2 ** 31], [-1, -1, -1]], np.int32)
    lengths = np.array([3, 4, 5, -3, 50, 0], np.int32)
    for counts in ([2, 5, 5, 1, 1, 1], [-4, 0, 2, 2 ** 31 - 1, 2 ** 31 - 1, 2], [9, 9, 9, 9, 9, 9], [0, 0, 0, 0, 0, 2 ** 31 - 1],
                   [1, 8, 1, 4, 0, 4]):
        run(lib, refs, 4, tables, lengths, None, np.array(counts, np.int32), 30)


def test_holes_in_rows_of_several_turns(lib):
    """Rows whose entries name pages here and there, over more free pages than a turn
    has: a free page every third."""
    rng = np.random.default_rng(3)
    pages, width = 40000, 9000
    refs = (np.arange(pages) % 3 != 0).astype(np.int32)
    tables = -np.ones((2, width), np.int32)
    taken = np.nonzero(refs)[0]
    for b in range(2):
        where = rng.choice(width, 3000, replace=False)
        tables[b, where] = taken[b * 3000: b * 3000 + 3000]
    run(lib, refs, 1, tables, np.array([0, 5], np.int32), None, np.array([8000, 7000], np.int32), 15000)


def test_no_free_page(lib):
    refs = np.ones(5000, np.int32)
    tables = -np.ones((3, 4), np.int32)
    granted, _ = run(lib, refs, 2, tables, np.array([0, 3, 1], np.int32), None, np.array([1, 1, 0], np.int32), 2)
    assert granted.tolist() == [0, 1, 0]       # (the second has room in its page, the third asks for nothing)


def test_release_and_share(lib):
    rng = np.random.default_rng(7)
    for rows, width, page, pages in ((1, 3, 4, 9), (40, 17, 8, 900), (300, 33, 16, 6000)):
        refs, tables, lengths, nxt = state(rng, rows, width, page, pages, 0.2)
        sources = np.where(rng.random(rows) < 0.4, rng.integers(0, rows, rows), -1).astype(np.int32)
        sources[0] = 0
        if rows > 3:
            sources[1], sources[2] = 2 ** 31 - 1, 3
        counts = rng.integers(-2, width * page + 9, rows).astype(np.int32)
        d_refs, d_tab, d_len, d_pos, d_src, d_cnt = dev(refs, tables, lengths, nxt, sources, counts)
        p = lib.kv_pages_from(d_refs, page)
        w = [np.array(x, np.int64) for x in (refs, tables, lengths, nxt)]

        def same(what):
            torch.cuda.synchronize()
            for got, ref, name in zip((d_refs, d_tab, d_len, d_pos), w, ("refs", "tables", "lengths", "next_pos")):
                assert np.array_equal(got.cpu().numpy(), ref), (what, name)
        p.share(d_tab, d_len, d_src, d_cnt, next_pos=d_pos)
        serve_ref.share(w[0], page, w[1], w[2], w[3], sources, counts)
        same("share")
        p.share(d_tab, d_len, d_src, d_cnt)                  # again: what they took goes back first
        serve_ref.share(w[0], page, w[1], w[2], None, sources, counts)
        same("share again")
        cut = np.minimum(w[2], rng.integers(-1, width * page, rows)).astype(np.int32)
        d_cut = dev(cut)[0]
        p.release(d_tab, d_cut)
        serve_ref.release(w[0], page, w[1], cut)
        same("release")
        d_cut.zero_()
        p.release(d_tab, d_cut)
        serve_ref.release(w[0], page, w[1], np.zeros(rows, int))
        same("release all")
        assert (w[1] == -1).all()
        p.release(d_tab, d_cut)                              # nothing left
        same("release again")


def test_release_of_pages_that_are_not_counted(lib):
    """A page that refs has as free, named twice: it stays free."""
    refs, tab, n = dev(np.array([0, 1, 2], np.int32), np.array([[0, 1], [0, 2], [5, -9]], np.int32), np.zeros(3, np.int32))
    lib.kv_pages_from(refs, 4).release(tab, n)
    torch.cuda.synchronize()
    assert refs.tolist() == [0, 0, 1] and tab.tolist() == [[-1, -1], [-1, -1], [5, -9]]
