"""Append with rotation, pages, attention behind shared prefixes and over picked pages:
their entry points reject bad arguments before they touch the device (-1 and a reason),
calls of nothing do nothing, and the binding checks its tensors.  CPU only (the pointers
passed are never dereferenced: every check runs first)."""
import ctypes as C

import pytest
import torch

import sneppx_quant as sq
from test_kv_args import CACHES, struct
from test_rotary_args import rotary


@pytest.fixture(scope="module")
def L():
    return sq.load()


P = C.c_void_p(64)                     # stand-in device pointers, never read
A, B, D, E = (C.c_void_p(4096 * i) for i in (1, 2, 3, 4))


def of(c):
    return C.byref(c) if c else None


def append(L, cache=None, r=None, q=P, qs=512, qo=P, qos=512, hq=8, k=P, ks=128, v=P, vs=128, tokens=3, slots=P, pos=P,
           ko=None, vo=None):
    return L.fn["SNEPPX_kv_append_rotated"](of(cache if cache is not None else struct()), of(r if r is not None else rotary()),
                                            q, qs, qo, qos, hq, k, ks, v, vs, tokens, slots, pos, ko, vo, None)


def shared(L, cache=None, q=P, qs=512, out=P, os=512, odt=0, tab=P, width=4, ln=P, rows=3, hq=8, most=64, starts=P, prefix=P,
           groups=2, scale=0.1):
    return L.fn["SNEPPX_kv_attention_shared"](of(cache if cache is not None else struct()), q, qs, out, os, odt, tab, width,
                                              ln, rows, hq, most, starts, prefix, groups, 32, 32, scale, None)


def bounds(L, cache=None, to=P, tab=P, width=4, ln=P, counts=None, most=1, rows=3):
    return L.fn["SNEPPX_kv_key_bounds"](of(cache if cache is not None else struct()), to, tab, width, ln, counts, most, rows,
                                        None)


def pick(L, cache=None, bd=P, q=P, qs=512, hq=8, tab=P, width=4, ln=A, rows=3, most=64, budget=3, first=1, recent=1, to=P,
         new=B):
    return L.fn["SNEPPX_kv_pick"](of(cache if cache is not None else struct()), bd, q, qs, hq, tab, width, ln, rows, most,
                                  budget, first, recent, to, new, None)


def picked(L, cache=None, q=P, qs=512, out=P, os=512, odt=0, tab=P, width=4, ln=P, rows=3, hq=8, acc=0):
    return L.fn["SNEPPX_kv_attention_picked"](of(cache if cache is not None else struct()), q, qs, out, os, odt, tab, width,
                                              ln, rows, hq, 0.1, acc, None)


def reserve(L, refs=P, pages=8, size=16, tab=P, width=4, ln=A, nxt=None, counts=None, rows=3, starts=P, granted=B, slots=P,
            pos=None, tokens=3):
    return L.fn["SNEPPX_kv_reserve"](refs, pages, size, tab, width, ln, nxt, counts, rows, starts, granted, slots, pos,
                                     tokens, None)


def release(L, refs=P, pages=8, size=16, tab=P, width=4, ln=A, rows=3):
    return L.fn["SNEPPX_kv_release"](refs, pages, size, tab, width, ln, rows, None)


def share(L, refs=P, pages=8, size=16, tab=P, width=4, ln=A, nxt=None, src=B, counts=D, rows=3):
    return L.fn["SNEPPX_kv_share"](refs, pages, size, tab, width, ln, nxt, src, counts, rows, None)


@pytest.mark.parametrize("call", [append, shared, bounds, pick, picked], ids=lambda f: f.__name__)
@pytest.mark.parametrize("cache,reason", CACHES, ids=lambda x: x if isinstance(x, str) else "")
def test_bad_caches(L, call, cache, reason):
    assert call(L, cache=cache) == -1
    assert reason in L.last_error()


@pytest.mark.parametrize("call", [shared, bounds, pick, picked], ids=lambda f: f.__name__)
@pytest.mark.parametrize("kw,reason", [(dict(tab=None), "NULL block_tables"), (dict(ln=None), "NULL block_tables or lengths"),
                                       (dict(width=0), "empty block_tables"), (dict(width=1 << 40), "too large"),
                                       (dict(rows=1 << 32), "too many")])
def test_bad_rows(L, call, kw, reason):
    assert call(L, **kw) == -1
    assert reason in L.last_error()


@pytest.mark.parametrize("call", [reserve, release, share], ids=lambda f: f.__name__)
@pytest.mark.parametrize("kw,reason", [
    (dict(pages=0), "no pages"), (dict(size=0), "no pages"), (dict(pages=1 << 28), "31 bits"), (dict(size=1 << 31), "31 bits"),
    (dict(refs=None), "NULL refs"), (dict(tab=None), "NULL refs, block_tables"), (dict(ln=None), "or lengths"),
    (dict(width=0), "empty block_tables"), (dict(width=1 << 40), "too large"), (dict(rows=1 << 30), "too many")])
def test_bad_pages(L, call, kw, reason):
    assert call(L, **kw) == -1
    assert reason in L.last_error()


@pytest.mark.parametrize("call,kw,reason", [
    (append, dict(r=False), "NULL rotary"), (append, dict(r=rotary(dims=72)), "up to head_dim 64"),
    (append, dict(k=None), "NULL pointer"), (append, dict(v=None), "NULL pointer"), (append, dict(slots=None), "NULL pointer"),
    (append, dict(pos=None), "NULL pointer"), (append, dict(q=None), "NULL q"), (append, dict(qo=None), "NULL q"),
    (append, dict(ko=P), "go together"), (append, dict(vo=P), "go together"), (append, dict(hq=70000), "too many"),
    (append, dict(tokens=1 << 40), "too many"), (append, dict(ks=127), "below its row"), (append, dict(vs=127), "below its row"),
    (append, dict(qs=511), "below its row"), (append, dict(qos=511), "below its row"), (append, dict(qos=520), "q in place"),
    (append, dict(cache=struct(pages=1 << 27, kv_heads=1)), "31 bits"),
    (shared, dict(q=None), "NULL pointer"), (shared, dict(out=None), "NULL pointer"), (shared, dict(odt=8), "out_dtype"),
    (shared, dict(hq=7), "not a multiple"), (shared, dict(hq=0), "not a multiple"), (shared, dict(qs=511), "q_stride"),
    (shared, dict(os=511), "out_stride"), (shared, dict(starts=None), "NULL group_starts"),
    (shared, dict(prefix=None), "NULL group_starts or prefix_lengths"), (shared, dict(groups=4), "4 groups of 3 rows"),
    (bounds, dict(to=None), "NULL bounds"), (bounds, dict(to=C.c_void_p(72)), "16-byte aligned"),
    (pick, dict(bd=None), "NULL bounds"), (pick, dict(bd=C.c_void_p(72)), "16-byte aligned"), (pick, dict(q=None), "NULL pointer"),
    (pick, dict(hq=7), "not a multiple"), (pick, dict(qs=511), "q_stride"), (pick, dict(to=None), "NULL bounds, picked"),
    (pick, dict(new=None), "picked_lengths"), (pick, dict(budget=0), "budget 0"), (pick, dict(budget=1 << 40), "too large"),
    (pick, dict(recent=0), "do not fit"), (pick, dict(recent=4), "do not fit"), (pick, dict(first=3), "do not fit"),
    (pick, dict(new=A), "must not be lengths"), (pick, dict(new=C.c_void_p(4096 + 8)), "nor overlap"),
    (picked, dict(q=None), "NULL pointer"), (picked, dict(out=None), "NULL pointer"), (picked, dict(odt=8), "out_dtype"),
    (picked, dict(hq=9), "not a multiple"), (picked, dict(cache=struct(weights=None), acc=1), "needs the cache's weights"),
    (picked, dict(qs=511), "q_stride"), (picked, dict(os=511), "out_stride"),
    (reserve, dict(starts=None), "NULL starts"), (reserve, dict(granted=None), "NULL starts or granted"),
    (reserve, dict(slots=None), "NULL slots"), (reserve, dict(tokens=1 << 40), "too many"),
    (reserve, dict(granted=A), "overlap"), (reserve, dict(nxt=A), "overlap"), (reserve, dict(counts=A), "overlap"),
    (reserve, dict(counts=B), "overlap"), (reserve, dict(nxt=C.c_void_p(8192 + 4)), "overlap"),
    (reserve, dict(nxt=D, counts=D), "overlap"),
    (share, dict(src=None), "NULL sources"), (share, dict(counts=None), "NULL sources or counts"),
    (share, dict(src=A), "overlap"), (share, dict(counts=A), "overlap"), (share, dict(nxt=A), "overlap"),
    (share, dict(nxt=B), "overlap"), (share, dict(nxt=D), "overlap"),
], ids=lambda x: getattr(x, "__name__", None) or (x if isinstance(x, str) else ""))
def test_bad_arguments(L, call, kw, reason):
    assert call(L, **kw) == -1
    assert reason in L.last_error()


@pytest.mark.parametrize("call,kw", [
    (append, dict(tokens=0, q=None, k=None, v=None, slots=None, pos=None, qo=None)),
    (shared, dict(rows=0, q=None, out=None, tab=None, ln=None, starts=None, prefix=None, groups=0)),
    (bounds, dict(rows=0, to=None, tab=None, ln=None)), (bounds, dict(most=0)),
    (pick, dict(rows=0, q=None, bd=None, tab=None, ln=None, to=None, new=None)),
    (picked, dict(rows=0, q=None, out=None, tab=None, ln=None)),
    (reserve, dict(rows=0, refs=None, tab=None, ln=None, starts=None, granted=None, slots=None)),
    (release, dict(rows=0, refs=None, tab=None, ln=None)), (share, dict(rows=0, refs=None, tab=None, ln=None, src=None, counts=None)),
], ids=lambda x: getattr(x, "__name__", ""))
def test_nothing_to_do(L, call, kw):
    assert call(L, **kw) == 0
    assert L.last_error() == ""


# ------------------------------------------------------------- the binding
BF, I32 = torch.bfloat16, torch.int32


@pytest.fixture
def cache(L):
    return L.kv_cache(8, 16, 2, 64, device="cpu")


def rows(n=3, heads=4, dim=64):
    return torch.zeros((n, heads, dim), dtype=BF)


def ints(*shape):
    return torch.zeros(shape, dtype=I32)


def test_append_binding(L, cache):
    r = L.rotary(64, device="cpu")
    ok = dict(rotary=r, q=rows(), k=rows(heads=2), v=rows(heads=2), slots=ints(3), positions=ints(3))
    for kw, reason in ((dict(k=rows(heads=4)), "k must"), (dict(v=rows(2, 2)), "v 2"), (dict(q=rows(2)), "q 2"),
                       (dict(q_out=rows(2)), "q_out has 2"), (dict(q_out=rows(heads=2)), "q_out must"),
                       (dict(slots=ints(4)), "slots must"), (dict(positions=ints(3).long()), "positions must"),
                       (dict(rotary=None), "rotary must"), (dict(rotary=L.rotary(128, device="cpu")), "rotary must"),
                       (dict(k_stored=rows(heads=4), v_stored=rows(heads=2)), "k_stored must"), ({}, "run on a GPU")):
        with pytest.raises(ValueError, match=reason):
            cache.append_rotated(**{**ok, **kw})


def test_shared_binding(cache):
    ok = dict(q=rows(), out=rows(), tables=ints(3, 4), lengths=ints(3), max_length=64, groups=ints(2), prefix=ints(1),
              max_prefix=32, max_own=32)
    for kw, reason in ((dict(out=rows(2)), "out 2"), (dict(prefix=3), "prefix must"), (dict(groups=ints(3)), "groups must"),
                       (dict(prefix=ints(1).long()), "prefix must"), (dict(max_length=-1), "max_length"),
                       (dict(max_prefix=-1), "max_prefix"), (dict(max_own=1 << 64), "max_own"), (dict(q=rows().float()), "q must"),
                       ({}, "run on a GPU")):
        with pytest.raises(ValueError, match=reason):
            cache.attention_shared(**{**ok, **kw})


def test_pick_binding(cache):
    bd = torch.zeros((8, 2, 2, 64), dtype=BF)
    ok = dict(q=rows(), bounds=bd, tables=ints(3, 4), lengths=ints(3), max_length=64, picked=ints(3, 2, 2),
              picked_lengths=ints(3))
    for kw, reason in ((dict(bounds=bd[:7]), "bounds must"), (dict(picked=ints(3, 1, 2)), "picked must"),
                       (dict(picked=ints(2, 2, 2), picked_lengths=ints(2)), "picked 2"), (dict(picked=None), "picked must"),
                       (dict(picked_lengths=ints(2)), "picked_lengths must"), (dict(first=-1), "first"), ({}, "run on a GPU")):
        with pytest.raises(ValueError, match=reason):
            cache.pick(**{**ok, **kw})
    with pytest.raises(ValueError, match="bounds must"):
        cache.key_bounds(bd.float(), ints(3, 4), ints(3))
    with pytest.raises(ValueError, match="counts must"):
        cache.key_bounds(bd, ints(3, 4), ints(3), counts=ints(2))
    with pytest.raises(ValueError, match="max_count"):
        cache.key_bounds(bd, ints(3, 4), ints(3), max_count=-1)
    with pytest.raises(ValueError, match="out 2"):
        cache.attention_picked(rows(), rows(2), ints(3, 2, 2), ints(3))
    with pytest.raises(ValueError, match="run on a GPU"):
        cache.attention_picked(rows(), rows(), ints(3, 2, 2), ints(3))


def test_pages_binding(L):
    for refs, size in ((ints(8).long(), 16), (ints(8, 2), 16), (ints(16)[::2], 16), (None, 16), (ints(8), -1)):
        with pytest.raises(ValueError):
            L.kv_pages_from(refs, size)
    p = L.kv_pages(8, 16, device="cpu")
    tab, n = ints(3, 4), ints(3)
    for call, kw, reason in ((p.reserve, dict(slots=5), "slots must"), (p.reserve, dict(slots=ints(3).long()), "slots must"),
                             (p.reserve, dict(slots=ints(3), positions=ints(4)), "positions must"),
                             (p.reserve, dict(slots=ints(3), counts=ints(2)), "counts must"),
                             (p.reserve, dict(slots=ints(3), next_pos=ints(2)), "next_pos must"),
                             (p.reserve, dict(slots=ints(3), starts=ints(3)), "starts must"),
                             (p.reserve, dict(slots=ints(3), granted=ints(4)), "granted must"),
                             (p.share, dict(sources=ints(2), counts=n), "sources must"),
                             (p.share, dict(sources=n, counts=ints(2)), "counts must"),
                             (p.share, dict(sources=n, counts=n, next_pos=ints(2)), "next_pos must"),
                             (p.release, {}, "run on a GPU")):
        with pytest.raises(ValueError, match=reason):
            call(tab, n, **kw)
    with pytest.raises(ValueError, match="tables must"):
        p.release(ints(3), n)
    with pytest.raises(ValueError, match="lengths must"):
        p.release(tab, ints(2))
