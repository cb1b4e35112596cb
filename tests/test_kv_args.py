"""The key-value cache's entry points reject bad arguments before they touch
the device: -1 and a reason.  CPU only (the pointers passed are never
dereferenced: every check runs first), and the binding's own checks on CPU
tensors."""
import ctypes as C

import pytest
import torch

import sneppx_quant as sq


@pytest.fixture(scope="module")
def L():
    return sq.load()


P = C.c_void_p(64)                     # stand-in device pointer, never read


def struct(**kw):
    f = dict(k=64, v=64, k_scales=None, v_scales=None, weights=64, positions=64, dtype=sq.SNEPPX_BFLOAT16, pages=8,
             page_size=16, kv_heads=2, head_dim=64)
    f.update(kw)
    return sq._KVCacheStruct(**f)


def append(L, cache=None, k=P, v=P, ks=128, vs=128, tokens=3, starts=None, ko=None, vo=None, tab=P, width=4, ln=P,
           nxt=P, rows=3):
    c = cache if cache is not None else struct()
    return L.fn["SNEPPX_kv_append"](C.byref(c) if c else None, k, ks, v, vs, tokens, starts, ko, vo, tab, width, ln, nxt,
                                    rows, None)


def attention(L, cache=None, q=P, qs=512, out=P, os=512, odt=0, tab=P, width=4, ln=P, rows=3, hq=8, most=64, acc=0):
    c = cache if cache is not None else struct()
    return L.fn["SNEPPX_kv_attention"](C.byref(c) if c else None, q, qs, out, os, odt, tab, width, ln, rows, hq, most,
                                       0.1, acc, None)


def evict(L, cache=None, tab=P, width=4, ln=P, nxt=P, new=None, rows=3, most=64, budget=10, recent=3):
    c = cache if cache is not None else struct()
    return L.fn["SNEPPX_kv_evict"](C.byref(c) if c else None, tab, width, ln, nxt, new, rows, most, budget, recent, None)


CACHES = [
    (False, "NULL cache"),
    (struct(k=None), "NULL pointer in the cache"),
    (struct(v=None), "NULL pointer in the cache"),
    (struct(k=72), "16-byte aligned"),
    (struct(dtype=sq.SNEPPX_FLOAT16), "neither bf16 nor int8"),
    (struct(dtype=sq.SNEPPX_INT8), "needs k_scales"),
    (struct(pages=0), "empty cache"),
    (struct(page_size=0), "empty cache"),
    (struct(head_dim=60), "multiple of 8"),
    (struct(head_dim=264), "multiple of 8"),
    (struct(dtype=sq.SNEPPX_INT8, k_scales=64, v_scales=64, head_dim=72), "multiple of 16"),
    (struct(pages=1 << 31), "too large"),
    (struct(pages=1 << 30, page_size=16), "too large"),
    (struct(kv_heads=1 << 20), "too large"),
]


@pytest.mark.parametrize("call", [append, attention, evict], ids=lambda f: f.__name__)
@pytest.mark.parametrize("cache,reason", CACHES, ids=lambda x: x if isinstance(x, str) else "")
def test_bad_caches(L, call, cache, reason):
    assert call(L, cache=cache) == -1
    assert reason in L.last_error()


@pytest.mark.parametrize("call", [append, attention, evict], ids=lambda f: f.__name__)
@pytest.mark.parametrize("kw,reason", [(dict(tab=None), "NULL block_tables"), (dict(ln=None), "NULL block_tables or lengths"),
                                       (dict(width=0), "empty block_tables"), (dict(width=1 << 40), "too large"),
                                       (dict(rows=1 << 32), "too many")])
def test_bad_rows(L, call, kw, reason):
    assert call(L, **kw) == -1
    assert reason in L.last_error()


@pytest.mark.parametrize("call,kw,reason", [
    (append, dict(k=None), "NULL pointer"),
    (append, dict(v=None), "NULL pointer"),
    (append, dict(ko=P), "go together"),
    (append, dict(nxt=None), "needs next_pos"),
    (append, dict(tokens=5), "without starts"),
    (append, dict(tokens=1 << 31, starts=P), "too many"),
    (append, dict(ks=100), "strides"),
    (attention, dict(q=None), "NULL pointer"),
    (attention, dict(out=None), "NULL pointer"),
    (attention, dict(odt=sq.SNEPPX_FLOAT16), "out_dtype"),
    (attention, dict(hq=7), "multiple of"),
    (attention, dict(hq=0), "multiple of"),
    (attention, dict(qs=100), "strides"),
    (attention, dict(os=511), "strides"),
    (attention, dict(acc=1, cache=struct(weights=None)), "accumulate needs"),
    (evict, dict(nxt=None), "NULL next_pos"),
    (evict, dict(cache=struct(weights=None)), "weights and positions"),
    (evict, dict(cache=struct(positions=None)), "weights and positions"),
    (evict, dict(budget=0), "budget == 0"),
    (evict, dict(recent=11), "beyond the budget"),
    (evict, dict(new=P), "must not be lengths"),
])
def test_bad_arguments(L, call, kw, reason):
    assert call(L, **kw) == -1
    assert reason in L.last_error()


def test_nothing_to_do(L):
    """No rows, no tokens: 0, without a device."""
    assert append(L, tokens=0, rows=0) == 0
    assert append(L, tokens=0, starts=P) == 0
    assert attention(L, rows=0) == 0
    assert evict(L, rows=0) == 0


def cache(L, **kw):
    return L.kv_cache(8, 16, 2, 64, device="cpu", **kw)


def test_binding_checks_the_cache(L):
    k = torch.zeros((8, 2, 16, 64), dtype=torch.bfloat16)
    plane = torch.zeros((8, 2, 16))
    for args in ((k.float(), k), (k[0], k[0]), (k, k[:, :1]), (k, k.transpose(0, 1).contiguous().transpose(0, 1)),
                 (k, k.to(torch.int8)), (k.to(torch.int8), k.to(torch.int8)), (k, k, plane, plane),
                 (k, k, None, None, plane.double()), (k, k, None, None, plane[:4]), (k, k, None, None, None, plane)):
        with pytest.raises(ValueError):
            L.kv_cache_from(*args)
    with pytest.raises(ValueError):
        L.kv_cache(8, 16, 2, 64, dtype="fp8", device="cpu")


def test_binding_checks_the_call(L):
    c = cache(L, weights=True, positions=True)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)     # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)   # noqa: E731
    tab, ln = i32(3, 4), i32(3)
    bad = [
        lambda: c.append(bf(3, 2, 32), bf(3, 2, 32), tab, ln, ln),
        lambda: c.append(bf(3, 2, 64).float(), bf(3, 2, 64), tab, ln, ln),
        lambda: c.append(bf(3, 2, 64), bf(2, 2, 64), tab, ln, ln),
        lambda: c.append(bf(3, 64, 2).transpose(1, 2), bf(3, 2, 64), tab, ln, ln),
        lambda: c.append(bf(3, 2, 64), bf(3, 2, 64), tab.long(), ln, ln),
        lambda: c.append(bf(3, 2, 64), bf(3, 2, 64), tab, i32(2), ln),
        lambda: c.append(bf(3, 2, 64), bf(3, 2, 64), tab, ln, ln, starts=i32(3)),
        lambda: c.append(bf(3, 2, 64), bf(3, 2, 64), tab, ln, ln, k_stored=bf(3, 2, 32), v_stored=bf(3, 2, 64)),
        lambda: c.attention(bf(3, 8, 64), bf(3, 4, 64), tab, ln, 64),
        lambda: c.attention(bf(2, 8, 64), bf(2, 8, 64), tab, ln, 64),
        lambda: c.attention(bf(3, 8, 64), bf(3, 8, 64).half(), tab, ln, 64),
        lambda: c.attention(bf(3, 8, 64), bf(3, 8, 64), tab[:, ::2], ln, 64),
        lambda: c.evict(tab, ln, None, None, 64, 10, 3),
        lambda: c.evict(tab, ln, ln, i32(4), 64, 10, 3),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
