"""Calls of no rows or no tokens do nothing, also through empty arrays, whose
address is NULL.  CPU only: nothing reaches the device."""
import ctypes as C

import pytest
import torch

import sneppx_quant as sq

P = C.c_void_p(64)                     # stand-in device pointer, never read


@pytest.fixture(scope="module")
def L():
    return sq.load()


@pytest.fixture(scope="module")
def struct():
    return sq._KVCacheStruct(k=64, v=64, weights=64, positions=64, dtype=sq.SNEPPX_BFLOAT16, pages=8, page_size=16,
                             kv_heads=2, head_dim=64)


def test_an_empty_tensor_has_no_address():
    assert torch.empty((0, 2, 64)).data_ptr() == 0


@pytest.mark.parametrize("width", [0, 4])
def test_no_rows(L, struct, width):
    c = C.byref(struct)
    L.check(L.fn["SNEPPX_kv_append"](c, None, 128, None, 128, 0, None, None, None, None, width, None, None, 0, None), "append")
    L.check(L.fn["SNEPPX_kv_append"](c, None, 128, None, 128, 0, P, None, None, None, width, None, None, 0, None), "append")
    L.check(L.fn["SNEPPX_kv_attention"](c, None, 512, None, 512, 0, None, width, None, 0, 8, 64, 0.1, 1, None), "attention")
    L.check(L.fn["SNEPPX_kv_evict"](c, None, width, None, None, None, 0, 64, 10, 3, None), "evict")


def test_no_tokens(L, struct):
    L.check(L.fn["SNEPPX_kv_append"](C.byref(struct), None, 128, None, 128, 0, P, None, None, P, 4, P, P, 3, None), "append")


def test_what_is_not_empty_is_still_needed(L, struct):
    c = C.byref(struct)
    assert L.fn["SNEPPX_kv_append"](c, None, 128, None, 128, 0, P, None, None, None, 4, P, P, 3, None) == -1
    assert "NULL block_tables" in L.last_error()
    assert L.fn["SNEPPX_kv_append"](c, None, 128, P, 128, 1, P, None, None, P, 4, P, P, 3, None) == -1
    assert "NULL pointer" in L.last_error()
    assert L.fn["SNEPPX_kv_attention"](c, None, 512, None, 512, 0, None, 4, None, 0, 7, 64, 0.1, 1, None) == -1
    assert "multiple of" in L.last_error()
    assert L.fn["SNEPPX_kv_evict"](c, None, 4, None, None, None, 0, 64, 0, 0, None) == -1
    assert "budget == 0" in L.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_no_rows_and_no_tokens_through_the_binding(lib, dtype):
    print(f"[gpu] kv calls of nothing {dtype}", flush=True)
    dev = "cuda"
    c = lib.kv_cache(8, 16, 2, 64, dtype, weights=True, positions=True, device=dev)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)      # noqa: E731
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=dev)    # noqa: E731
    for t in (c.k, c.v, c.weights, c.positions):
        t.fill_(3)
    for width in (0, 4):
        tab = i32(0, width)
        c.append(bf(0, 2, 64), bf(0, 2, 64), tab, i32(0), i32(0))
        c.append(bf(0, 2, 64), bf(0, 2, 64), tab, i32(0), i32(0), starts=i32(1), k_stored=bf(0, 2, 64), v_stored=bf(0, 2, 64))
        c.attention(bf(0, 8, 64), bf(0, 8, 64), tab, i32(0), 64, accumulate=True)
        c.evict(tab, i32(0), i32(0), i32(0), 64, 10, 3)
        c.evict(tab, i32(0), i32(0), None, 64, 10, 3)
    c.append(bf(0, 2, 64), bf(0, 2, 64), i32(3, 4), i32(3), i32(3), starts=i32(4))
    torch.cuda.synchronize()
    for t in (c.k, c.v, c.weights, c.positions):
        assert bool((t == 3).all())
