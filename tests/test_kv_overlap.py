"""An eviction writes its new lengths while other workgroups still read the old ones
and the positions: arrays that overlap them are refused, before the device is
touched (the CPU tests' pointers are never read)."""
import ctypes as C

import pytest
import torch

import sneppx_quant as sq


@pytest.mark.parametrize("new", [4096, 4096 + 4, 4096 + 8, 4096 - 4, 4096 - 8])
def test_overlap(new):
    """Three rows of four bytes."""
    L = sq.load()
    c = sq._KVCacheStruct(k=64, v=64, weights=64, positions=64, dtype=sq.SNEPPX_BFLOAT16, pages=8, page_size=16, kv_heads=2,
                          head_dim=64)
    for lengths, next_pos, name in ((4096, 8192, "lengths"), (8192, 4096, "next_pos")):
        assert L.fn["SNEPPX_kv_evict"](C.byref(c), 64, 4, lengths, next_pos, new, 3, 64, 10, 3, None) == -1
        assert f"must not be {name}" in L.last_error()


@pytest.mark.gpu
def test_beside_one_another(lib):
    print("[gpu] kv_evict arrays side by side", flush=True)
    dev, rows = "cuda", 3
    c = lib.kv_cache(rows * 4, 16, 2, 64, weights=True, positions=True, device=dev)
    for t in (c.k, c.v, c.weights, c.positions):
        t.fill_(1)
    tables = torch.arange(rows * 4, dtype=torch.int32, device=dev).view(rows, 4)
    for order in ((0, 1, 2), (1, 0, 2), (2, 0, 1), (0, 2, 1)):
        three = torch.full((3, rows), 7, dtype=torch.int32, device=dev)
        lengths, new, next_pos = (three[i] for i in order)
        lengths.copy_(torch.tensor([40, 10, 3], dtype=torch.int32))
        next_pos.fill_(50)
        c.evict(tables, lengths, next_pos, new, 64, 10, 3)
        torch.cuda.synchronize()
        assert lengths.tolist() == [40, 10, 3] and next_pos.tolist() == [50] * 3 and new.tolist() == [10, 10, 3]
