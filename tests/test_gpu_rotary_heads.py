"""Rotation where a lane has several heads of a token and not all lanes as many, in heads of
each width, for SNEPPX_rotary_apply and SNEPPX_kv_append_rotated; tolerances as in
test_gpu_rotary.py."""
import numpy as np
import pytest
import torch

from test_gpu_rotary import DEV, BF, close, make

pytestmark = pytest.mark.gpu

# tokens * heads * lanes of a head (8, 16 or 32) / 64 is above 8192, heads 1, 2 or 3 modulo 4
CASES = [
    # tokens, q heads, kv heads, dim, dims, norm, interleaved
    (2500, 30, 1, 64, 64, True, False),
    (3200, 20, 1, 48, 24, False, True),
    (1100, 32, 2, 128, 128, True, True),
    (1300, 25, 1, 80, 80, True, False),
    (600, 28, 1, 256, 128, True, False),
    (750, 21, 2, 240, 240, False, True),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_apply(lib, case):
    print(f"[gpu] rotary {case}", flush=True)
    tokens, hq, hk, dim, dims, norm, inter = case
    r, q, k, v, pos, (wq, tq), (wk, tk) = make(lib, tokens, hq, hk, dim, dims, norm, dim + hq, 8192, inter, 1.1)
    before = v.clone()
    qo, ko = (torch.full(x.shape, 7.0, dtype=BF, device=DEV) for x in (q, k))
    r.apply(q, k, pos, qo, ko)
    torch.cuda.synchronize()
    close(qo, wq, tq)
    close(ko, wk, tk)
    r.apply(q, k, pos)
    torch.cuda.synchronize()
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(v, before)


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_append(lib, case, dtype):
    print(f"[gpu] kv_append_rotated {case} {dtype}", flush=True)
    tokens, hq, hk, dim, dims, norm, inter = case
    r, q, k, v, pos, (wq, tq), (wk, tk) = make(lib, tokens, hq, hk, dim, dims, norm, 2 * dim + hq, 8192, inter, 1.1)
    page = 16
    pages = tokens // page + 2
    c = lib.kv_cache(pages, page, hk, dim, dtype)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:tokens].to(torch.int32)
    slots[5] = -1
    qo = torch.empty((tokens, hq, dim), dtype=BF, device=DEV)
    ko, vo = (torch.full((tokens, hk, dim), 7.0, dtype=BF, device=DEV) for _ in range(2))
    c.append_rotated(r, q, k, v, slots.to(DEV), pos, qo, ko, vo)
    torch.cuda.synchronize()
    close(qo, wq, tq)
    keep = np.arange(tokens) != 5
    pg, off = slots.numpy()[keep] // page, slots.numpy()[keep] % page
    for name, want, tol, out in (("k", wk, tk, ko), ("v", v.cpu().double().numpy(), 0.0, vo)):
        want, tol = want[keep], np.broadcast_to(tol, want.shape)[keep]
        got = getattr(c, name).cpu().double().numpy()[pg, :, off]
        if dtype == "int8":
            scale = getattr(c, name + "_scales").cpu().double().numpy()[pg, :, off]
            top = np.abs(want).max(-1)
            assert (np.abs(scale - top / 127) <= tol.max(-1) / 127 + 2.0 ** -22 * top).all()
            assert (np.abs(got - want / scale[..., None]) <= 0.5 + tol / scale[..., None] + 127 * 2.0 ** -21).all()
            got = got * scale[..., None]
            assert (np.abs(out.cpu().double().numpy()[keep] - got) <= 2.0 ** -8 * np.abs(got) + 1e-38).all()
        else:
            assert (np.abs(got - want) <= tol + 2.0 ** -8 * np.abs(want)).all()
            assert (out.cpu().double().numpy()[keep] == got).all()
        assert (out[5].float() == 7.0).all()
