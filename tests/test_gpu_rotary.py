"""SNEPPX_rotary_apply and SNEPPX_kv_append_rotated against the definition in float64
(serve_ref.turn).

Tolerances: serve_ref.turn's bound of fp32 rounding; a bf16 result adds 2^-8 of
itself.  An int8 code is off by half a step of its row's scale and what fp32 moves the
value (127 steps to the largest) and the two divisions by; a scale by the bound of the
row's largest value and two roundings."""
import numpy as np
import pytest
import torch

import serve_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def make(lib, tokens, hq, hk, dim, dims, norm, seed, far=8192, interleaved=False, magnitude=1.0, pad=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    rows = (torch.randn((tokens, (hq + 2 * hk) * dim + pad), generator=g) * std).to(BF).to(DEV)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in rows[:, : (hq + 2 * hk) * dim].split((hq * dim, hk * dim, hk * dim), 1))
    qn, kn = (None, None) if not norm else (1 + 0.3 * torch.randn(dim, generator=g) for _ in range(2))
    freqs = torch.from_numpy(lib.rotary_frequencies(dims, 500000.0)[0])
    pos = torch.randint(0, far, (tokens,), generator=g, dtype=torch.int32)
    r = lib.rotary_from(freqs.to(DEV), dim, interleaved, magnitude, None if qn is None else qn.to(DEV),
                        None if kn is None else kn.to(DEV), 1e-5)

    def want(x, n):
        return serve_ref.turn(x.cpu().double().numpy(), pos.numpy(), freqs.numpy(), interleaved, r._c.magnitude,
                              None if n is None else n.double().numpy(), 1e-5)
    return r, q, k, v, pos.to(DEV), want(q, qn), want(k, kn)


def close(got, want, tol):
    got = got.cpu().double().numpy()
    tol = tol + 2.0 ** -8 * np.abs(want) + 1e-38
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


CASES = [
    # tokens, q heads, kv heads, dim, dims, norm, interleaved, far
    (1, 32, 8, 128, 128, False, False, 10),
    (1, 1, 1, 8, 8, True, True, 10),
    (3, 3, 1, 80, 80, True, False, 100),
    (3, 3, 1, 80, 40, False, True, 100),
    (5, 5, 5, 96, 24, True, False, 8192),
    (7, 6, 2, 64, 16, True, True, 100000),
    (16, 32, 8, 128, 128, True, False, 131072),
    (33, 20, 1, 256, 64, True, False, 1000000),
    (33, 9, 3, 240, 240, False, True, 2 ** 31 - 1),
    (2, 0, 3, 128, 128, True, False, 50),
    (2, 3, 0, 128, 128, True, True, 50),
    (4, 4, 2, 64, 0, True, False, 50),
    (4, 4, 2, 64, 0, False, False, 50),
    (1500, 32, 8, 128, 64, True, True, 8192),       # several heads to a lane
    (1301, 33, 1, 64, 64, False, False, 8192),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("inplace", [False, True])
def test_apply(lib, case, inplace):
    print(f"[gpu] rotary {case} inplace={inplace}", flush=True)
    tokens, hq, hk, dim, dims, norm, inter, far = case
    r, q, k, v, pos, (wq, tq), (wk, tk) = make(lib, tokens, hq, hk, dim, dims, norm, 3 * dim + hq, far, inter, 1.3)
    before = v.clone()
    if inplace:
        r.apply(q if hq else None, k if hk else None, pos)
        qo, ko = q, k
    else:
        qo, ko = (torch.full(x.shape, 7.0, dtype=BF, device=DEV) for x in (q, k))
        kept = q.clone(), k.clone()
        r.apply(q if hq else None, k if hk else None, pos, qo if hq else None, ko if hk else None)
        assert torch.equal(q, kept[0]) and torch.equal(k, kept[1])
    torch.cuda.synchronize()
    if hq:
        close(qo, wq, tq)
    if hk:
        close(ko, wk, tk)
    assert torch.equal(v, before)          # what lies beside them in the rows


@pytest.mark.parametrize("pad", [1, 3, 4, 8])
def test_rows_of_any_alignment(lib, pad):
    r, q, k, _, pos, (wq, tq), (wk, tk) = make(lib, 9, 4, 2, 72, 72, True, pad, pad=pad)
    wide = torch.zeros((9, 6 * 72 + pad), dtype=BF, device=DEV)
    qo, ko = wide[:, : 4 * 72].unflatten(1, (4, 72)), wide[:, 4 * 72: 6 * 72].unflatten(1, (2, 72))
    r.apply(q, k, pos, qo, ko)
    torch.cuda.synchronize()
    close(qo, wq, tq)
    close(ko, wk, tk)
    assert (wide[:, 6 * 72:] == 0).all()


def test_far_positions_keep_their_angle(lib):
    """A turn by -position after one by position gives the heads back, as far as one
    rounding to bf16 in between does."""
    r, q, _, _, pos, _, _ = make(lib, 64, 4, 0, 128, 128, False, 1, far=2 ** 31 - 1)
    there, back = torch.empty_like(q), torch.empty_like(q)
    r.apply(q, None, pos, there)
    r.apply(there, None, -pos, back)
    torch.cuda.synchronize()
    x = q.cpu().double().numpy()
    a, b = np.abs(x[..., :64]), np.abs(x[..., 64:])
    size = np.concatenate([a + b, a + b], -1)
    # (two roundings to bf16, each of numbers no larger than a + b, the first turned once more)
    assert (np.abs(back.cpu().double().numpy() - x) <= 3 * 2.0 ** -8 * size).all()


def test_nan_and_infinity_stay_in_their_pair_or_head(lib):
    r, q, _, _, pos, (wq, tq), _ = make(lib, 4, 4, 0, 64, 32, False, 2)
    q[1, 2, 3] = float("nan")
    q[2, 1, 40] = float("inf")
    out = torch.empty_like(q)
    r.apply(q, None, pos, out)
    o = out.cpu()
    assert torch.isnan(o[1, 2, 3]) and torch.isnan(o[1, 2, 19]) and o[2, 1, 40] == float("inf")
    bad = torch.isnan(o) | torch.isinf(o)
    assert int(bad.sum()) == 3
    keep = ~bad.numpy()
    assert (np.abs(o.double().numpy() - wq)[keep] <= (tq + 2.0 ** -8 * np.abs(wq))[keep]).all()


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("case", [c for c in CASES if c[2] and (c[3] % 16 == 0)], ids=str)
def test_append(lib, case, dtype):
    print(f"[gpu] kv_append_rotated {case} {dtype}", flush=True)
    tokens, hq, hk, dim, dims, norm, inter, far = case
    r, q, k, v, pos, (wq, tq), (wk, tk) = make(lib, tokens, hq, hk, dim, dims, norm, 5 * dim + hq, far, inter)
    page = 16 if tokens > 20 else 3
    pages = -(-tokens // page) + 2
    c = lib.kv_cache(pages, page, hk, dim, dtype, weights=True, positions=True)
    for x in (c.k, c.v):
        x.fill_(7)
    c.weights.fill_(3.0)
    c.positions.fill_(-5)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:tokens].to(torch.int32)
    if tokens > 2:
        slots[1], slots[tokens - 1] = -1, pages * page      # no slot, and one outside the pool
    stored = tokens != 3
    ko, vo = (torch.full((tokens, hk, dim), 7.0, dtype=BF, device=DEV) if stored else None for _ in range(2))
    qo = torch.empty((tokens, hq, dim), dtype=BF, device=DEV)
    c.append_rotated(r, q if hq else None, k, v, slots.to(DEV), pos, qo if hq else None, ko, vo)
    torch.cuda.synchronize()
    if hq:
        close(qo, wq, tq)
    s = slots.numpy()
    keep = (s >= 0) & (s < pages * page)
    pg, off = s[keep] // page, s[keep] % page
    used = np.zeros((pages, page), bool)
    used[pg, off] = True
    hole = torch.from_numpy(~used).to(DEV)
    for name, want, tol, out in (("k", wk, tk, ko), ("v", v.cpu().double().numpy(), 0.0, vo)):
        pool = getattr(c, name)
        want, tol = want[keep], np.broadcast_to(tol, want.shape)[keep]
        got = pool.cpu().double().numpy()[pg, :, off]
        if dtype == "int8":
            scale = getattr(c, name + "_scales").cpu().double().numpy()[pg, :, off]
            top = np.abs(want).max(-1)
            assert (np.abs(scale - top / 127) <= tol.max(-1) / 127 + 2.0 ** -22 * top).all()
            # (in steps: half of one, and the value's and the divisions' rounding)
            off_by = np.abs(got - want / scale[..., None])
            assert (off_by <= 0.5 + tol / scale[..., None] + 127 * 2.0 ** -21).all(), off_by.max()
            got = got * scale[..., None]
            if stored:
                assert (np.abs(out.cpu().double().numpy()[keep] - got) <= 2.0 ** -8 * np.abs(got) + 1e-38).all()
        else:
            assert (np.abs(got - want) <= tol + 2.0 ** -8 * np.abs(want)).all()
            if name == "v":
                assert (got == want).all()
            if stored:
                assert (out.cpu().double().numpy()[keep] == got).all()
        if stored:
            assert (out.cpu().float().numpy()[~keep] == 7.0).all()
        assert (pool.transpose(1, 2)[hole] == 7).all()
    w, p = c.weights.cpu().numpy(), c.positions.cpu().numpy()
    assert (w[pg, :, off] == 0).all() and (p[pg, :, off] == pos.cpu().numpy()[keep][:, None]).all()
    assert (c.weights.transpose(1, 2)[hole] == 3).all() and (c.positions.transpose(1, 2)[hole] == -5).all()


def test_append_without_rotation_is_append(lib):
    """No norm, no turned part: the same bits as SNEPPX_kv_append leaves."""
    for dtype in ("bf16", "int8"):
        _, _, k, v, pos, _, _ = make(lib, 50, 4, 4, 64, 64, False, 9)
        r = lib.rotary(64, dims=0)
        a, b = (lib.kv_cache(8, 8, 4, 64, dtype) for _ in range(2))
        tables = torch.randperm(8, generator=torch.Generator().manual_seed(2)).to(torch.int32).view(1, 8).to(DEV)
        lengths = torch.tensor([50], dtype=torch.int32, device=DEV)
        starts = torch.tensor([0, 50], dtype=torch.int32, device=DEV)
        for x in (a, b):
            x.k.zero_()
            x.v.zero_()
        a.append(k, v, tables, lengths, starts=starts)
        t = torch.arange(50, device=DEV)
        slots = (tables[0, t // 8] * 8 + t % 8).to(torch.int32)
        b.append_rotated(r, None, k, v, slots, pos)
        torch.cuda.synchronize()
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
        if dtype == "int8":
            assert torch.equal(a.k_scales, b.k_scales) and torch.equal(a.v_scales, b.v_scales)
