"""The rotary entry points reject bad arguments before they touch the device, and the
frequencies of the scalings are those of their formulas.  CPU only (the pointers
passed are never dereferenced: every check runs first)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import sneppx_quant as sq


@pytest.fixture(scope="module")
def L():
    return sq.load()


P = C.c_void_p(64)                     # stand-in device pointer, never read


def rotary(**kw):
    f = dict(freqs=64, dims=64, interleaved=0, magnitude=1.0, q_norm=None, k_norm=None, eps=1e-6)
    f.update(kw)
    return sq._RotaryStruct(**f)


def apply(L, r=None, q=P, qs=512, qo=P, qos=512, hq=4, k=P, ks=512, ko=P, kos=512, hk=2, dim=64, pos=P, tokens=3):
    r = r if r is not None else rotary()
    return L.fn["SNEPPX_rotary_apply"](C.byref(r) if r else None, q, qs, qo, qos, hq, k, ks, ko, kos, hk, dim, pos, tokens,
                                       None)


@pytest.mark.parametrize("kw,reason", [
    (dict(r=False), "NULL rotary"), (dict(r=rotary(freqs=None)), "NULL freqs"), (dict(r=rotary(dims=60)), "multiple of 8"),
    (dict(r=rotary(dims=72)), "up to head_dim 64"), (dict(r=rotary(freqs=72)), "16-byte aligned"),
    (dict(r=rotary(q_norm=68)), "16-byte aligned"), (dict(r=rotary(k_norm=68)), "16-byte aligned"),
    (dict(dim=0), "head_dim"), (dict(dim=68), "multiple of 8"), (dict(dim=264), "up to 256"), (dict(hq=1 << 20), "too many"),
    (dict(hk=1 << 20), "too many"), (dict(tokens=1 << 40), "too many"), (dict(pos=None), "NULL positions"),
    (dict(q=None), "NULL q"), (dict(qo=None), "NULL q"), (dict(k=None), "NULL k"), (dict(ko=None), "NULL k"),
    (dict(qs=255), "below its row"), (dict(qos=255), "below its row"), (dict(ks=127), "below its row"),
    (dict(kos=127), "below its row"), (dict(qos=520), "q in place"), (dict(kos=520), "k in place"),
])
def test_bad_arguments(L, kw, reason):
    assert apply(L, **kw) == -1
    assert reason in L.last_error()


@pytest.mark.parametrize("kw", [dict(tokens=0), dict(hq=0, hk=0, q=None, k=None, qo=None, ko=None),
                                dict(tokens=0, q=None, qo=None, k=None, ko=None, pos=None)])
def test_nothing_to_do(L, kw):
    assert apply(L, **kw) == 0


def freqs(L, *a, **kw):
    return L.rotary_frequencies(*a, **kw)


def test_plain_frequencies(L):
    f, m = freqs(L, 128, 500000.0)
    assert m == 1.0
    np.testing.assert_allclose(f, 500000.0 ** (-np.arange(64) / 64), rtol=1e-14)


def test_linear_and_base(L):
    plain, _ = freqs(L, 64)
    f, m = freqs(L, 64, scaling="linear", factor=4.0)
    np.testing.assert_allclose(f, plain / 4, rtol=1e-14)
    assert m == 1.0
    f, m = freqs(L, 64, scaling="base", factor=4.0)
    np.testing.assert_allclose(f, (10000.0 * 4 ** (64 / 62)) ** (-np.arange(32) / 32), rtol=1e-13)
    np.testing.assert_allclose([f[0], f[-1]], [1.0, plain[-1] / 4], rtol=1e-12)
    assert m == 1.0


def test_bands(L):
    plain, _ = freqs(L, 128, 500000.0)
    f, m = freqs(L, 128, 500000.0, scaling="bands", factor=8.0, original=8192, low=1.0, high=4.0)
    turns = 8192 * plain / (2 * math.pi)
    want = np.where(turns >= 4, plain, np.where(turns <= 1, plain / 8,
                                                (1 - (turns - 1) / 3) * plain / 8 + (turns - 1) / 3 * plain))
    np.testing.assert_allclose(f, want, rtol=1e-13)
    assert m == 1.0 and (f == plain).any() and np.isclose(f, plain / 8, rtol=1e-14).any()


def test_ramp(L):
    plain, _ = freqs(L, 128)
    f, m = freqs(L, 128, scaling="ramp", factor=16.0, original=4096, low=1.0, high=32.0)

    def pair(turns):
        return 128 * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(10000.0))
    first, last = math.floor(pair(32)), math.ceil(pair(1))
    r = np.clip((np.arange(64) - first) / (last - first), 0, 1)
    np.testing.assert_allclose(f, plain * (1 - r) + plain / 16 * r, rtol=1e-13)
    assert m == np.float32(0.1 * math.log(16) + 1)


@pytest.mark.parametrize("kw,reason", [
    (dict(dims=63), "do not pair"), (dict(base=1.0), "above 1"), (dict(base=math.nan), "above 1"),
    (dict(scaling="linear", factor=0.5), "factor"), (dict(scaling="linear", factor=math.inf), "factor"),
    (dict(dims=2, scaling="base", factor=2.0), "single pair"), (dict(scaling="bands", factor=2.0), "original"),
    (dict(scaling="ramp", factor=2.0, original=100.0, low=4.0, high=4.0), "low"),
    (dict(scaling="bands", factor=2.0, original=100.0, low=0.0), "low"),
])
def test_bad_frequencies(L, kw, reason):
    with pytest.raises(sq.SneppxError, match=reason):
        L.rotary_frequencies(**{"dims": 64, **kw})


def test_unknown_scaling(L):
    out = (C.c_double * 4)()
    assert L.fn["SNEPPX_rotary_frequencies"](out, None, 8, 10000.0, 5, 1.0, 1.0, 1.0, 2.0) == -1
    assert "unknown scaling" in L.last_error()
    with pytest.raises(ValueError, match="scaling"):
        L.rotary_frequencies(64, scaling="other")
    with pytest.raises(ValueError, match="dims"):
        L.rotary_frequencies(-2)


def test_binding_refuses(L):
    f = torch.zeros(32, dtype=torch.float64)
    with pytest.raises(ValueError, match="freqs"):
        L.rotary_from(f.float(), 64)
    with pytest.raises(ValueError, match="freqs"):
        L.rotary_from(torch.zeros(64, dtype=torch.float64)[::2], 64)
    with pytest.raises(ValueError, match="q_norm"):
        L.rotary_from(f, 64, q_norm=torch.ones(32))
    with pytest.raises(ValueError, match="k_norm"):
        L.rotary_from(f, 64, k_norm=torch.ones(64, dtype=torch.float64))
    r = L.rotary_from(f, 64)
    q, pos = torch.zeros((3, 4, 64), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    for bad, reason in (((q.float(), None, pos), "q must"), ((q[..., :32], None, pos), "q must"),
                        ((q, q[:2], pos), "k has 2 tokens"), ((q, None, pos[:2]), "q has 3 tokens"),
                        ((q, None, pos.long()), "positions must"), ((q, None, pos, q[:, :2]), "q_out must"),
                        ((q, None, pos, q[:2]), "its output 2"), ((q, None, 3), "positions must")):
        with pytest.raises(ValueError, match=reason):
            r.apply(*bad)
    with pytest.raises(ValueError, match="run on a GPU"):
        r.apply(q, None, pos)
