"""What the KVCache binding itself refuses and arranges, on CPU tensors: nothing
reaches the device."""
import pytest
import torch

import sneppx_quant as sq


@pytest.fixture(scope="module")
def L():
    return sq.load()


def i32(*s):
    return torch.zeros(s, dtype=torch.int32)


def bf(*s):
    return torch.zeros(s, dtype=torch.bfloat16)


def calls(c, stream=0, max_length=64, budget=10, recent=3):
    """Calls whose arguments are right."""
    tab, ln = i32(3, 4), i32(3)
    return {"append": lambda: c.append(bf(3, 2, 64), bf(3, 2, 64), tab, ln, ln, stream=stream),
            "attention": lambda: c.attention(bf(3, 8, 64), bf(3, 8, 64), tab, ln, max_length, stream=stream),
            "evict": lambda: c.evict(tab, ln, ln, i32(3), max_length, budget, recent, stream=stream)}


@pytest.mark.parametrize("call", ["append", "attention", "evict"])
@pytest.mark.parametrize("stream", [None, 0])
def test_a_cache_in_host_memory_runs_nothing(L, call, stream):
    c = L.kv_cache(8, 16, 2, 64, weights=True, positions=True, device="cpu")
    with pytest.raises(ValueError, match="on cpu"):
        calls(c, stream)[call]()


@pytest.mark.parametrize("kw", [dict(max_length=-1), dict(max_length=1 << 64), dict(budget=-1), dict(budget=(1 << 64) + 10),
                                dict(recent=-1), dict(recent=1 << 64)], ids=str)
def test_numbers_that_are_no_counts(L, kw):
    """Negative numbers and those that 64 bits do not hold (they would reach the library
    as the largest ones, or as small ones)."""
    c = L.kv_cache(8, 16, 2, 64, weights=True, positions=True, device="cpu")
    name = next(iter(kw))
    with pytest.raises(ValueError, match=f"{name} must be a count"):
        calls(c, **kw)["evict"]()
    if name == "max_length":
        with pytest.raises(ValueError, match="max_length must be a count"):
            calls(c, **kw)["attention"]()


@pytest.mark.parametrize("call", ["append", "attention", "evict"])
@pytest.mark.parametrize("stream", [None, 77])
@pytest.mark.parametrize("current", [0, 1])
def test_calls_run_on_the_caches_device(L, monkeypatch, call, stream, current):
    """The library takes workspaces of the current device, which has to be the cache's
    whichever it was before, and is that again afterwards.  (Devices by number alone.)"""
    c = L.kv_cache(8, 16, 2, 64, weights=True, positions=True, device="cpu")
    now, seen = [current], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    c._index = 1
    setattr(c, f"_{call}", lambda *args: seen.append((now[0], args[-1])) or 0)
    calls(c, stream)[call]()
    assert seen == [(1, 101 if stream is None else 77)] and now == [current]
