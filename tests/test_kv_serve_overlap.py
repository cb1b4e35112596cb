"""Page and pick calls refuse arrays that overlap where one is written while another is
read, before they touch the device.  CPU only (the pointers are never dereferenced)."""
import ctypes as C

import pytest
import torch

from test_kv_serve_args import L, pick, reserve  # noqa: F401

# ten entries apart, more than any array below has
AT = dict(refs=1 << 20, tab=2 << 20, ln=40960, nxt=41000, counts=41040, starts=41080, granted=41120, slots=41160, pos=41200)
ENTRIES = dict(ln=3, nxt=3, counts=3, starts=4, granted=3, slots=5, pos=5)


def args(**at):
    return {k: C.c_void_p(v) for k, v in {**AT, **at}.items()}


@pytest.mark.parametrize("a", ENTRIES)
@pytest.mark.parametrize("b", ENTRIES)
def test_reserve(L, a, b):  # noqa: F811
    if a == b:
        return
    for to in (AT[b], AT[b] + 4 * (ENTRIES[b] - 1), AT[b] - 4 * (ENTRIES[a] - 1)):
        assert reserve(L, tokens=5, **args(**{a: to})) == -1
        assert "overlap" in L.last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the call goes on to a launch, which only a machine without a GPU refuses")
def test_arrays_of_no_entries_meet_nothing(L):  # noqa: F811
    """No tokens: where slots and positions would be does not matter."""
    assert reserve(L, tokens=0, **args(slots=AT["counts"] + 4, pos=AT["starts"] + 4)) == -1
    assert "overlap" not in L.last_error()


def test_pick(L):  # noqa: F811
    """3 rows of 4 entries; 2 heads, so picked [3][2][3]."""
    tab, ln, to, new = 40960, 50000, 60000, 70000

    def call(tab=tab, ln=ln, to=to, new=new):
        assert pick(L, tab=C.c_void_p(tab), ln=C.c_void_p(ln), to=C.c_void_p(to), new=C.c_void_p(new)) == -1
        assert "overlap" in L.last_error()
    for kw in (dict(to=tab), dict(to=tab + 44), dict(to=tab - 68), dict(new=tab), dict(new=tab + 44), dict(to=ln), dict(to=ln + 8),
               dict(to=ln - 68), dict(new=to), dict(new=to + 68), dict(new=to - 8), dict(new=ln)):
        call(**kw)
