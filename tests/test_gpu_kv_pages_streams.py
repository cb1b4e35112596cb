"""KVPages.reserve on a stream other than torch's current one, without starts and granted of
the caller's: the new ones are of that stream's memory, so that work still waiting on the
current one does not write over them."""
import numpy as np
import pytest
import torch

import serve_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("given", [(), ("starts",), ("granted",)], ids=lambda g: "-".join(g) or "none")
def test_new_outputs_belong_to_the_stream(lib, given):
    rows, page, pages = 1000, 4, 6000
    rng = np.random.default_rng(1)
    counts = rng.integers(0, 9, rows).astype(np.int32)
    p = lib.kv_pages(pages, page)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    tables, lengths, slots = ints(rows, 6) - 1, ints(rows), ints(int(counts.sum()))
    d_counts = torch.from_numpy(counts).to(DEV)
    own = {n: ints(rows + (n == "starts")) for n in given}
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    freed = [torch.empty(rows + 1, dtype=torch.int32, device=DEV) for _ in range(64)]
    torch.cuda._sleep(10_000_000)
    for t in freed:
        t.fill_(77)
    del freed, t
    starts, granted = p.reserve(tables, lengths, slots, counts=d_counts, stream=st.cuda_stream, **own)
    torch.cuda.synchronize()
    want = [np.zeros(pages, np.int64), -np.ones((rows, 6), np.int64), np.zeros(rows, np.int64)]
    w_starts, w_granted, w_slots, _ = serve_ref.reserve(want[0], page, want[1], want[2], None, counts, len(slots))
    assert np.array_equal(slots.cpu().numpy(), w_slots)
    assert np.array_equal(starts.cpu().numpy(), w_starts) and np.array_equal(granted.cpu().numpy(), w_granted)


def test_the_current_stream_by_its_number(lib):
    p = lib.kv_pages(8, 4)
    tables, lengths = torch.full((2, 3), -1, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    for st in (None, torch.cuda.current_stream().cuda_stream, torch.cuda.Stream().cuda_stream):
        torch.cuda.synchronize()
        starts, granted = p.reserve(tables, lengths, torch.zeros(2, dtype=torch.int32, device=DEV), stream=st)
        torch.cuda.synchronize()
        assert starts.tolist() == [0, 1, 2] and granted.tolist() == [1, 1]
    assert lengths.tolist() == [3, 3]


def test_recorded_without_outputs_of_the_callers(lib):
    """A stream that nothing was allocated for: nothing is allocated while it is recorded
    that the recording could not bear."""
    p = lib.kv_pages(80, 4)
    tables, lengths = torch.full((2, 9), -1, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    slots, st = torch.zeros(2, dtype=torch.int32, device=DEV), torch.cuda.Stream()
    spare = [torch.empty(3, dtype=torch.int32, device=DEV) for _ in range(4)]
    del spare
    torch.cuda.synchronize()
    kept = []
    graph = lib.capture(lambda: kept.append(p.reserve(tables, lengths, slots, stream=st.cuda_stream)), stream=st.cuda_stream)
    for i in range(1, 6):
        lib.graph_launch(graph, stream=st.cuda_stream)
        torch.cuda.synchronize()
        assert lengths.tolist() == [i, i] and kept[0][0].tolist() == [0, 1, 2] and kept[0][1].tolist() == [1, 1]
    lib.graph_destroy(graph)
