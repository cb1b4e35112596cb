"""SNEPPX_kv_pick where rows have more pages than a workgroup takes at a time (4096), and
where a lane has several pages one after the other, against plain loops (serve_ref)."""
import numpy as np
import pytest
import torch

import serve_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(lib, have, heads, group, dim, budget, first, recent, seed, whole=False):
    """Rows of so many pages of one token each; `whole`: bounds and queries of a few whole
    numbers, so that many scores are equal."""
    g = torch.Generator().manual_seed(seed)
    pages = sum(have) + 3
    draw = (lambda *s: torch.randint(-2, 3, s, generator=g).float()) if whole else (lambda *s: torch.randn(s, generator=g))
    bounds = draw(pages, heads, 2, dim).sort(2)[0].to(torch.bfloat16)
    q = draw(len(have), heads * group, dim).to(torch.bfloat16)
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    tables = -torch.ones((len(have), max(have) + 2), dtype=torch.int32)
    at = 0
    for r, n in enumerate(have):
        tables[r, :n] = perm[at:at + n]
        at += n
    c = lib.kv_cache(pages, 1, heads, dim)
    picked = torch.full((len(have), heads, budget), 77, dtype=torch.int32, device=DEV)
    new = torch.zeros(len(have), dtype=torch.int32, device=DEV)
    c.pick(q.to(DEV), bounds.to(DEV), tables.to(DEV), torch.tensor(have, dtype=torch.int32, device=DEV), max(have), picked, new,
           first, recent)
    torch.cuda.synchronize()
    want, want_len = serve_ref.pick(q.double().numpy(), bounds.double().numpy(), tables.numpy(), have, 1, budget, first, recent)
    assert np.array_equal(new.cpu().numpy(), want_len)
    assert np.array_equal(picked.cpu().numpy(), want)


LONG = [
    # pages of the rows, budget, first, recent, equal scores
    ([10000], 60, 1, 2, False),
    ([10000], 5000, 0, 1, True),              # equal scores at the border, in all three chunks
    ([8192, 8193, 4096, 4097], 3000, 3, 1, True),
    ([12289], 10000, 4097, 5000, False),      # the first and the newest each beyond a chunk
    ([9000], 8999, 4096, 4902, True),         # all but one
    ([9000, 50], 4097, 1, 4096, True),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-{c[3]}{'-equal' if c[4] else ''}")
def test_rows_of_several_chunks(lib, case):
    have, budget, first, recent, whole = case
    print(f"[gpu] kv_pick {case}", flush=True)
    check(lib, have, 2, 2, 8, budget, first, recent, sum(have), whole)


@pytest.mark.parametrize("group", [1, 4, 5])
@pytest.mark.parametrize("dim,most", [(64, 17000), (40, 17000), (128, 9000), (80, 9000), (256, 4500), (200, 4500)])
def test_several_pages_to_a_lane(lib, dim, most, group):
    """From 16 waves a CU twice over on (256 CUs, 8, 16 or 32 lanes a page) a lane has two
    pages and more: ragged rows, one of which has nothing to pick and one no pages."""
    print(f"[gpu] kv_pick {most} pages of {dim}, {group} query heads", flush=True)
    have = [most, most - 1, most // 3, 30, 0]
    check(lib, have, 1, group, dim, 37, 2, 3, dim + group)
