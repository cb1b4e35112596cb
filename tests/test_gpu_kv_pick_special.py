"""SNEPPX_kv_pick at infinite bounds in heads that do not fill their lanes, at queries of
zero against infinite bounds, and at bounds far apart, against plain loops (serve_ref)."""
import math

import numpy as np
import pytest
import torch

import serve_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(lib, bounds, q, budget, first=0, recent=1):
    """bounds [pages][heads][2][dim], q [1][q_heads][dim]; one row of all pages."""
    pages, heads, _, dim = bounds.shape
    c = lib.kv_cache(pages, 4, heads, dim)
    tables = torch.arange(pages, dtype=torch.int32, device=DEV).view(1, pages)
    lengths = torch.tensor([4 * pages], dtype=torch.int32, device=DEV)
    picked = torch.zeros((1, heads, budget), dtype=torch.int32, device=DEV)
    new = torch.zeros(1, dtype=torch.int32, device=DEV)
    c.pick(q, bounds.to(DEV), tables, lengths, 4 * pages, picked, new, first, recent)
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        want, _ = serve_ref.pick(q.cpu().double().numpy(), bounds.double().numpy(), tables.cpu().numpy(), [4 * pages], 4,
                                 budget, first, recent)
    assert np.array_equal(picked.cpu().numpy(), want)


@pytest.mark.parametrize("group", [1, 3, 7])
@pytest.mark.parametrize("dim", [8, 40, 64, 80, 96, 128, 240])
def test_infinite_bounds(lib, dim, group):
    """They count where queries do: in the head's own elements."""
    g = torch.Generator().manual_seed(3 * dim + group)
    pages = 30
    b = torch.randn((pages, 1, 2, dim), generator=g).sort(2)[0]
    q = torch.randn((1, group, dim), generator=g)
    q[..., :3] = q[..., :3].abs() + 0.1
    for e, page in enumerate((3, 7, 8, 12, 20)):
        b[page, :, 0, e % 3] = -math.inf         # (no positive query takes these)
    b[16, :, 1, 1] = math.inf                    # (and all take this)
    for budget in (2, 10, 20, 28):
        check(lib, b.to(torch.bfloat16), q.to(torch.bfloat16).to(DEV), budget)


@pytest.mark.parametrize("group", [1, 3, 7])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_zeros_of_a_query_against_infinite_bounds(lib, dim, group):
    """0 * inf is NaN at either end, and ranks the page below every number."""
    g = torch.Generator().manual_seed(dim)
    pages = 30
    b = torch.randn((pages, 1, 2, dim), generator=g).sort(2)[0]
    q = torch.randn((1, group, dim), generator=g)
    q[..., 5] = 0.0
    b[3, :, 1, 5] = math.inf
    b[7, :, 0, 5] = -math.inf
    b[11, :, 1, 6] = math.inf              # (a number against infinity: infinite, and first)
    b[13, :, 0, 5], b[13, :, 1, 5] = -math.inf, math.inf
    for budget in (2, 10, 28, 29):
        check(lib, b.to(torch.bfloat16), q.to(torch.bfloat16).to(DEV), budget)


@pytest.mark.parametrize("group", [1, 3, 7])
@pytest.mark.parametrize("dim", [8, 64, 128, 256])
@pytest.mark.parametrize("power", [10, 30, 60, 100])
def test_bounds_far_apart(lib, power, dim, group):
    """Where a query takes the smaller end of a wide range, the other end does not count."""
    g = torch.Generator().manual_seed(power + dim)
    pages = 40
    b = torch.randn((pages, 2, 2, dim), generator=g).sort(2)[0]
    q = torch.randn((1, 2 * group, dim), generator=g)
    # element 1 reaches far down, and all queries point up there; element 2 the other way
    b[::2, :, 0, 1] = -(2.0 ** power)
    b[::3, :, 1, 2] = 2.0 ** power
    q[..., 1], q[..., 2] = q[..., 1].abs() + 0.1, -q[..., 2].abs() - 0.1
    check(lib, b.to(torch.bfloat16), q.to(torch.bfloat16).to(DEV), 9)


@pytest.mark.parametrize("dim", [64, 80])
def test_bounds_in_no_order(lib, dim):
    """Pages whose bounds were never written are ranked by what they hold, the larger product
    of each element, whichever end it is of."""
    g = torch.Generator().manual_seed(dim)
    b, q = torch.randn((50, 2, 2, dim), generator=g), torch.randn((1, 6, dim), generator=g)
    check(lib, b.to(torch.bfloat16), q.to(torch.bfloat16).to(DEV), 12)
