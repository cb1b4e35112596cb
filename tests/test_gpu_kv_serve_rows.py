"""examples/kv_serve.py with rows that do not share the prompt, or share another length of
it: every step's attention against float64 over each row's own table."""
import numpy as np
import pytest
import torch

import kv_ref
from test_gpu_kv_serve import DEV, make, pool_of, tokens

pytestmark = pytest.mark.gpu


def step_and_check(block, g):
    x = tokens(g, 5)
    block.step(x)
    torch.cuda.synchronize()
    raw = block.project(x[1:])[0]
    q = torch.empty((4, 8, 64), dtype=torch.bfloat16, device=DEV)
    block.rotary.apply(raw, None, block.next_pos[1:] - 1, q)
    qn, pool = q.cpu().double().numpy(), pool_of(block.cache)
    tables, lengths = block.tables[1:].cpu().numpy(), block.lengths[1:].cpu().numpy()
    assert lengths.tolist() == block.held[1:]
    want, tol, _, _ = kv_ref.attention(pool, qn, tables, lengths, 0.125)
    size, _, _, _ = kv_ref.attention(kv_ref.Pool(pool.k, np.abs(pool.v), pool.ks, pool.vs), qn, tables, lengths, 0.125)
    got = block.out[1:].cpu().double().numpy()
    assert (np.abs(got - want) <= tol + 64 * 2.0 ** -24 * size + 2.0 ** -8 * np.abs(want)).all()


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_rows_that_do_not_share(lib, dtype):
    """A row that ends and begins with a prompt of its own, longer than the common one; one
    that ends and decodes from nothing to beyond it."""
    block = make(lib, dtype, 0, pages=90)
    g = torch.Generator(device=DEV).manual_seed(11)
    block.extend(tokens(g, 40), [40, 0, 0, 0, 0])
    block.share(range(1, 5))
    block.extend(tokens(g, 14), [0, 2, 3, 4, 5])
    step_and_check(block, g)
    block.end([2, 4])
    block.extend(tokens(g, 100), [0, 0, 100, 0, 0])
    for _ in range(40):
        step_and_check(block, g)


def test_rows_that_share_more_of_a_longer_prompt(lib):
    block = make(lib, "bf16", 0, pages=90)
    g = torch.Generator(device=DEV).manual_seed(12)
    block.extend(tokens(g, 40), [40, 0, 0, 0, 0])
    block.share([1, 2])
    block.extend(tokens(g, 60), [30, 20, 10, 0, 0])
    block.share([3, 4])
    assert block.common == 64
    block.extend(tokens(g, 50), [0, 20, 20, 5, 5])
    for _ in range(3):
        step_and_check(block, g)
