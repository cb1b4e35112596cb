"""SNEPPX_kv_attention_shared over an int8 cache with an infinite value scale: results of
the rows that attend to that token are infinite by the signs of its codes, as with
SNEPPX_kv_attention, and those of others as they were."""
import math

import pytest
import torch

from test_gpu_kv_shared_nan import build

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("o", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("own", [[5, 9], [1] * 20], ids=["narrow", "wide"])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_infinite_value_scales(lib, where, own, o):
    c, tables, dlen, lengths, groups, pre, q = build(lib, 70, own, "int8")

    def run():
        out = torch.full(q.shape, 7.0, dtype=o, device=DEV)
        c.attention_shared(q, out, tables, dlen, max(lengths), groups, pre, 70, max(own))
        return out.float()
    before = run()
    row = int(tables[0, 66 if where == "prefix" else 70])
    c.v_scales[row] = math.inf
    c.v[row, 0, 0, 0::2] = 3
    c.v[row, 0, 0, 1::2] = -100
    after = run()
    hit = slice(0, len(own)) if where == "prefix" else slice(0, 1)
    assert (after[hit, :, 0::2] == math.inf).all() and (after[hit, :, 1::2] == -math.inf).all()
    others = torch.ones(len(lengths), dtype=torch.bool)
    others[hit] = False
    assert torch.isfinite(after[others]).all() and torch.equal(after[others], before[others])
