"""SNEPPX_kv_attention over the range of the cache's values: results stay those of
the definition where values come near the largest that bf16 holds."""
import pytest
import torch

from test_gpu_kv_attention import build

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("n,heads", [(40, 4), (900, 2), (5000, 1)])
def test_weights_of_zero_add_nothing(lib, n, heads, dtype):
    """One token of zeros has all the weight: the result is zero, whatever the values
    whose weights are 2^-512 and less, and so zero in fp32."""
    print(f"[gpu] kv_attention zero weights n={n} {dtype}", flush=True)
    c, ref, tables, dtab, dlen = build(lib, [n], heads, 64, 16, dtype, 40 + n, garbage=False)
    c.k.zero_()
    at = n // 3
    page, off = int(tables[0, at // 16]), at % 16
    c.k[page, :, off] = 64
    if dtype == "int8":
        c.k_scales.fill_(1.0)
        c.v.fill_(100)
    else:
        c.v.fill_(1e30)
    c.v[page, :, off] = 0
    q = torch.ones((1, 2 * heads, 64), dtype=torch.bfloat16, device=DEV)
    out = torch.full((1, 2 * heads, 64), 3.0, device=DEV)
    c.attention(q, out, dtab, dlen, n, 0.125)       # 64 * 64 / 8 = 512 over 0
    torch.cuda.synchronize()
    assert bool((out == 0).all()), float(out.abs().max())
