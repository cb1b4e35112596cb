"""Attention over int8 caches whose scales have either sign (a caller's own tensors):
SNEPPX_kv_attention, _shared and _picked against float64, tolerances as in
test_gpu_kv_attention.py and test_gpu_kv_shared.py."""
import numpy as np
import pytest
import torch

import kv_ref
from test_gpu_kv_attention import build

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dim", [64, 128, 240])
@pytest.mark.parametrize("which", ["v", "k", "both"])
def test_scales_of_either_sign(lib, which, dim):
    lengths = [70, 300, 1, 33]
    c, ref, tables, dtab, dlen = build(lib, lengths, 2, dim, 16, "int8", dim, garbage=False)
    g = torch.Generator(device=DEV).manual_seed(dim)
    for s, name in ((c.k_scales, "k"), (c.v_scales, "v")):
        if which in (name, "both"):
            s.mul_(torch.randint(0, 2, s.shape, device=DEV, generator=g) * 2 - 1)
    ref.ks, ref.vs = (s.cpu().double().numpy() for s in (c.k_scales, c.v_scales))
    q = torch.randn((4, 8, dim), device=DEV, generator=g).to(torch.bfloat16)
    want, tol, _, _ = kv_ref.attention(ref, q.cpu().double().numpy(), tables, lengths, dim ** -0.5)
    size, _, _, _ = kv_ref.attention(kv_ref.Pool(ref.k, np.abs(ref.v), ref.ks, np.abs(ref.vs)), q.cpu().double().numpy(), tables,
                                     lengths, dim ** -0.5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for call, more in ((lambda o: c.attention(q, o, dtab, dlen, 320), 0),
                       (lambda o: c.attention_shared(q, o, dtab, dlen, 320, i32([0, 1, 2, 4]), i32([64, 200, 0]), 200, 120), 1),
                       (lambda o: c.attention_picked(q, o, dtab[:, None].repeat(1, 2, 1), dlen), 0)):
        out = torch.zeros(q.shape, device=DEV)
        call(out)
        torch.cuda.synchronize()
        off = np.abs(out.cpu().double().numpy() - want) - tol - more * 64 * 2.0 ** -24 * size
        assert (off <= 0).all(), float((off / size).max())
