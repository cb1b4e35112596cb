"""SNEPPX_kv_attention_shared where tokens of a prefix have NaN logits: they make the rows
that attend to them NaN wherever in the prefix they are, alone in a span, beside nothing or
beside logits of -inf, as with SNEPPX_kv_attention."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def build(lib, prefix, own, dtype, seed=1, dim=64):
    """Rows behind a prefix, in pages of one token, then one row of no group; positive
    queries of four heads."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    lengths = [prefix + n for n in own] + [21]
    width = max(lengths)
    rows = len(lengths)
    c = lib.kv_cache(prefix + rows * width, 1, 1, dim, dtype)
    tables = prefix + torch.arange(rows * width, dtype=torch.int32, device=DEV).view(rows, width)
    tables[:-1, :prefix] = torch.arange(prefix, dtype=torch.int32, device=DEV)
    for x, s in ((c.k, c.k_scales), (c.v, c.v_scales)):
        r = torch.randn(x.shape, device=DEV, generator=g)
        x.copy_(r if s is None else (40 * r).clamp(-127, 127))
        if s is not None:
            s.fill_(0.02)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    q = torch.rand((rows, 4, dim), device=DEV, generator=g).add(0.1).to(torch.bfloat16)
    return c, tables, i32(lengths), lengths, i32([0, len(own)]), i32([prefix]), q


def put(c, tokens, value):
    """Keys whose logits are NaN or -inf."""
    for t in tokens:
        if c.k_scales is None:
            c.k[t] = value
        else:
            c.k[t] = -1
            c.k_scales[t] = abs(value)


def both(c, tables, dlen, lengths, groups, prefix, q, o, max_own):
    out, plain = (torch.full(q.shape, 7.0, dtype=o, device=DEV) for _ in range(2))
    c.attention_shared(q, out, tables, dlen, max(lengths), groups, prefix, int(prefix[0]), max_own)
    c.attention(q, plain, tables, dlen, max(lengths))
    torch.cuda.synchronize()
    assert torch.equal(torch.isnan(out), torch.isnan(plain))
    return out


CASES = [
    # prefix, tokens of it with NaN, with -inf
    (32, range(32), []),                 # all of a prefix
    (1, [0], []),
    (65, [64], []),                      # the only token of a span's last step
    (80, range(64, 80), []),
    (64, range(32), range(32, 64)),      # beside a half without a finite logit
    (64, range(32, 64), range(32)),
    (96, range(96), []),                 # in either half of the last step
    (100, [70], [t for t in range(64, 100) if t != 70]),
    (100, [99], [t for t in range(64, 100) if t != 99]),
    (64, [3], [t for t in range(64) if t != 3]),
    (640, [639], range(576, 639)),
]


@pytest.mark.parametrize("o", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("own", [[5, 9], [3, 40], [0, 1, 2] * 5, [7] * 17], ids=lambda n: f"{len(n)}rows")
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"p{c[0]}-nan{len(c[1])}-inf{len(c[2])}")
def test_nan_in_a_prefix(lib, case, own, dtype, o):
    prefix, nans, infs = case
    c, tables, dlen, lengths, groups, pre, q = build(lib, prefix, own, dtype)
    put(c, infs, -math.inf)
    put(c, nans, math.nan)
    out = both(c, tables, dlen, lengths, groups, pre, q, o, max(own))
    assert torch.isnan(out[:-1]).all() and torch.isfinite(out[-1]).all()


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("prefix", [1, 32, 33, 64, 65])
def test_a_nan_query_of_a_row_that_is_its_prefix(lib, prefix, dtype):
    c, tables, dlen, lengths, groups, pre, q = build(lib, prefix, [0, 3, 0], dtype)
    q[0] = math.nan
    q[2, 1] = math.nan
    out = both(c, tables, dlen, lengths, groups, pre, q, torch.float32, 3)
    assert torch.isnan(out[0]).all() and torch.isnan(out[2, 1]).all()
    assert torch.isfinite(out[1]).all() and torch.isfinite(out[2, 2:]).all() and torch.isfinite(out[2, 0]).all()
