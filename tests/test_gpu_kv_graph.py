"""Append, attention and eviction recorded into one graph, by the library's capture
and by torch's.  Replays follow the lengths on the device: each equals the eager
calls at the same lengths bit for bit, in outputs, sums and all that the cache holds."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bits(t):
    return t.contiguous().view(torch.uint8)


# each set is of 4 rows; with 64 heads there are 8 shares of up to 12 steps of 128 tokens
LENGTHS = [[3000, 2500, 1200, 2900],     # shares across rows
           [1, 1, 1, 1],
           [0, 1, 3000, 700],
           [3000, 0, 0, 0],              # one row in all shares
           [2500, 2500, 0, 129],
           [128, 128, 127, 1],
           [3000, 3000, 3000, 3000],
           [701, 700, 699, 2]]           # one too many


@pytest.mark.parametrize("how", ["lib", "torch", "torch, cold"])
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_a_recorded_step(lib, dtype, how):
    print(f"[gpu] kv graph of a step {dtype} {how}", flush=True)
    rows, heads, dim, page, width, budget, recent = 4, 64, 16, 16, 188, 700, 50
    most = width * page
    c = lib.kv_cache(rows * width, page, heads, dim, dtype, weights=True, positions=True)
    g = torch.Generator(device=DEV).manual_seed(7)
    tables = torch.randperm(rows * width, device=DEV, generator=g).to(torch.int32).view(rows, width)
    if dtype == "int8":
        for t in (c.k, c.v):
            t.copy_(torch.randint(-127, 128, t.shape, device=DEV, generator=g))
        for t in (c.k_scales, c.v_scales):
            t.copy_(torch.rand(t.shape, device=DEV, generator=g) * 0.02 + 0.005)
    else:
        for t in (c.k, c.v):
            t.copy_(torch.randn(t.shape, device=DEV, generator=g))
    c.weights.copy_(torch.rand(c.weights.shape, device=DEV, generator=g))
    c.positions.copy_(torch.randint(0, 3000, c.positions.shape, device=DEV, generator=g))
    planes = [t for t in (c.k, c.v, c.k_scales, c.v_scales, c.weights, c.positions) if t is not None]
    before = [t.clone() for t in planes]
    lengths, next_pos, new = (torch.zeros(rows, dtype=torch.int32, device=DEV) for _ in range(3))
    qkv = torch.randn((rows, 3 * heads * dim), device=DEV, generator=g).to(torch.bfloat16)
    q, k, v = qkv.unflatten(1, (3 * heads, dim)).split(heads, 1)
    summed, plain = (torch.zeros((rows, heads, dim), device=DEV) for _ in range(2))
    results = planes + [new, summed, plain]

    def step(stream):
        c.append(k, v, tables, lengths, next_pos, stream=stream)
        c.attention(q, plain, tables, lengths, most, stream=stream)
        c.attention(q, summed, tables, lengths, most, accumulate=True, stream=stream)
        c.evict(tables, lengths, next_pos, new, most, budget, recent, stream=stream)

    st = torch.cuda.Stream()

    def run(at, call):
        for t, x in zip(planes, before):
            t.copy_(x)
        lengths.copy_(torch.tensor(at, dtype=torch.int32))
        next_pos.copy_(lengths + 9)
        for t in (new, summed, plain):
            t.fill_(-3)
        torch.cuda.synchronize()
        call()
        st.synchronize()
        return [t.clone() for t in results]

    if how != "torch, cold":         # (workspaces that the recorded calls find)
        run(LENGTHS[0], lambda: step(st.cuda_stream))
    lengths.copy_(torch.tensor(LENGTHS[1], dtype=torch.int32))
    torch.cuda.synchronize()
    if how == "lib":
        rec = lib.capture(lambda: step(st.cuda_stream), stream=st.cuda_stream)
        replay = lambda: lib.graph_launch(rec, stream=st.cuda_stream)      # noqa: E731
    else:
        rec = torch.cuda.CUDAGraph()
        with torch.cuda.graph(rec, stream=st):
            step(None)

        def replay():
            with torch.cuda.stream(st):
                rec.replay()

    names = [n for n in ("k", "v", "k_scales", "v_scales", "weights", "positions") if getattr(c, n) is not None]
    for at in LENGTHS + LENGTHS[::-1]:
        want = run(at, lambda: step(st.cuda_stream))
        got = run(at, replay)
        for name, x, y in zip(names + ["new_lengths", "summed", "plain"], want, got):
            assert torch.equal(bits(x), bits(y)), (at, name)
        assert got[-3].tolist() == [min(n, budget) for n in at]
        assert bool((got[-1][[n == 0 for n in at]] == 0).all())
    if how == "lib":
        lib.graph_destroy(rec)
    else:
        rec.reset()
    lib.fn["SNEPPX_qlinear_release_workspaces"](st.cuda_stream)
