"""examples/kv_serve.py, the operators together as a server runs them: rows share a
prompt, decode and end.  Every step is checked against float64: which pages and slots
its tokens got, what the cache holds of them, and the attention over all of a row's
tokens (or the picked pages); and a whole step in a graph, replayed between eager work."""
import os
import sys

import numpy as np
import pytest
import torch

import kv_ref
import serve_ref

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
from kv_serve import ServeBlock  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 16


def pool_of(c):
    f = lambda t: None if t is None else t.cpu().double().numpy()     # noqa: E731
    return kv_ref.Pool(f(c.k), f(c.v), f(c.k_scales), f(c.v_scales))


def make(lib, dtype, pick, rows=5, pages=60):
    return ServeBlock(lib, rows, pages, 12, hidden=256, q_heads=8, kv_heads=2, dim=64, page=PAGE, dtype=dtype, pick=pick, seed=3)


def tokens(g, n):
    return torch.randn((n, 256), device=DEV, generator=g).to(torch.bfloat16)


def check_pages(block, state):
    """Tables, counts and lengths against the plain loops' state."""
    for got, want in zip((block.free.refs, block.tables, block.lengths, block.next_pos), state):
        assert np.array_equal(got.cpu().numpy(), want)
    held = np.bincount(state[1][state[1] >= 0], minlength=len(state[0]))
    assert np.array_equal(held, state[0])


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
@pytest.mark.parametrize("pick", [0, 4])
def test_streams_come_and_go(lib, dtype, pick):
    print(f"[gpu] kv serve example {dtype} pick={pick}", flush=True)
    block = make(lib, dtype, pick)
    g = torch.Generator(device=DEV).manual_seed(5)
    state = [np.zeros(60, np.int64), -np.ones((5, 12), np.int64), np.zeros(5, np.int64), np.zeros(5, np.int64)]

    def extend(x, counts):
        q = block.extend(x, counts)
        _, granted, slots, pos = serve_ref.reserve(state[0], PAGE, state[1], state[2], state[3], counts, x.shape[0])
        assert granted.tolist() == counts
        raw_q, raw_k, raw_v = (t.cpu().double().numpy() for t in block.project(x))
        f = block.rotary
        for raw, got, norm in ((raw_q, q, f.q_norm), (raw_k, None, f.k_norm)):
            want, tol = serve_ref.turn(raw, pos, f.freqs.cpu().numpy(), False, 1.0, norm.cpu().double().numpy(), 1e-6)
            if got is None:
                pool = pool_of(block.cache)
                got = pool.k[slots // PAGE, :, slots % PAGE]
                if dtype == "int8":
                    # (a step of the row's scale for each code, and what fp32 moves it by)
                    s = pool.ks[slots // PAGE, :, slots % PAGE][..., None]
                    assert (np.abs(got * s - want) <= 0.5 * s + tol + 127 * 2.0 ** -21 * s).all()
                    continue
            else:
                got = got.cpu().double().numpy()
            assert (np.abs(got - want) <= tol + 2.0 ** -8 * np.abs(want)).all()
        check_pages(block, state)
        return q

    def step():
        x = tokens(g, 5)
        held = block.held[:]
        y = block.step(x).clone()
        _, granted, slots, _ = serve_ref.reserve(state[0], PAGE, state[1], state[2], state[3], [0, 1, 1, 1, 1], 4)
        torch.cuda.synchronize()
        check_pages(block, state)
        assert block.held[1:] == [n + 1 for n in held[1:]] and state[2].tolist()[1:] == block.held[1:]
        # the queries of the step again: turned out of place
        raw = block.project(x[1:])[0]
        q = torch.empty((4, 8, 64), dtype=torch.bfloat16, device=DEV)
        pos = torch.tensor(state[3][1:] - 1, dtype=torch.int32, device=DEV)
        block.rotary.apply(raw, None, pos, q)
        qn = q.cpu().double().numpy()
        tables, lengths = state[1][1:], state[2][1:]
        pool = pool_of(block.cache)
        got = block.out[1:].cpu().double().numpy()
        if not pick:
            want, tol, _, _ = kv_ref.attention(pool, qn, tables, lengths, 0.125)
            size, _, _, _ = kv_ref.attention(kv_ref.Pool(pool.k, np.abs(pool.v), pool.ks, pool.vs), qn, tables, lengths, 0.125)
            tol = tol + 64 * 2.0 ** -24 * size + 2.0 ** -15 * size
            assert (np.abs(got - want) <= tol + 2.0 ** -8 * np.abs(want)).all()
        else:
            picked, n = serve_ref.pick(qn, block.bounds.cpu().double().numpy(), tables, lengths, PAGE, pick, 1, 2)
            assert np.array_equal(block.picked[1:].cpu().numpy(), picked) and block.picked_lengths[1:].tolist() == n.tolist()
            for h in range(2):
                one = kv_ref.Pool(*(None if t is None else t[:, h:h + 1] for t in (pool.k, pool.v, pool.ks, pool.vs)))
                want, tol, _, _ = kv_ref.attention(one, qn[:, 4 * h:4 * h + 4], picked[:, h], n, 0.125)
                assert (np.abs(got[:, 4 * h:4 * h + 4] - want) <= tol + 2.0 ** -8 * np.abs(want)).all()
        assert torch.isfinite(y[1:].float()).all()

    extend(tokens(g, 70), [70, 0, 0, 0, 0])
    block.share(range(1, 5))
    serve_ref.share(state[0], PAGE, state[1], state[2], state[3], [-1, 0, 0, 0, 0], [64] * 5)
    check_pages(block, state)
    assert block.common == 64 and state[0].max() == 5
    extend(tokens(g, 60), [0, 9, 30, 1, 20])
    for _ in range(10):
        step()
    # two streams end, and begin anew behind the prompt
    block.end([2, 4])
    state[2][[2, 4]] = state[3][[2, 4]] = 0
    serve_ref.release(state[0], PAGE, state[1], state[2])
    check_pages(block, state)
    block.share([2, 4])
    serve_ref.share(state[0], PAGE, state[1], state[2], state[3], [-1, -1, 0, -1, 0], [64] * 5)
    extend(tokens(g, 24), [0, 0, 4, 0, 20])
    for _ in range(8):
        step()
    block.end(range(5))
    assert int(block.free.refs.sum()) == 0 and (block.tables == -1).all()


@pytest.mark.parametrize("how", ["lib", "torch"])
@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_a_recorded_step(lib, dtype, how):
    """Pages, rotation, append, both attentions and the picks in one graph: replays from
    the same state equal the eager calls, bit for bit, step after step, with eager work and
    synchronizations in between."""
    print(f"[gpu] kv serve graph {dtype} {how}", flush=True)
    block = make(lib, dtype, 3)
    g = torch.Generator(device=DEV).manual_seed(6)
    block.extend(tokens(g, 70), [70, 0, 0, 0, 0])
    block.share(range(1, 5))
    block.extend(tokens(g, 60), [0, 9, 30, 1, 20])
    qkv = torch.randn((4, 12 * 64), device=DEV, generator=g).to(torch.bfloat16)
    q, k, v = qkv.unflatten(1, (12, 64)).split((8, 2, 2), 1)
    c, tables = block.cache, block.tables[1:]
    ints = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
    slots, positions, starts, granted, groups = ints(6), ints(6), ints(5), ints(4), torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    lengths, next_pos = block.lengths[1:].clone(), block.next_pos[1:].clone()
    turned = torch.zeros((4, 8, 64), dtype=torch.bfloat16, device=DEV)
    shared, over = (torch.zeros((4, 8, 64), device=DEV) for _ in range(2))
    planes = [t for t in (c.k, c.v, c.k_scales, c.v_scales) if t is not None]
    state = planes + [block.free.refs, tables, lengths, next_pos, block.bounds]
    results = state + [slots, positions, starts, granted, turned, shared, over, block.picked, block.picked_lengths]

    def step(st):
        block.free.reserve(tables, lengths, slots, next_pos=next_pos, positions=positions, starts=starts, granted=granted, stream=st)
        c.append_rotated(block.rotary, q, k, v, slots[:4], positions[:4], turned, stream=st)
        c.attention_shared(turned, shared, tables, lengths, 192, groups, block.prefix, 64, 128, stream=st)
        c.key_bounds(block.bounds, tables, lengths, stream=st)
        c.pick(turned, block.bounds, tables, lengths, 192, block.picked[1:], block.picked_lengths[1:], stream=st)
        c.attention_picked(turned, over, block.picked[1:], block.picked_lengths[1:], stream=st)

    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    before = [t.clone() for t in state]
    with torch.cuda.stream(st):
        for _ in range(2):
            step(st.cuda_stream)                     # (workspaces are taken)
    torch.cuda.synchronize()
    if how == "lib":
        graph = lib.capture(lambda: step(st.cuda_stream), stream=st.cuda_stream)
        replay = lambda: lib.graph_launch(graph, stream=st.cuda_stream)  # noqa: E731
    else:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            step(torch.cuda.current_stream().cuda_stream)

        def replay():
            with torch.cuda.stream(st):
                graph.replay()
    wants = []
    for t, b in zip(state, before):
        t.copy_(b)
    for _ in range(5):
        torch.cuda.synchronize()
        step(st.cuda_stream)
        torch.cuda.synchronize()
        wants.append([t.clone() for t in results])
    for t, b in zip(state, before):
        t.copy_(b)
    for i, want in enumerate(wants):
        for t in (shared, over, turned, slots):
            t.fill_(7)
        torch.cuda.synchronize()
        replay()
        if i % 2:
            torch.cuda.synchronize()
        st.synchronize()
        for t, w in zip(results, want):
            assert torch.equal(t.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8)), i
        _ = float(torch.randn(1000, device=DEV).sum())           # eager work of the program
    if how == "lib":
        lib.graph_destroy(graph)


def test_two_streams_at_once(lib):
    """The same calls on two streams without waiting in between: each stream's scratch is
    its own."""
    block = make(lib, "bf16", 3)
    g = torch.Generator(device=DEV).manual_seed(7)
    block.extend(tokens(g, 70), [70, 0, 0, 0, 0])
    block.share(range(1, 5))
    block.extend(tokens(g, 110), [0, 9, 80, 1, 20])
    c, tables, lengths = block.cache, block.tables[1:], block.lengths[1:]
    groups = torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    qs = [torch.randn((4, 8, 64), device=DEV, generator=g).to(torch.bfloat16) for _ in range(2)]
    outs = [[torch.zeros((4, 8, 64), device=DEV) for _ in range(2)] for _ in range(3)]
    picks = [(torch.zeros((4, 2, 3), dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)) for _ in range(3)]

    def run(i, slot, st):
        c.attention_shared(qs[i], outs[slot][0], tables, lengths, 192, groups, block.prefix, 64, 128, stream=st)
        c.pick(qs[i], block.bounds, tables, lengths, 192, *picks[slot], stream=st)
        c.attention_picked(qs[i], outs[slot][1], *picks[slot], stream=st)
    want = []
    for i in range(2):
        run(i, 2, None)
        torch.cuda.synchronize()
        want.append([t.clone() for t in (*outs[2], *picks[2])])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(50):
        for i in range(2):
            run(i, i, streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        for t, w in zip((*outs[i], *picks[i]), want[i]):
            assert torch.equal(t, w)


def test_the_example_runs(lib, capsys, monkeypatch):
    import kv_serve
    monkeypatch.setattr(sys, "argv", ["kv_serve.py", "--rows", "3", "--prompt", "100", "--own", "20", "--steps", "2", "--dtype", "int8",
                                      "--pick", "4"])
    kv_serve.main()
    assert "us a step" in capsys.readouterr().out
