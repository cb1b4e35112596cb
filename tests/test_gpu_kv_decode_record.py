"""examples/kv_decode.py against a plain record of the same tokens: every token's key
and value as the QKV projection gave them, and which of them each head still holds.
After every step the attention's output, the sums of weights and what the cache
holds are compared with it, also where the step evicts."""
import os
import sys

import numpy as np
import pytest
import torch

import kv_ref

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
from kv_decode import AttentionBlock  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"
HEADS, QH, DIM, HIDDEN = 2, 8, 64, 256


class Record:
    """Of each row and head: the positions in its slots, and the sums of their weights
    with a bound of their error; of each token the stored rows."""

    def __init__(self, block, oracle):
        self.block, self.oracle, self.i8 = block, oracle, block.cache.k_scales is not None
        self.tables = block.tables.cpu().numpy()
        self.rows, self.page = self.tables.shape[0], block.cache.page_size
        self.slots = [[[] for _ in range(HEADS)] for _ in range(self.rows)]
        self.sums = [[[] for _ in range(HEADS)] for _ in range(self.rows)]
        self.tol = [[[] for _ in range(HEADS)] for _ in range(self.rows)]
        self.stored = [[] for _ in range(self.rows)]       # by position: ((codes, scales) of k, of v)

    def store(self, x):
        x = x.cpu().float().numpy()
        if not self.i8:
            return x, np.ones(HEADS, np.float32)
        _, codes, scales = self.oracle.quantize_int8_channel(x)
        return codes.astype(np.float32), scales

    def append(self, b, k, v):
        for h in range(HEADS):
            self.slots[b][h].append(len(self.stored[b]))
            self.sums[b][h].append(0.0)
            self.tol[b][h].append(0.0)
        self.stored[b].append((self.store(k), self.store(v)))

    def length(self, b):
        return len(self.slots[b][0])

    def at(self, b):
        t = np.arange(self.length(b))
        return self.tables[b][t // self.page], t % self.page

    def attend(self, q, out, weights):
        """Compares one step's output and the sums after it (before any eviction)."""
        for b in range(self.rows):
            n = self.length(b)
            page, off = self.at(b)
            # this row as a pool of one page, in the order of its slots
            of = [[[self.stored[b][p][x] for p in self.slots[b][h]] for h in range(HEADS)] for x in (0, 1)]
            codes = [np.array([[s[0][h] for s in of[x][h]] for h in range(HEADS)], np.float64)[None] for x in (0, 1)]
            scales = [np.array([[s[1][h] for s in of[x][h]] for h in range(HEADS)], np.float64)[None] for x in (0, 1)]
            pool = kv_ref.Pool(codes[0], codes[1], *scales)
            want, tol, added, added_tol = kv_ref.attention(pool, q[b:b + 1], np.zeros((1, 1), np.int32), [n], DIM ** -0.5)
            assert (np.abs(out[b] - want[0]) <= tol[0] + 2.0 ** -8 * np.abs(want[0])).all(), b
            for h in range(HEADS):
                sums = np.array(self.sums[b][h]) + added[0, h]
                bound = np.array(self.tol[b][h]) + added_tol[0, h] + 2.0 ** -23 * sums
                assert (np.abs(weights[page, h, off] - sums) <= bound).all(), (b, h)
                self.sums[b][h], self.tol[b][h] = list(sums), list(bound)

    def evict(self, weights, budget, recent):
        """Cuts as the definition has it, ranked by the cache's own sums (which attend()
        has compared: two that lie within their bounds may rank either way)."""
        for b in range(self.rows):
            n, last = self.length(b), len(self.stored[b])
            if n <= budget:
                continue
            page, off = self.at(b)
            for h in range(HEADS):
                s, w = self.slots[b][h], weights[page, h, off]
                kept = sorted(range(n), key=lambda t: (0, 0.0, t) if s[t] >= last - recent else (1, -w[t], t))[:budget]
                holes = [t for t in range(budget) if t not in set(kept)]
                come = sorted(t for t in kept if t >= budget)
                for plane in (s, self.sums[b][h], self.tol[b][h]):
                    for to, frm in zip(holes, come, strict=True):
                        plane[to] = plane[frm]
                    del plane[budget:]

    def holds(self):
        """The cache holds these tokens, bit for bit, in these slots."""
        c = self.block.cache
        k, v, pos = c.k.cpu().float().numpy(), c.v.cpu().float().numpy(), c.positions.cpu().numpy()
        scales = [None if s is None else s.cpu().numpy() for s in (c.k_scales, c.v_scales)]
        assert self.block.lengths.tolist() == [self.length(b) for b in range(self.rows)]
        assert self.block.next_pos.tolist() == [len(s) for s in self.stored]
        for b in range(self.rows):
            page, off = self.at(b)
            for h in range(HEADS):
                assert pos[page, h, off].tolist() == self.slots[b][h]
                for x, pool in ((0, k), (1, v)):
                    of = [self.stored[b][p][x] for p in self.slots[b][h]]
                    assert np.array_equal(pool[page, h, off], np.array([s[0][h] for s in of], np.float32))
                    if self.i8:
                        assert np.array_equal(scales[x][page, h, off], np.array([s[1][h] for s in of], np.float32))


def decoding(lib, oracle, dtype, capacity, budget, recent, rows, seed):
    """The block, its record, and functions that run prompts and steps on both."""
    block = AttentionBlock(lib, rows, capacity, budget, recent, hidden=HIDDEN, q_heads=QH, kv_heads=HEADS, dim=DIM,
                           dtype=dtype, seed=seed)
    rec = Record(block, oracle)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    before = {}
    evict = block.cache.evict

    def noted(*args):
        torch.cuda.synchronize()
        before["weights"] = block.cache.weights.cpu().double().numpy()
        evict(*args)

    block.cache.evict = noted

    def prompt(counts):
        x = torch.randn((sum(counts), HIDDEN), device=DEV, generator=g).to(torch.bfloat16)
        block.prompt(x, counts)
        torch.cuda.synchronize()
        _, k, v = block.project(x)
        at = 0
        for b, n in enumerate(counts):
            for _ in range(n):
                rec.append(b, k[at], v[at])
                at += 1
        rec.holds()

    def step():
        """True where a row was cut."""
        x = torch.randn((rows, HIDDEN), device=DEV, generator=g).to(torch.bfloat16)
        before.clear()
        y = block.step(x).clone()
        torch.cuda.synchronize()
        q, k, v = block.project(x)
        for b in range(rows):
            rec.append(b, k[b], v[b])
        weights = before.get("weights", None)
        if weights is None:
            weights = block.cache.weights.cpu().double().numpy()
        rec.attend(q.cpu().double().numpy(), block.out.cpu().double().numpy(), weights)
        cut = any(rec.length(b) > budget for b in range(rows))
        assert cut == ("weights" in before)
        rec.evict(weights, budget, recent)
        rec.holds()
        # y is the O projection of that output
        qw, sc, qz = block.o_w
        again = torch.empty_like(y)
        lib.qlinear_w4a16(block.out.flatten(1), qw, sc, qz, None, sc.shape[1], again, 128)
        torch.cuda.synchronize()
        assert torch.equal(again.view(torch.int16), y.view(torch.int16)) and bool(torch.isfinite(y.float()).all())
        return cut

    return block, rec, prompt, step


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_every_step_against_the_record(lib, oracle, dtype):
    print(f"[gpu] kv decode record {dtype}", flush=True)
    block, rec, prompt, step = decoding(lib, oracle, dtype, 64, 50, 12, 4, seed=11)
    prompt([30, 47, 9, 44])
    cuts = [step() for _ in range(12)]
    assert cuts == [False] * 3 + [True] * 9


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_a_second_prompt(lib, oracle, dtype):
    """Prompts go behind what the rows hold, and steps reach all of it."""
    print(f"[gpu] kv decode second prompt {dtype}", flush=True)
    block, rec, prompt, step = decoding(lib, oracle, dtype, 80, 70, 8, 3, seed=21)
    prompt([40, 5, 1])
    assert not step()
    prompt([3, 50, 2])
    for _ in range(3):
        assert not step()
    prompt([1, 1, 30])
    assert [step() for _ in range(14)] == [False] * 10 + [True] * 4


def test_more_than_the_capacity(lib, oracle):
    """Refused before anything changes."""
    print("[gpu] kv decode capacity", flush=True)
    block, rec, prompt, step = decoding(lib, oracle, "bf16", 32, 32, 4, 2, seed=31)
    prompt([20, 31])
    x = torch.zeros((14, HIDDEN), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="capacity"):
        block.prompt(x, [13, 1])
    rec.holds()
    step()
    with pytest.raises(ValueError, match="capacity"):
        block.step(x[:2])
    rec.holds()
