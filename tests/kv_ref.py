"""Plain 64-bit implementations of the paged key-value cache's operations
(include/sneppx_kv.h), on the CPU with numpy, one token at a time."""
import numpy as np


class Pool:
    """k, v float64 [pages][heads][page_size][dim] (int8: codes and scales
    kept apart), planes [pages][heads][page_size]."""

    def __init__(self, k, v, ks=None, vs=None, weights=None, positions=None):
        self.k, self.v, self.ks, self.vs, self.weights, self.positions = k, v, ks, vs, weights, positions
        self.pages, self.heads, self.page_size, self.dim = k.shape

    def place(self, table, slot):
        """(page, offset), or None where the page is not there."""
        page = int(table[slot // self.page_size])
        return (page, slot % self.page_size) if 0 <= page < self.pages else None


def _length(n, table, page_size, most=None):
    n = min(max(int(n), 0), len(table) * page_size)
    return n if most is None else min(n, most)


def attention(p, q, tables, lengths, scale, most=None):
    """(out [rows][q_heads][dim], sums added to the weights, and bounds of what
    fp32 rounding moves them by).  The bounds take every rounding error as
    independent: 4 sqrt(n) 2^-24 of the sum of magnitudes for a sum of n terms,
    and twice the error of a logit as that of its weight."""
    rows, hq, dim = q.shape
    group = hq // p.heads
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    added, added_tol = np.zeros((p.pages, p.heads, p.page_size)), np.zeros((p.pages, p.heads, p.page_size))
    eps = 2.0 ** -24
    for b in range(rows):
        at = [p.place(tables[b], t) for t in range(_length(lengths[b], tables[b], p.page_size, most))]
        at = [a for a in at if a is not None]
        if not at:
            continue
        pg, off = (np.array(x) for x in zip(*at))
        for h in range(p.heads):
            k, v = p.k[pg, h, off], p.v[pg, h, off]
            if p.ks is not None:
                k, v = k * p.ks[pg, h, off, None], v * p.vs[pg, h, off, None]
            for j in range(h * group, (h + 1) * group):
                s = k @ q[b, j] * scale
                err = (4 * np.sqrt(dim) + 4) * eps * (np.abs(k) @ np.abs(q[b, j])) * abs(scale)
                w = np.exp(s - s.max())
                w /= w.sum()
                rel = 2 * err.max() + (4 * np.sqrt(len(at)) + 8) * eps
                out[b, j] = w @ v
                tol[b, j] = rel * (w @ np.abs(v)) + 1e-30
                added[pg, h, off] += w
                added_tol[pg, h, off] += rel * w + 1e-30
    return out, tol, added, added_tol


def append_slots(starts, lengths, next_pos, tokens):
    """(token, row, slot, position) of every token that belongs to a row."""
    rows = len(lengths)
    if starts is None:
        starts = list(range(rows + 1))
    for b in range(rows):
        n = int(starts[b + 1]) - int(starts[b])
        for i in range(n):
            if starts[b] + i < tokens:
                yield int(starts[b]) + i, b, int(lengths[b]) - n + i, int(next_pos[b]) - n + i


def evict(p, planes, tables, lengths, next_pos, budget, recent, most=None):
    """In place over the arrays `planes` (each indexed [page, head, offset]);
    returns the new lengths."""
    new = []
    for b in range(len(lengths)):
        n = _length(lengths[b], tables[b], p.page_size, most)
        at = [p.place(tables[b], t) for t in range(n)]
        if n <= budget or any(a is None for a in at):
            new.append(n)
            continue
        new.append(budget)
        for h in range(p.heads):
            def rank(t):
                w = float(p.weights[at[t][0], h, at[t][1]])
                if int(p.positions[at[t][0], h, at[t][1]]) >= int(next_pos[b]) - recent:
                    return (0, 0.0, t)
                return (2, 0.0, t) if np.isnan(w) else (1, -w, t)
            kept = sorted(sorted(range(n), key=rank)[:budget])
            stay = set(kept)
            holes = [t for t in range(budget) if t not in stay]
            come = [t for t in kept if t >= budget]
            assert len(holes) == len(come)
            for to, of in zip(holes, come):
                for a in planes:
                    a[at[to][0], h, at[to][1]] = a[at[of][0], h, at[of][1]]
    return np.array(new, np.int32)
