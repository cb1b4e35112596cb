"""Plain 64-bit implementations of what stands around the paged key-value cache
(include/sneppx_rotary.h and the later parts of include/sneppx_kv.h), on the CPU with
numpy, one row at a time."""
import numpy as np

EPS32 = 2.0 ** -24          # half a step of fp32, relative


def turn(x, positions, freqs, interleaved=False, magnitude=1.0, norm=None, eps=1e-6):
    """(heads [tokens][heads][dim] turned, bounds of what fp32 moves them by).

    The bounds, in units of 2^-24 of the magnitudes: a normalised element is off by the
    rounding of its factors and of the mean (a sum over up to 8 + 5 levels, a division, a
    root, a reciprocal and two products: 18); a turned one by cos and sin (2 units each, the
    angle's own rounding 2 pi / 4 and the magnitude's 1), the products 1 and the sum 1: 6."""
    x = np.asarray(x, np.float64)
    tol = np.zeros_like(x)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(norm, np.float64)
        tol = 18 * EPS32 * np.abs(x)
    d = 2 * len(freqs)
    y = x.copy()
    if d:
        angle = np.asarray(positions, np.float64)[:, None] * np.asarray(freqs, np.float64)[None]
        c, s = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * magnitude
        i = np.arange(d // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + d // 2)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size = abs(magnitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
        t = 6 * EPS32 * size + abs(magnitude) * (tol[..., a] + tol[..., b])
        tol[..., a] = tol[..., b] = t
    return y, tol


def _clip(n, most):
    return min(max(int(n), 0), most)


def reserve(refs, page_size, tables, lengths, next_pos, counts, tokens):
    """In place over refs, tables, lengths and next_pos (or None); returns (starts,
    granted, slots, positions)."""
    rows, width = tables.shape
    pages, most = len(refs), width * page_size
    starts, granted = np.zeros(rows + 1, np.int64), np.zeros(rows, np.int64)
    slots, positions = -np.ones(tokens, np.int64), -np.ones(tokens, np.int64)
    free = [p for p in range(pages) if refs[p] == 0]
    asked = 0
    for b in range(rows):
        want = 1 if counts is None else max(0, int(counts[b]))
        starts[b + 1] = min(starts[b] + want, 2 ** 31 - 1)
        n = _clip(lengths[b], most)
        if n + want > most:
            continue
        entries = [e for e in range(-(-n // page_size), -(-(n + want) // page_size)) if not 0 <= tables[b, e] < pages]
        mine = range(asked, asked + len(entries))
        asked += len(entries)
        if entries and asked > len(free):
            continue
        for e, i in zip(entries, mine):
            tables[b, e] = free[i]
            refs[free[i]] = 1
        first = n if next_pos is None else int(next_pos[b])
        for i in range(want):
            t = starts[b] + i
            if t >= tokens:
                break
            page = int(tables[b, (n + i) // page_size])
            if 0 <= page < pages:
                slots[t] = page * page_size + (n + i) % page_size
            positions[t] = first + i
        if want:
            granted[b] = want
            lengths[b] = n + want
            if next_pos is not None:
                next_pos[b] += want
    return starts, granted, slots, positions


def release(refs, page_size, tables, lengths):
    rows, width = tables.shape
    for b in range(rows):
        for e in range(-(-_clip(lengths[b], width * page_size) // page_size), width):
            if 0 <= tables[b, e] < len(refs):
                if refs[tables[b, e]] > 0:
                    refs[tables[b, e]] -= 1
                tables[b, e] = -1


def share(refs, page_size, tables, lengths, next_pos, sources, counts):
    rows, width = tables.shape

    def takes(b):
        return 0 <= sources[b] < rows and sources[b] != b
    for b in range(rows):
        if not takes(b) or takes(sources[b]):
            continue
        a = sources[b]
        k = min(max(0, int(counts[b])), _clip(lengths[a], width * page_size)) // page_size
        for e in range(k):
            was, page = tables[b, e], tables[a, e]
            tables[b, e] = page
            if 0 <= page < len(refs):
                refs[page] += 1
            if 0 <= was < len(refs) and refs[was] > 0:
                refs[was] -= 1
        lengths[b] = k * page_size
        if next_pos is not None:
            next_pos[b] = k * page_size


def key_bounds(keys, bounds, tables, lengths, counts, page_size):
    """keys [pages][heads][page_size][dim] as the cache gives them back; bounds
    [pages][heads][2][dim], in place."""
    rows, width = tables.shape
    for b in range(rows):
        n = _clip(lengths[b], width * page_size)
        c = _clip(1 if counts is None else counts[b], n)
        if c == 0:
            continue
        for e in range((n - c) // page_size, (n - 1) // page_size + 1):
            page = tables[b, e]
            if 0 <= page < len(keys):
                k = keys[page][:, : min(page_size, n - e * page_size)]
                bounds[page, :, 0], bounds[page, :, 1] = k.min(1), k.max(1)


def pick(q, bounds, tables, lengths, page_size, budget, first, recent, most=None):
    """(picked [rows][heads][budget], picked_lengths)."""
    rows, width = tables.shape
    pages, heads = bounds.shape[:2]
    group = q.shape[1] // heads
    picked, new = -np.ones((rows, heads, budget), np.int64), np.zeros(rows, np.int64)
    for b in range(rows):
        n = _clip(lengths[b], width * page_size if most is None else min(most, width * page_size))
        have = -(-n // page_size)
        new[b] = n - max(0, have - budget) * page_size
        for h in range(heads):
            kept = list(range(have))
            if have > budget:
                def rank(e):
                    page = tables[b, e]
                    if e < first or e >= have - recent:
                        return (0, 0.0, e)
                    if not 0 <= page < pages:
                        return (2, 0.0, e)
                    lo, hi = bounds[page, h]
                    s = max_nan(np.maximum(q[b, h * group + j] * lo, q[b, h * group + j] * hi).sum() for j in range(group))
                    s = np.float32(s)
                    return (2, 0.0, e) if np.isnan(s) else (1, -s, e)
                kept = sorted(sorted(range(have), key=rank)[:budget])
            picked[b, h, : len(kept)] = [tables[b, e] for e in kept]
    return picked, new


def max_nan(xs):
    xs = list(xs)
    return np.nan if any(np.isnan(x) for x in xs) else max(xs)
