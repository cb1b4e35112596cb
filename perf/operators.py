"""Performance cases of the key-value cache: what a program that decodes with
this library's linears does between the QKV projection and the O projection.

  append     the new tokens' keys and values, slices of the QKV rows, into the
             pages of their rows (bf16, or int8 with a scale per token and head)
  attention  one new token per row over its pages (bf16 or int8), optionally
             adding its softmax weights to the cache's sums
  evict      a row's cache cut to a budget: the newest positions and, of the
             others, the tokens with the largest sums stay

Layouts: k, v [pages][kv_heads][page_size][head_dim]; k_scales, v_scales,
weights (fp32) and positions (int32) [pages][kv_heads][page_size]; tables int32
[rows][width]; lengths int32 [rows].  Sizes are those of the Llama-3-8B-shaped
layer of bench.py (32 query heads, 8 key-value heads, head 128, QKV rows of
6144), of one rank of its TP=8 form (4 and 1 heads), and generic others.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
FLT_MIN = 1.1754943508222875e-38


def _lib():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sneppx-alg_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import sneppx_quant
    return sneppx_quant.load()


# ------------------------------------------------------------------- cases
def _attn(name, rows, length, q_heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", ragged=True, weights=False,
          out="bf16", absent=False):
    return {"name": name, "kind": "attention", "rows": rows, "length": length, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged, "weights": weights,
            "out": out, "absent": absent}


def _evict(name, rows, length, budget, recent, kv_heads=8, dim=128, page=16, dtype="bf16", ragged=False):
    return {"name": name, "kind": "evict", "rows": rows, "length": length, "budget": budget, "recent": recent,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged}


def _append(name, decode, chunks, chunk, past, q_heads=32, kv_heads=8, dim=128, page=16, dtype="bf16", stored=False):
    return {"name": name, "kind": "append", "decode": decode, "chunks": chunks, "chunk": chunk, "past": past,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "stored": stored}


def listed():
    return [
        # 16 streams decoding: one token each into its page, sums and positions
        # kept for eviction; the smallest call, where launches and latency count
        _append("append_step", 16, 0, 0, 640),
        # a packed batch of 16 decode rows and 8 prefill chunks of up to 512
        # tokens into an int8 cache, the stored rows returned for the chunks'
        # own attention
        _append("append_prompt_int8", 16, 8, 512, 200, page=64, dtype="int8", stored=True),
        # single-stream decoding after a short prompt
        _attn("attn_token", 1, 531, ragged=False),
        # 16 streams of 0 to 4096 tokens decoding together
        _attn("attn_batch16", 16, 4096),
        # one rank of a TP=8 group, 32 streams up to 8192 tokens, int8 cache
        _attn("attn_shard_int8", 32, 8192, q_heads=4, kv_heads=1, page=64, dtype="int8"),
        # one stream at the end of a context of 128K tokens
        _attn("attn_long", 1, 131072, page=64, ragged=False),
        # a loaded server: 64 streams up to 8192 tokens, int8 cache
        _attn("attn_batch64_int8", 64, 8192, page=32, dtype="int8"),
        # 16 streams over caches held at a budget of 2048, the weights summed
        _attn("attn_weights", 16, 2049, ragged=False, weights=True),
        # every head its own keys and values, head 80, odd pages of which some
        # are absent, fp32 rows for an fp32 layer
        _attn("attn_mha_odd", 5, 1003, q_heads=12, kv_heads=12, dim=80, page=24, out="f32", absent=True),
        # each decode step of those 16 streams: one token too many
        _evict("evict_step", 16, 2049, 2048, 256),
        # 8 prompts of 8192 tokens halved before decoding starts
        _evict("evict_prompt", 8, 8192, 4096, 512),
        # two long streams cut back to a sixth, int8 cache, ragged
        _evict("evict_long_int8", 2, 30001, 5000, 333, page=64, dtype="int8", ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "evict"])
    dtype = rng.choice(["bf16", "bf16", "int8"])
    dim = rng.choice([128, 128, 128, 64, 80, 96, 256])
    page = rng.choice([16, 16, 32, 64, 128, 24, 1])
    kv_heads = rng.choice([8, 8, 1, 2, 4, 12])
    q_heads = kv_heads * rng.choice([4, 4, 1, 2, 7, 8, 16, 20])
    per_token = 2 * kv_heads * dim * (1 if dtype == "int8" else 2)
    if kind == "append":
        past = _log(rng, 1, 2000)
        c = _append("", rng.choice([0, _log(rng, 1, 256)]), rng.choice([0, _log(rng, 1, 12)]), _log(rng, 8, 900), past,
                    q_heads, kv_heads, dim, page, dtype, rng.random() < 0.3)
        if c["decode"] + c["chunks"] == 0:
            c["decode"] = _log(rng, 1, 256)
    elif kind == "attention":
        while True:
            rows, length = _log(rng, 1, 128), _log(rng, 2, 131072)
            if rows * length * per_token <= 400e6 and rows * length * kv_heads <= 4 << 20:
                break
        c = _attn("", rows, length, q_heads, kv_heads, dim, page, dtype, rng.random() < 0.6, rng.random() < 0.25,
                  rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.15)
    else:
        while True:
            rows, length = _log(rng, 1, 64), _log(rng, 64, 60000)
            if rows * length * per_token <= 200e6 and rows * length * kv_heads <= 2 << 20:
                break
        budget = length - 1 if rng.random() < 0.4 else max(2, int(length * rng.uniform(0.1, 0.9)))
        c = _evict("", rows, length, budget, max(1, int(budget * rng.uniform(0.05, 0.5))), kv_heads, dim, page, dtype,
                   rng.random() < 0.3)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _lengths(c):
    """The rows' lengths: all the same, or from none to the largest."""
    n = c["rows"]
    if not c["ragged"] or n == 1:
        return [c["length"]] * n
    at = [int(round(c["length"] * (0.37 + 0.618034 * i) % c["length"])) for i in range(n)]
    at[0] = c["length"]
    if n >= 4:
        at[1], at[2] = 0, 1
    return at


def _counts(c):
    """New tokens of each row of an append: the decode rows, then the chunks."""
    return [1] * c["decode"] + [max(1, round(c["chunk"] * (i + 1) / c["chunks"])) for i in range(c["chunks"])]


def _codes(x):
    """int8 codes (as fp32 values) and scales of rows: s = max|x| / 127, the
    codes x * (1 / s) rounded half away from zero."""
    m = x.abs().amax(-1)
    s = torch.where(m < FLT_MIN, torch.ones_like(m), m / 127.0)
    v = x * (1.0 / s).unsqueeze(-1)
    a = v.abs()
    whole = a.floor()
    whole = whole + (a - whole >= 0.5).to(F32)
    return (torch.sign(v) * whole).clamp(-128, 127), s


def _rows(g, shape):
    return torch.randn(shape, device=DEV, generator=g)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    H, D, ps = c["kv_heads"], c["dim"], c["page"]
    if c["kind"] == "append":
        counts = _counts(c)
        lengths = [n + (c["past"] * (i % 5 + 1)) // 5 for i, n in enumerate(counts)]
    else:
        lengths = _lengths(c)
    B = len(lengths)
    width = max(1, -(-max(lengths) // ps))
    pages = B * width + 3
    perm = torch.randperm(pages, device=DEV, generator=g)[: B * width].to(torch.int32)
    s = {"case": c, "tables": perm.view(B, width).clone(),
         "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEV)}
    if c.get("absent"):
        # a row whose first pages were given back, and one without any
        s["tables"][0, : max(1, width // 5)] = -1
        s["tables"][B - 1] = -1
    shape = (pages, H, ps, D)
    k = _rows(g, shape)
    # a direction that queries share and that some tokens answer: a few weights
    # are large, as in a trained model's maps
    u = _rows(g, (1, H, 1, D)) / math.sqrt(D)
    k += 4.0 * u * (torch.rand((pages, H, ps, 1), device=DEV, generator=g) < 0.02)
    v = _rows(g, shape)
    if c["dtype"] == "int8":
        ck, sk = _codes(k)
        cv, sv = _codes(v)
        s.update(k=ck.to(torch.int8), v=cv.to(torch.int8), k_scales=sk, v_scales=sv)
        del ck, cv
    else:
        s.update(k=k.to(BF16), v=v.to(BF16), k_scales=None, v_scales=None)
    del k, v
    s.update(weights=None, positions=None)
    marks = (pages, H, ps)
    if c["kind"] != "attention" or c["weights"]:
        s["weights"] = torch.rand(marks, device=DEV, generator=g).pow(8) * 40.0
    s["next_pos"] = s["lengths"] + 17
    if c["kind"] == "append":
        T, G = sum(counts), c["q_heads"]
        s["positions"] = torch.zeros(marks, dtype=torch.int32, device=DEV)
        qkv = _rows(g, (T, (G + 2 * H) * D)).to(BF16)
        s["qkv"] = qkv
        s["new_k"] = qkv[:, G * D:(G + H) * D].unflatten(1, (H, D))
        s["new_v"] = qkv[:, (G + H) * D:].unflatten(1, (H, D))
        s["starts"] = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=DEV)
        s["k_stored"] = s["v_stored"] = None
        if c["stored"]:
            s["k_stored"], s["v_stored"] = (torch.zeros((T, H, D), dtype=BF16, device=DEV) for _ in range(2))
    elif c["kind"] == "attention":
        q = _rows(g, (B, c["q_heads"], D)) + 2.0 * math.sqrt(D) * u.view(H, 1, D).expand(
            H, c["q_heads"] // H, D).reshape(c["q_heads"], D)
        # queries as the QKV projection leaves them: the first part of its rows
        qkv = torch.zeros((B, (c["q_heads"] + 2 * H) * D), dtype=BF16, device=DEV)
        s["q"] = qkv[:, : c["q_heads"] * D].unflatten(1, (c["q_heads"], D))
        s["q"].copy_(q)
        s["out"] = torch.zeros((B, c["q_heads"], D), dtype=BF16 if c["out"] == "bf16" else F32, device=DEV)
        s["scale"] = 1.0 / math.sqrt(D)
    else:
        # positions: older ones in any order (an earlier cut moved rows), the
        # newest at the end
        t = torch.arange(width * ps, device=DEV, dtype=torch.int32)
        page, off = s["tables"][:, (t // ps).long()].long(), (t % ps).long()
        pos = torch.empty((B, H, width * ps), dtype=torch.int32, device=DEV)
        pos[:] = (s["next_pos"] - s["lengths"])[:, None, None] + t
        mix = torch.rand((B, H, width * ps), device=DEV, generator=g)
        old = t[None] < (s["lengths"] - c["recent"])[:, None]
        mix = torch.where(old[:, None], mix, 2.0 + t.to(F32))
        pos = pos.gather(2, mix.argsort(2))
        s["positions"] = torch.zeros(marks, dtype=torch.int32, device=DEV)
        s["positions"][page[:, None, :], torch.arange(H, device=DEV)[None, :, None], off] = pos
        # one buffer for both planes and a copy of it, to begin each pass with
        s["marks"] = torch.stack([s["weights"].view(torch.int32), s["positions"]])
        s["marks_before"] = s["marks"].clone()
        s["weights"], s["positions"] = s["marks"][0].view(F32), s["marks"][1]
        s["new_lengths"] = torch.zeros_like(s["lengths"])
    if own:   # the handle that a program keeps for its cache
        s["cache"] = _lib().kv_cache_from(s["k"], s["v"], s["k_scales"], s["v_scales"], s["weights"], s["positions"])
    return s


# --------------------------------------------------------------- the passes
def run(state):
    s, c = state, state["case"]
    if c["kind"] == "append":
        (_append_own if own else _append_plain)(s)
        return {"k": s["k"] if c["dtype"] == "bf16" else None, "v": s["v"] if c["dtype"] == "bf16" else None,
                "k_stored": s["k_stored"], "v_stored": s["v_stored"], "k_scales": s["k_scales"],
                "v_scales": s["v_scales"], "weights": s["weights"], "positions": s["positions"]}
    if c["kind"] == "attention":
        (_attention_own if own else _attention_plain)(s)
        return {"out": s["out"], "weights": s["weights"]}
    s["marks"].copy_(s["marks_before"])      # sums and positions as at the first pass: the same rows move each time
    (_evict_own if own else _evict_plain)(s)
    return {"k": s["k"], "v": s["v"], "k_scales": s["k_scales"], "v_scales": s["v_scales"], "weights": s["weights"],
            "positions": s["positions"], "new_lengths": s["new_lengths"]}


def _append_own(s):
    c = s["case"]
    s["cache"].append(s["new_k"], s["new_v"], s["tables"], s["lengths"], s["next_pos"],
                      starts=s["starts"] if c["chunks"] else None, k_stored=s["k_stored"], v_stored=s["v_stored"])


def _attention_own(s):
    c = s["case"]
    s["cache"].attention(s["q"], s["out"], s["tables"], s["lengths"], c["length"], s["scale"], accumulate=c["weights"])


def _evict_own(s):
    c = s["case"]
    s["cache"].evict(s["tables"], s["lengths"], s["next_pos"], s["new_lengths"], c["length"], c["budget"], c["recent"])


def _append_plain(s):
    starts, ps = s["starts"], s["k"].shape[2]
    T = s["new_k"].shape[0]
    t = torch.arange(T, device=DEV)
    row = torch.searchsorted(starts, t, right=True, out_int32=True).long() - 1
    back = starts[row + 1] - t                       # tokens from here to the row's end
    slot = (s["lengths"][row] - back).long()
    page, off = s["tables"][row, slot // ps].long(), slot % ps
    for new, pool, scales, stored in ((s["new_k"], s["k"], s["k_scales"], s["k_stored"]),
                                      (s["new_v"], s["v"], s["v_scales"], s["v_stored"])):
        x = new.to(F32)
        if scales is not None:
            code, sc = _codes(x)
            scales[page, :, off] = sc
            pool[page, :, off] = code.to(torch.int8)
            x = code * sc.unsqueeze(-1)
        else:
            pool[page, :, off] = x.to(BF16)
        if stored is not None:
            stored.copy_(x)
    s["weights"][page, :, off] = 0.0
    s["positions"][page, :, off] = (s["next_pos"][row] - back).to(torch.int32).unsqueeze(1)


def _gathered(pool, scales, page, off, valid):
    x = pool[page, :, off].to(F32)                   # [rows][length][kv_heads][dim]
    if scales is not None:
        x = x * scales[page, :, off].unsqueeze(-1)
    return torch.where(valid[:, :, None, None], x, torch.zeros_like(x)).transpose(1, 2).contiguous()


def _attention_plain(s):
    c, ps = s["case"], s["k"].shape[2]
    B, Hq, D = s["q"].shape
    H = s["k"].shape[1]
    t = torch.arange(c["length"], device=DEV)
    page = s["tables"][:, t // ps].long()
    valid = (t[None] < s["lengths"][:, None]) & (page >= 0) & (page < s["k"].shape[0])
    page, off = torch.where(valid, page, 0), (t % ps).expand(B, -1)
    K = _gathered(s["k"], s["k_scales"], page, off, valid)
    q = s["q"].to(F32).reshape(B, H, Hq // H, D)
    logits = torch.matmul(q, K.transpose(2, 3)) * s["scale"]
    del K
    there = valid[:, None, None, :]
    logits = torch.where(there, logits, torch.full_like(logits, -math.inf))
    top = logits.amax(-1, keepdim=True)
    p = torch.where(there, torch.exp(logits - top), torch.zeros_like(logits))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    V = _gathered(s["v"], s["v_scales"], page, off, valid)
    s["out"].copy_(torch.matmul(p, V).reshape(B, Hq, D))
    if c["weights"]:
        head = torch.arange(H, device=DEV)
        s["weights"].index_put_((page[:, None, :], head[None, :, None], off[:, None, :]), p.sum(2), accumulate=True)


def _evict_plain(s):
    c, ps = s["case"], s["k"].shape[2]
    H, L, budget = s["k"].shape[1], c["length"], c["budget"]
    B = s["lengths"].numel()
    n = min(budget, L - budget)
    lengths = s["lengths"].long()[:, None, None]
    t = torch.arange(L, device=DEV).expand(B, H, L)
    head = torch.arange(H, device=DEV)[None, :, None]

    def place(slot):
        return s["tables"].long()[:, None].expand(B, H, -1).gather(2, slot // ps), head, slot % ps

    at = place(t)
    w, pos = s["weights"][at], s["positions"][at]
    key = torch.where(torch.isnan(w), torch.full_like(w, -math.inf), w)
    key = torch.where(pos >= s["next_pos"][:, None, None] - c["recent"], torch.full_like(w, math.inf), key)
    key = torch.where(t < lengths, key, torch.full_like(w, -math.inf))
    order = torch.argsort(key, dim=2, descending=True, stable=True)
    kept = torch.zeros_like(t, dtype=torch.bool).scatter(2, order[..., :budget], True) & (t < lengths)
    hole = ~kept & (t < budget) & (lengths > budget)
    far = kept & (t >= budget)
    pad = (lengths - 1).clamp(min=0).expand(B, H, n + 1)
    dst = pad.scatter(2, torch.where(hole, hole.long().cumsum(2) - 1, n), t)[..., :n]
    src = pad.scatter(2, torch.where(far, far.long().cumsum(2) - 1, n), t)[..., :n]
    moved = torch.arange(n, device=DEV) < hole.long().sum(2, keepdim=True)
    dst, src = torch.where(moved, dst, pad[..., :n]), torch.where(moved, src, pad[..., :n])
    to, of = place(dst), place(src)
    for plane in (s["k"], s["v"], s["k_scales"], s["v_scales"], s["weights"], s["positions"]):
        if plane is not None:
            plane[to] = plane[of]
    s["new_lengths"].copy_(s["lengths"].clamp(max=budget))


# -------------------------------------------------------------- the numbers
def work(case):
    c = case
    H, D = c["kv_heads"], c["dim"]
    one = D * (1 if c["dtype"] == "int8" else 2) + (4 if c["dtype"] == "int8" else 0)   # a stored row
    if c["kind"] == "append":
        counts = _counts(c)
        T, B = sum(counts), len(counts)
        n = T * H * (2 * 2 * D + 2 * one + 8 + (2 * 2 * D if c["stored"] else 0))
        return {"bytes": n + 12 * B + 4 * T, "flops": (6 if c["dtype"] == "int8" else 1) * 2 * T * H * D}
    total, B = sum(_lengths(c)), c["rows"]
    if c["kind"] == "attention":
        Hq = c["q_heads"]
        n = total * H * (2 * one + (8 if c["weights"] else 0)) + total * 4 / c["page"]
        return {"bytes": n + B * Hq * D * (2 + (2 if c["out"] == "bf16" else 4)), "flops": 4.0 * total * Hq * D}
    n = moved = 0.0
    for length in _lengths(c):
        b, r = c["budget"], c["recent"]
        if length > b:
            tail = length - b
            new = min(r, tail)
            moved += new + (tail - new) * max(0, b - r) / max(1, length - r)
            n += 8 * length
    return {"bytes": H * (n + moved * 2 * (2 * one + 8)), "flops": H * sum(_lengths(c))}


def exact(case, seed):
    """The outputs in 64 bits, row by row, from the definitions."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"append": _append_exact, "attention": _attention_exact, "evict": _evict_exact}[case["kind"]](case, s)


def _append_exact(c, s):
    res = {"k": None, "v": None, "k_stored": None, "v_stored": None, "k_scales": None, "v_scales": None}
    ps = c["page"]
    starts, lengths, last = s["starts"].tolist(), s["lengths"].tolist(), s["next_pos"].tolist()
    tables = s["tables"].tolist()
    weights, positions = s["weights"].double(), s["positions"].clone()
    where = []
    for b in range(len(lengths)):
        n = starts[b + 1] - starts[b]
        for i in range(n):
            at = lengths[b] - n + i
            where.append((tables[b][at // ps], at % ps, last[b] - n + i))
    page, off, pos = (torch.tensor(x, device=DEV) for x in zip(*where))
    weights[page, :, off] = 0.0
    positions[page, :, off] = pos.to(torch.int32)[:, None]
    for x in "kv":
        new = s["new_" + x].double()
        if c["dtype"] == "int8":
            sc = new.abs().amax(-1) / 127.0
            q = new / sc[..., None]
            q = torch.sign(q) * torch.floor(q.abs() + 0.5)
            pool = s[x + "_scales"].double()
            pool[page, :, off] = sc
            res[x + "_scales"] = pool
            new = q * sc[..., None]
        else:
            pool = s[x].double()
            pool[page, :, off] = new
            res[x] = pool
        if c["stored"]:
            res[x + "_stored"] = new
    return {**res, "weights": weights, "positions": None}


def _attention_exact(c, s):
    B, Hq, D = s["q"].shape
    H, ps, pages = c["kv_heads"], c["page"], s["k"].shape[0]
    out = torch.zeros((B, Hq, D), dtype=torch.float64, device=DEV)
    weights = s["weights"].double() if c["weights"] else None
    for b, n in enumerate(s["lengths"].tolist()):
        t = torch.arange(n, device=DEV)
        page = s["tables"][b, t // ps].long()
        t = t[(page >= 0) & (page < pages)]
        page, off = s["tables"][b, t // ps].long(), t % ps
        if t.numel() == 0:
            continue
        for h in range(H):
            k, v = s["k"][page, h, off].double(), s["v"][page, h, off].double()
            if c["dtype"] == "int8":
                k, v = k * s["k_scales"][page, h, off].double()[:, None], v * s["v_scales"][page, h, off].double()[:, None]
            heads = slice(h * (Hq // H), (h + 1) * (Hq // H))
            p = torch.softmax((s["q"][b, heads].double() @ k.T) * s["scale"], 1)
            out[b, heads] = p @ v
            if weights is not None:
                weights[page, h, off] += p.sum(0)
    return {"out": out, "weights": weights}


def _evict_exact(c, s):
    w, pos = s["weights"].double().cpu().numpy(), s["positions"].cpu().numpy()
    tables, lengths, last = s["tables"].cpu().numpy(), s["lengths"].tolist(), s["next_pos"].tolist()
    new_w = w.copy()
    for b, n in enumerate(lengths):
        if n <= c["budget"]:
            continue
        t = np.arange(n)
        page, off = tables[b][t // c["page"]], t % c["page"]
        for h in range(c["kv_heads"]):
            x = w[page, h, off].copy()
            x[pos[page, h, off] >= last[b] - c["recent"]] = np.inf
            stay = np.sort(np.lexsort((t, -x))[: c["budget"]])
            free = np.setdiff1d(t[: c["budget"]], stay)
            come = stay[stay >= c["budget"]]
            new_w[page[free], h, off[free]] = w[page[come], h, off[come]]
    return {"k": None, "v": None, "k_scales": None, "v_scales": None, "weights": torch.from_numpy(new_w),
            "positions": None, "new_lengths": None}
