"""Performance cases of what a serving program does around the paged key-value
cache, between the QKV projection and the O projection of a step:

  rotate   queries and keys of packed tokens normalised head by head (or not) and
           rotated to their positions, in both layouts, whole heads or their
           first part, with frequencies scaled for long contexts
  append   the same with the keys and the values written to the cache in the same
           pass, at the slots that a map gives (bf16, or int8 with a scale per
           token and head)
  pages    block tables and slot maps from the rows' lengths: pages of ended rows
           given back, a common prompt's pages shared, new pages taken, and the
           slot and position of every new token
  prefix   attention of one new token per row, where rows of a group share their
           first pages, which are read once for the group
  blocks   attention over the pages that a bound on their logits picks for each
           row and key-value head: bounds of the newest pages renewed, pages
           picked, attention over them

Layouts: k, v [pages][kv_heads][page_size][head_dim]; k_scales, v_scales (fp32)
[pages][kv_heads][page_size]; bounds bf16 [pages][kv_heads][2][head_dim] (least and
largest of the page's keys); tables int32 [rows][width]; lengths int32 [rows].
Sizes are those of the Llama-3-8B-shaped layer of bench.py (32 query heads, 8
key-value heads, head 128, QKV rows of 6144), of one rank of its TP=8 form (4 and 1
heads), and generic others.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
F32, F64, BF16, I32 = torch.float32, torch.float64, torch.bfloat16, torch.int32
FLT_MIN = 1.1754943508222875e-38


def _lib():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sneppx-alg_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import sneppx_quant
    return sneppx_quant.load()


# ------------------------------------------------------------------- cases
def _rotate(name, tokens, q_heads=32, kv_heads=8, dim=128, dims=128, interleaved=False, norm=False, far=8192):
    return {"name": name, "kind": "rotate", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "dims": dims, "interleaved": interleaved, "norm": norm, "far": far}


def _append(name, tokens, page=16, dtype="bf16", stored=False, **kw):
    return {**_rotate(name, tokens, **kw), "kind": "append", "page": page, "dtype": dtype, "stored": stored}


def _pages(name, rows, most, past, pages, page=16, shared=0, ended=0):
    return {"name": name, "kind": "pages", "rows": rows, "most": most, "past": past, "pages": pages, "page": page,
            "shared": shared, "ended": ended}


def _prefix(name, rows, groups, prefix, own_tokens, q_heads=32, kv_heads=8, dim=128, page=16, dtype="bf16",
            ragged=True, out="bf16"):
    return {"name": name, "kind": "prefix", "rows": rows, "groups": groups, "prefix": prefix, "own": own_tokens,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged,
            "out": out}


def _blocks(name, rows, length, budget, q_heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", ragged=True,
            out="bf16"):
    return {"name": name, "kind": "blocks", "rows": rows, "length": length, "budget": budget, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged, "out": out}


def listed():
    return [
        # 16 streams decoding, the layer's own queries and keys: the smallest call,
        # where launches and latency count
        _rotate("rotate_step", 16),
        # a packed batch of prompts, heads normalised first
        _rotate("rotate_prompt", 2320, norm=True),
        # the same 16 streams with their keys and values into the cache at once
        _append("append_step", 16, norm=True),
        # a batch of prompt chunks far into a long context: neighbouring pairs of
        # half of the head, an int8 cache, the stored rows returned
        _append("append_prompt_int8", 2320, page=64, dtype="int8", stored=True, dims=64, interleaved=True, far=131072),
        # 64 streams, each one token further
        _pages("pages_step", 64, 1, 4096, 20000),
        # prompts of up to 4096 tokens admitted to a large pool, most of them behind a
        # common one of 1024, while other rows have ended
        _pages("pages_prompts", 48, 4096, 0, 131072, shared=1024, ended=16),
        # 4 samples of one prompt of some 1100 tokens, just begun
        _prefix("prefix_token", 4, 1, 1104, 50),
        # 64 streams behind one prompt of 4096 tokens, with up to 512 of their own
        _prefix("prefix_batch64", 64, 1, 4096, 512),
        # one rank of a TP=8 group: five prompts of up to 8192, int8 cache, fp32 rows
        _prefix("prefix_groups_int8", 48, 5, 8192, 700, q_heads=4, kv_heads=1, page=64, dtype="int8", out="f32"),
        # 256 streams behind a document of 16384 tokens
        _prefix("prefix_wide", 256, 1, 16384, 128, page=64),
        # one stream at the end of a context of 128K tokens, 4096 of them attended to
        _blocks("blocks_long", 1, 131072, 64, ragged=False),
        # 16 streams of up to 32768 tokens, int8 cache, 2048 of them attended to
        _blocks("blocks_batch16_int8", 16, 32768, 64, page=32, dtype="int8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "pages", "prefix", "prefix", "blocks", "blocks"])
    dtype = rng.choice(["bf16", "bf16", "int8"])
    dim = rng.choice([128, 128, 128, 64, 80, 96, 256])
    page = rng.choice([16, 16, 32, 64, 128, 24])
    kv_heads = rng.choice([8, 8, 1, 2, 4, 12])
    q_heads = kv_heads * rng.choice([4, 4, 1, 2, 7, 8, 16])
    out = rng.choice(["bf16", "bf16", "f32"])
    per_token = 2 * kv_heads * dim * (1 if dtype == "int8" else 2)
    if kind in ("rotate", "append"):
        while True:
            tokens = _log(rng, 1, 6000)
            if tokens * (q_heads + 2 * kv_heads) * dim <= 40e6:
                break
        kw = dict(q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                  dims=max(8, int(dim * rng.choice([1, 1, 0.5, 0.25])) // 8 * 8), interleaved=rng.random() < 0.4,
                  norm=rng.random() < 0.5, far=_log(rng, 100, 1000000))
        c = _rotate("", tokens, **kw) if kind == "rotate" else \
            _append("", tokens, page, dtype, dtype == "int8" or rng.random() < 0.3, **kw)
    elif kind == "pages":
        rows, most = _log(rng, 1, 500), rng.choice([1, 1, _log(rng, 2, 4096)])
        if rows * most > 400000:
            most = 400000 // rows
        past = _log(rng, 1, 8000)
        if rows * past > 1000000:
            past = 1000000 // rows
        need = rows * (-(-(most + past) // page) + 1)
        c = _pages("", rows, most, past, int(need * rng.uniform(0.8, 6.0)) + 8, page,
                   rng.choice([0, 0, _log(rng, page, 2000)]), rng.choice([0, rows // 4]))
    elif kind == "prefix":
        while True:
            rows, prefix, mine = _log(rng, 1, 256), _log(rng, 100, 16384), _log(rng, 1, 1000)
            if rows * (prefix + mine) * kv_heads * dim * 4 <= 6e9 and rows * mine * per_token <= 400e6 \
                    and rows * prefix * q_heads * dim <= 256 * 16384 * 32 * 128:
                break
        c = _prefix("", rows, min(rows, rng.choice([1, 1, 2, 5])), prefix, mine, q_heads, kv_heads, dim, page, dtype,
                    rng.random() < 0.7, out)
    else:
        while True:
            rows, length = _log(rng, 1, 32), _log(rng, 200, 131072)
            if rows * length * per_token <= 600e6 and rows * length // page * q_heads * dim <= 64e6:
                break
        c = _blocks("", rows, length, rng.choice([16, 32, 64, 37]), q_heads, kv_heads, dim, page, dtype,
                    rng.random() < 0.7, out)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _spread(most, n, least=0):
    """n numbers from `least` to `most`, in no order."""
    at = [least + int((most - least) * ((0.37 + 0.618034 * i) % 1.0)) for i in range(n)]
    at[0] = most
    return at


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


def _freqs(c):
    """Radians per position of each pair: base 500000, and for contexts beyond
    8192 the long wavelengths stretched by how much further they reach."""
    f = 500000.0 ** (-2.0 * np.arange(c["dims"] // 2) / c["dims"])
    if c["far"] > 8192:
        turns = 8192 * f / (2 * math.pi)
        keep = np.clip((turns - 1) / 3, 0, 1)
        f = f * (keep + (1 - keep) * 8192 / c["far"])
    return torch.from_numpy(f).to(DEV)


def _rows(g, shape):
    return torch.randn(shape, device=DEV, generator=g)


def _pool(s, g, c, pages):
    """Keys and values of every page; a direction that queries share and some
    tokens answer, so that a few weights are large, as in a trained model's maps."""
    shape = (pages, c["kv_heads"], c["page"], c["dim"])
    u = _rows(g, (1, shape[1], 1, shape[3])) / math.sqrt(shape[3])
    for name in "kv":
        x = _rows(g, shape)
        if name == "k":
            x += 4.0 * u * (torch.rand(shape[:3] + (1,), device=DEV, generator=g) < 0.02)
        s[name + "_scales"] = None
        if c["dtype"] == "int8":
            x, s[name + "_scales"] = _codes(x)
            s[name] = x.to(torch.int8)
        else:
            s[name] = x.to(BF16)
        del x
    return u


def _queries(s, g, c, u, rows):
    """Queries as the QKV projection leaves them: the first part of its rows."""
    G, H, D = c["q_heads"], c["kv_heads"], c["dim"]
    q = _rows(g, (rows, G, D)) + 2.0 * math.sqrt(D) * u.view(H, 1, D).expand(H, G // H, D).reshape(G, D)
    qkv = torch.zeros((rows, (G + 2 * H) * D), dtype=BF16, device=DEV)
    s["q"] = qkv[:, : G * D].unflatten(1, (G, D))
    s["q"].copy_(q)
    s["out"] = torch.zeros((rows, G, D), dtype=BF16 if c["out"] == "bf16" else F32, device=DEV)
    s["scale"] = 1.0 / math.sqrt(D)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    s = {"case": c}
    {"rotate": _prepare_rotate, "append": _prepare_rotate, "pages": _prepare_pages, "prefix": _prepare_prefix,
     "blocks": _prepare_blocks}[c["kind"]](c, s, g)
    if own:   # the handles that a program keeps
        lib = _lib()
        if "freqs" in s:
            s["rotary"] = lib.rotary_from(s["freqs"], c["dim"], c["interleaved"], s["magnitude"], s["q_norm"], s["k_norm"],
                                          s["eps"])
        if "k" in s:
            s["cache"] = lib.kv_cache_from(s["k"], s["v"], s["k_scales"], s["v_scales"])
        if "refs" in s:
            s["pool"] = lib.kv_pages_from(s["refs"], c["page"])
    return s


def _prepare_rotate(c, s, g):
    T, G, H, D = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"]
    qkv = _rows(g, (T, (G + 2 * H) * D)).to(BF16)
    s["q_in"], s["k_in"], s["v_in"] = (x.unflatten(1, (-1, D)) for x in qkv.split((G * D, H * D, H * D), 1))
    s["freqs"], s["eps"] = _freqs(c), 1e-6
    s["magnitude"] = 1.0 if c["far"] <= 8192 else 0.1 * math.log(c["far"] / 8192) + 1.0
    s["q_norm"] = s["k_norm"] = None
    if c["norm"]:
        s["q_norm"], s["k_norm"] = (1.0 + 0.2 * _rows(g, (D,)) for _ in range(2))
    s["positions"] = torch.randint(0, c["far"], (T,), device=DEV, generator=g, dtype=I32)
    s["q_out"] = torch.zeros((T, G, D), dtype=BF16, device=DEV)
    if c["kind"] == "rotate":
        s["k_out"] = torch.zeros((T, H, D), dtype=BF16, device=DEV)
        return
    pages = -(-T // c["page"]) + 3
    perm = torch.randperm(pages, device=DEV, generator=g).to(I32)
    t = torch.arange(T, device=DEV, dtype=I32)
    s["slots"] = perm[(t // c["page"]).long()] * c["page"] + t % c["page"]
    if T > 2:
        s["slots"][T // 2] = -1     # a token that nobody keeps
    _pool(s, g, c, pages)
    s["k_stored"] = s["v_stored"] = None
    if c["stored"]:
        s["k_stored"], s["v_stored"] = (torch.zeros((T, H, D), dtype=BF16, device=DEV) for _ in range(2))


def _prepare_pages(c, s, g):
    B, ps, pages = c["rows"], c["page"], c["pages"]
    counts = [c["most"]] * B if c["most"] == 1 else _spread(c["most"], B, 1)
    past = _spread(c["past"], B)
    shared = c["shared"] // ps
    width = max(-(-(n + p) // ps) for n, p in zip(counts, past)) + shared + 1
    # what the pool and the rows hold: row 0 the common prompt, the others what came
    # before; the rows that have ended hold pages that go back
    held = [-(-p // ps) for p in past]
    held[0] = max(held[0], shared)
    perm = torch.randperm(pages, device=DEV, generator=g).to(I32).cpu().numpy()
    tables = np.full((B, width), -1, np.int32)
    at = 0
    for b in range(B):
        n = max(0, min(held[b], pages // 2 - at))
        tables[b, :n] = perm[at:at + n]
        at += n
        past[b] = min(past[b], n * ps) if b or not shared else n * ps
    sources = np.full(B, -1, np.int32)
    for b in range(1, B):
        if b <= c["ended"]:
            past[b] = 0
        if shared and past[b] == 0 and past[0] >= shared * ps:
            sources[b] = 0
    refs = np.zeros(pages, np.int32)
    np.add.at(refs, tables[tables >= 0], 1)
    refs[perm[-(pages // 8):]] = 1      # pages that other rows hold
    parts = [refs, tables.ravel(), np.array(past, np.int32), np.array(past, np.int32) + 5]
    # one buffer for what a pass changes and a copy of it, to begin each pass with
    s["before"] = torch.from_numpy(np.concatenate(parts)).to(DEV)
    s["now"] = s["before"].clone()
    s["refs"], t, s["lengths"], s["next_pos"] = s["now"].split([x.size for x in parts])
    s["tables"] = t.view(B, width)
    s["counts"] = torch.tensor(counts, dtype=I32, device=DEV)
    s["sources"] = torch.from_numpy(sources).to(DEV)
    s["shared"] = torch.full((B,), shared * ps, dtype=I32, device=DEV)
    T = sum(counts) + 7                 # a batch padded by a few tokens
    s["slots"], s["positions"] = (torch.zeros(T, dtype=I32, device=DEV) for _ in range(2))
    s["starts"], s["granted"] = torch.zeros(B + 1, dtype=I32, device=DEV), torch.zeros(B, dtype=I32, device=DEV)


def _groups(c):
    """First row of each group (and behind the last), its prefix, and the rows'
    lengths: whole pages are shared, and of several groups the last row has none."""
    B, n, ps = c["rows"], c["groups"], c["page"]
    loose = 1 if n > 1 and B > n and c["ragged"] else 0
    starts = [(B - loose) * i * (i + 2) // (n * (n + 2)) for i in range(n + 1)]
    prefix = [x // ps * ps for x in (_spread(c["prefix"], n) if n > 1 else [c["prefix"]])]
    mine = _spread(c["own"], B) if c["ragged"] else [c["own"]] * B
    of = [next((i for i in range(n) if starts[i] <= b < starts[i + 1]), -1) for b in range(B)]
    return starts, prefix, of, [mine[b] + (prefix[of[b]] if of[b] >= 0 else 0) for b in range(B)]


def _prepare_prefix(c, s, g):
    B, ps = c["rows"], c["page"]
    starts, prefix, of, lengths = _groups(c)
    width = max(1, -(-max(lengths) // ps))
    shared = [prefix[i] // ps if i >= 0 else 0 for i in of]
    pages = sum({i: n for i, n in zip(of, shared)}.values()) + sum(-(-n // ps) - k for n, k in zip(lengths, shared)) + 3
    perm = torch.randperm(pages, device=DEV, generator=g).to(I32).cpu().numpy()
    tables, at, first = np.full((B, width), -1, np.int32), 0, {}
    for b in range(B):
        n, have = -(-lengths[b] // ps), shared[b]
        if of[b] not in first:
            first[of[b]] = perm[at:at + have]
            at += have
        tables[b, :have] = first[of[b]][:have]
        tables[b, have:n] = perm[at:at + n - have]
        at += n - have
    s["tables"] = torch.from_numpy(tables).to(DEV)
    s["lengths"] = torch.tensor(lengths, dtype=I32, device=DEV)
    s["groups"] = torch.tensor(starts, dtype=I32, device=DEV)
    s["prefix"] = torch.tensor(prefix, dtype=I32, device=DEV)
    s["longest"] = max(lengths)
    u = _pool(s, g, c, pages)
    _queries(s, g, c, u, B)


def _block_lengths(c):
    return _spread(c["length"], c["rows"]) if c["ragged"] else [c["length"]] * c["rows"]


def _prepare_blocks(c, s, g):
    B, ps, H = c["rows"], c["page"], c["kv_heads"]
    lengths = _block_lengths(c)
    width = max(1, -(-max(lengths) // ps))
    pages = B * width + 3
    s["tables"] = torch.randperm(pages, device=DEV, generator=g)[: B * width].to(I32).view(B, width).clone()
    s["lengths"] = torch.tensor(lengths, dtype=I32, device=DEV)
    u = _pool(s, g, c, pages)
    _queries(s, g, c, u, B)
    # the bounds as the steps before left them: of whole pages
    k = s["k"].to(F32)
    if c["dtype"] == "int8":
        k = (k * s["k_scales"].unsqueeze(-1)).to(BF16).to(F32)
    s["bounds"] = torch.stack([k.amin(2), k.amax(2)], 2).to(BF16)
    s["picked"] = torch.zeros((B, H, c["budget"]), dtype=I32, device=DEV)
    s["picked_lengths"] = torch.zeros(B, dtype=I32, device=DEV)
    s["first"], s["recent"] = 1, 2


# --------------------------------------------------------------- the passes
def run(state):
    s, c = state, state["case"]
    if c["kind"] == "rotate":
        (_rotate_own if own else _rotate_plain)(s)
        return {"q": s["q_out"], "k": s["k_out"]}
    if c["kind"] == "append":
        (_append_own if own else _append_plain)(s)
        b16 = c["dtype"] == "bf16"
        return {"q": s["q_out"], "k": s["k"] if b16 else None, "v": s["v"] if b16 else None, "k_scales": s["k_scales"],
                "v_scales": s["v_scales"], "k_stored": s["k_stored"], "v_stored": s["v_stored"]}
    if c["kind"] == "pages":
        s["now"].copy_(s["before"])     # pages, tables and lengths as at the first pass
        (_pages_own if own else _pages_plain)(s)
        return {"refs": s["refs"], "tables": s["tables"], "lengths": s["lengths"], "next_pos": s["next_pos"],
                "slots": s["slots"], "positions": s["positions"], "starts": s["starts"], "granted": s["granted"]}
    if c["kind"] == "prefix":
        (_prefix_own if own else _prefix_plain)(s)
        return {"out": s["out"]}
    (_blocks_own if own else _blocks_plain)(s)
    return {"out": s["out"], "bounds": s["bounds"], "picked": s["picked"], "picked_lengths": s["picked_lengths"]}


def _rotate_own(s):
    s["rotary"].apply(s["q_in"], s["k_in"], s["positions"], s["q_out"], s["k_out"])


def _append_own(s):
    s["cache"].append_rotated(s["rotary"], s["q_in"], s["k_in"], s["v_in"], s["slots"], s["positions"], s["q_out"],
                              k_stored=s["k_stored"], v_stored=s["v_stored"])


def _pages_own(s):
    p, c = s["pool"], s["case"]
    if c["ended"]:
        p.release(s["tables"], s["lengths"])
    if c["shared"]:
        p.share(s["tables"], s["lengths"], s["sources"], s["shared"], next_pos=s["next_pos"])
    p.reserve(s["tables"], s["lengths"], s["slots"], counts=s["counts"], next_pos=s["next_pos"],
              positions=s["positions"], starts=s["starts"], granted=s["granted"])


def _prefix_own(s):
    c = s["case"]
    s["cache"].attention_shared(s["q"], s["out"], s["tables"], s["lengths"], s["longest"], s["groups"], s["prefix"],
                                c["prefix"], c["own"], s["scale"])


def _blocks_own(s):
    c = s["case"]
    s["cache"].key_bounds(s["bounds"], s["tables"], s["lengths"])
    s["cache"].pick(s["q"], s["bounds"], s["tables"], s["lengths"], c["length"], s["picked"], s["picked_lengths"],
                    s["first"], s["recent"])
    s["cache"].attention_picked(s["q"], s["out"], s["picked"], s["picked_lengths"], s["scale"])


def _turned(s, x, norm):
    """Heads in 32 bits, normalised and rotated; the angles in 64 bits, for a far
    position's has no fraction left in 32."""
    c, d = s["case"], s["case"]["dims"]
    x = x.to(F32)
    if norm is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * norm
    angle = s["positions"].to(F64)[:, None, None] * s["freqs"]
    cos, sin = (angle.cos() * s["magnitude"]).to(F32), (angle.sin() * s["magnitude"]).to(F32)
    if c["interleaved"]:
        a, b = x[..., 0:d:2], x[..., 1:d:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., : d // 2], x[..., d // 2:d]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., d:]], -1)


def _rotate_plain(s):
    s["q_out"].copy_(_turned(s, s["q_in"], s["q_norm"]))
    s["k_out"].copy_(_turned(s, s["k_in"], s["k_norm"]))


def _put(pool, scales, stored, x, page, off, there):
    """Rows x to their places; those without one go where the page's first row is
    and leave it as it was."""
    code = x
    if scales is not None:
        code, sc = _codes(x)
        x = code * sc.unsqueeze(-1)
        scales[page, :, off] = torch.where(there[:, None], sc, scales[page, :, off])
    kept = pool[page, :, off]
    pool[page, :, off] = torch.where(there[:, None, None], code.to(pool.dtype), kept)
    if stored is not None:
        stored.copy_(torch.where(there[:, None, None], x.to(BF16), stored))


def _append_plain(s):
    ps = s["k"].shape[2]
    s["q_out"].copy_(_turned(s, s["q_in"], s["q_norm"]))
    there = s["slots"] >= 0
    last = s["k"].shape[0] * ps - 1        # (a slot that no token has)
    taken = torch.zeros(last + 1, dtype=torch.bool, device=DEV).index_fill(0, torch.where(there, s["slots"], s["slots"][0]).long(), True)
    free = torch.argmin(taken.to(torch.uint8))
    slot = torch.where(there, s["slots"].long(), free)
    page, off = slot // ps, slot % ps
    _put(s["k"], s["k_scales"], s["k_stored"], _turned(s, s["k_in"], s["k_norm"]), page, off, there)
    _put(s["v"], s["v_scales"], s["v_stored"], s["v_in"].to(F32), page, off, there)


def _pages_plain(s):
    c, refs, tables = s["case"], s["refs"], s["tables"]
    ps, pages = c["page"], c["pages"]
    B, W = tables.shape
    e = torch.arange(W, device=DEV, dtype=I32)
    trash = torch.zeros(1, dtype=I32, device=DEV)

    def up(n):
        return torch.div(n + ps - 1, ps, rounding_mode="floor")

    def add(where, page, by):
        """refs[page] += by, at the places of `where`."""
        at = torch.where(where, page, pages).long().flatten()
        refs.copy_(torch.cat([refs, trash]).index_add(0, at, torch.full_like(at, by, dtype=I32))[:pages])

    if c["ended"]:
        back = (e >= up(s["lengths"])[:, None]) & (tables >= 0)
        add(back, tables, -1)
        tables.copy_(torch.where(back, -1, tables))
    if c["shared"]:
        takes = (s["sources"] >= 0)[:, None] & (e < (s["shared"] // ps)[:, None])
        theirs = tables[s["sources"].clamp(min=0).long()]
        takes &= theirs >= 0
        tables.copy_(torch.where(takes, theirs, tables))
        add(takes, theirs, 1)
        took = s["sources"] >= 0
        s["lengths"].copy_(torch.where(took, s["shared"], s["lengths"]))
        s["next_pos"].copy_(torch.where(took, s["shared"], s["next_pos"]))
    n, want = s["lengths"], s["counts"]
    fits = n + want <= W * ps
    missing = (e >= up(n)[:, None]) & (e < up(n + want)[:, None]) & (tables < 0) & fits[:, None]
    need = missing.sum(1)
    ok = fits & ((need == 0) | (need.cumsum(0) <= (refs == 0).sum()))
    get = missing & ok[:, None]
    order = torch.argsort((refs != 0).to(torch.uint8), stable=True).to(I32)     # free pages, the lowest first
    nth = (get.flatten().cumsum(0) - 1).clamp(0, pages - 1)
    new = order[nth].view(B, W)
    tables.copy_(torch.where(get, new, tables))
    add(get, new, 1)
    s["starts"][1:] = want.cumsum(0)
    t = torch.arange(s["slots"].numel(), device=DEV, dtype=I32)
    row = (torch.searchsorted(s["starts"], t, right=True) - 1).clamp(max=B - 1)
    i = t - s["starts"][row]
    ok_t = ok[row] & (t < s["starts"][B])
    slot = n[row] + i
    page = tables[row, torch.where(ok_t, slot // ps, 0).long()]
    s["slots"].copy_(torch.where(ok_t & (page >= 0), page * ps + slot % ps, -1))
    s["positions"].copy_(torch.where(ok_t, s["next_pos"][row] + i, -1))
    s["granted"].copy_(torch.where(ok, want, 0))
    s["lengths"] += s["granted"]
    s["next_pos"] += s["granted"]


def _gathered(pool, scales, page, off, valid):
    x = pool[page, :, off].to(F32)                   # [rows][length][kv_heads][dim]
    if scales is not None:
        x = x * scales[page, :, off].unsqueeze(-1)
    return torch.where(valid[:, :, None, None], x, torch.zeros_like(x)).transpose(1, 2).contiguous()


def _softmax(logits, there):
    logits = torch.where(there, logits, torch.full_like(logits, -math.inf))
    top = logits.amax(-1, keepdim=True)
    p = torch.where(there, torch.exp(logits - top), torch.zeros_like(logits))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _prefix_plain(s):
    ps = s["k"].shape[2]
    B, Hq, D = s["q"].shape
    H = s["k"].shape[1]
    t = torch.arange(s["longest"], device=DEV)
    page = s["tables"][:, t // ps].long()
    valid = t[None] < s["lengths"][:, None]
    page, off = torch.where(valid, page, 0), (t % ps).expand(B, -1)
    K = _gathered(s["k"], s["k_scales"], page, off, valid)
    q = s["q"].to(F32).reshape(B, H, Hq // H, D)
    logits = torch.matmul(q, K.transpose(2, 3)) * s["scale"]
    del K
    p = _softmax(logits, valid[:, None, None, :])
    del logits
    V = _gathered(s["v"], s["v_scales"], page, off, valid)
    s["out"].copy_(torch.matmul(p, V).reshape(B, Hq, D))


def _blocks_plain(s):
    c, ps, n = s["case"], s["k"].shape[2], s["case"]["budget"]
    B, Hq, D = s["q"].shape
    H, W = s["k"].shape[1], s["tables"].shape[1]
    lengths, heads = s["lengths"].long(), torch.arange(H, device=DEV)
    # the newest page's least and largest keys
    any_ = lengths > 0
    page = torch.where(any_, s["tables"].gather(1, ((lengths - 1).clamp(min=0) // ps)[:, None])[:, 0], s["tables"][:, 0]).long()
    k = s["k"][page].to(F32)
    if c["dtype"] == "int8":
        k = (k * s["k_scales"][page].unsqueeze(-1)).to(BF16).to(F32)
    used = (torch.arange(ps, device=DEV) < ((lengths - 1) % ps + 1)[:, None])[:, None, :, None]
    new = torch.stack([torch.where(used, k, math.inf).amin(2), torch.where(used, k, -math.inf).amax(2)], 2).to(BF16)
    s["bounds"][page] = torch.where(any_[:, None, None, None], new, s["bounds"][page])
    # the largest logit that a page could have for any of the group's queries, in 64
    # bits, for pages next to the border; then in 32, and of equal ones the first
    bound = s["bounds"][s["tables"].long()].to(F64)                                   # [rows][pages][heads][2][dim]
    q = s["q"].to(F64).view(B, H, Hq // H, D)
    score = torch.matmul(q.clamp(min=0), bound[..., 1, :].permute(0, 2, 3, 1).contiguous()) \
        + torch.matmul(q.clamp(max=0), bound[..., 0, :].permute(0, 2, 3, 1).contiguous())
    del bound
    score = score.amax(2).to(F32)
    e = torch.arange(W, device=DEV)
    have = ((lengths + ps - 1) // ps)[:, None]
    stays = (e < s["first"]) | (e >= have - s["recent"])
    score = torch.where(stays[:, None], math.inf, score)
    score = torch.where((e < have)[:, None], score, -math.inf)
    order = torch.argsort(score, dim=2, descending=True, stable=True)
    few = torch.arange(W, device=DEV) < torch.minimum(have, torch.full_like(have, n))
    kept = torch.zeros((B, H, W), dtype=torch.bool, device=DEV).scatter(2, order, few[:, None].expand(B, H, W))
    to = torch.where(kept, kept.long().cumsum(2) - 1, n)
    picked = torch.full((B, H, n + 1), -1, dtype=I32, device=DEV)
    picked.scatter_(2, to, s["tables"][:, None].expand(B, H, W))
    s["picked"].copy_(picked[..., :n])
    cut = (have[:, 0] - n).clamp(min=0)
    s["picked_lengths"].copy_(lengths - cut * ps)
    # attention over them
    t = torch.arange(n * ps, device=DEV)
    valid = (t[None] < s["picked_lengths"][:, None])[:, None].expand(B, H, -1)
    page = torch.where(valid, s["picked"][:, :, t // ps], 0).long()
    off = (t % ps).expand(B, H, -1)

    def rows(pool, scales):
        x = pool[page, heads[None, :, None], off].to(F32)
        if scales is not None:
            x = x * scales[page, heads[None, :, None], off].unsqueeze(-1)
        return torch.where(valid[..., None], x, torch.zeros_like(x))

    logits = torch.matmul(s["q"].to(F32).view(B, H, Hq // H, D),
                          rows(s["k"], s["k_scales"]).transpose(2, 3).contiguous()) * s["scale"]
    p = _softmax(logits, valid[:, :, None, :])
    s["out"].copy_(torch.matmul(p, rows(s["v"], s["v_scales"])).reshape(B, Hq, D))


# -------------------------------------------------------------- the numbers
def work(case):
    c = case
    if c["kind"] == "pages":
        B, ps = c["rows"], c["page"]
        counts = [c["most"]] * B if c["most"] == 1 else _spread(c["most"], B, 1)
        T, new = sum(counts), sum(-(-n // ps) for n in counts)
        return {"bytes": 4 * (2 * T + 7 * B + 3 * new + (c["shared"] // ps) * B), "flops": 6 * T}
    H, D = c["kv_heads"], c["dim"]
    Hq = c["q_heads"]
    if c["kind"] in ("rotate", "append"):
        T = c["tokens"]
        n = T * (Hq + H) * D * 4 + 4 * T + 4 * c["dims"]
        flops = T * (Hq + H) * (3.0 * c["dims"] + (4 * D if c["norm"] else 0))
        if c["kind"] == "append":
            # (queries read and written, keys and values read, and written as the cache holds them)
            row = D * (1 if c["dtype"] == "int8" else 2) + (4 if c["dtype"] == "int8" else 0)
            n = T * (Hq * D * 4 + 2 * H * (D * 2 + row + (2 * D if c["stored"] else 0)) + 8) + 4 * c["dims"]
            flops += (12.0 if c["dtype"] == "int8" else 0.0) * T * H * D
        return {"bytes": n, "flops": flops}
    one = 2 * (D * (1 if c["dtype"] == "int8" else 2) + (4 if c["dtype"] == "int8" else 0))   # a token's key and value
    B = c["rows"]
    ends = B * Hq * D * (2 + (2 if c["out"] == "bf16" else 4))
    if c["kind"] == "prefix":
        starts, prefix, of, lengths = _groups(c)
        held = sum(p for i, p in enumerate(prefix) if starts[i + 1] > starts[i])
        held += sum(n - (prefix[of[b]] if of[b] >= 0 else 0) for b, n in enumerate(lengths))
        return {"bytes": held * H * one + held * 4 / c["page"] + ends, "flops": 4.0 * sum(lengths) * Hq * D}
    ps, n = c["page"], c["budget"]
    pages = [-(-x // ps) for x in _block_lengths(c)]
    seen = sum(x - max(0, p - n) * ps for x, p in zip(_block_lengths(c), pages))
    return {"bytes": sum(pages) * (H * 4 * D + 4) + B * H * ps * one / 2 + seen * H * one + ends,
            "flops": 4.0 * seen * Hq * D + 4.0 * sum(pages) * Hq * D}


def exact(case, seed):
    """The outputs in 64 bits, row by row, from the definitions."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "pages":
        return None
    return {"rotate": _rotate_exact, "append": _rotate_exact, "prefix": _prefix_exact,
            "blocks": _blocks_exact}[case["kind"]](case, s)


def _rotate_exact(c, s):
    d = c["dims"]

    def turn(x, norm):
        x = x.double()
        if norm is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * norm.double()
        i = torch.arange(d // 2, device=DEV)
        a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + d // 2)
        z = torch.complex(x[..., a], x[..., b])
        angle = s["positions"].double()[:, None] * s["freqs"][None]
        z = z * torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, None]
        x = x.clone()
        x[..., a], x[..., b] = z.real, z.imag
        return x

    res = {"q": turn(s["q_in"], s["q_norm"])}
    k, v = turn(s["k_in"], s["k_norm"]), s["v_in"].double()
    if c["kind"] == "rotate":
        return {**res, "k": k}
    keep = s["slots"] >= 0
    slot = s["slots"][keep].long()
    for name, x in (("k", k), ("v", v)):
        res[name] = res[name + "_scales"] = res[name + "_stored"] = None
        if c["dtype"] == "int8":
            sc = x.abs().amax(-1) / 127.0
            x = torch.sign(x) * torch.floor((x / sc[..., None]).abs() + 0.5) * sc[..., None]
            plane = s[name + "_scales"].double()
            plane[slot // c["page"], :, slot % c["page"]] = sc[keep]
            res[name + "_scales"] = plane
        else:
            pool = s[name].double()
            pool[slot // c["page"], :, slot % c["page"]] = x[keep]
            res[name] = pool
        if c["stored"]:
            res[name + "_stored"] = torch.where(keep[:, None, None], x, torch.zeros_like(x))
    return res


def _attend(c, s, b, h, page, off):
    group = c["q_heads"] // c["kv_heads"]
    k, v = s["k"][page, h, off].double(), s["v"][page, h, off].double()
    if c["dtype"] == "int8":
        k, v = k * s["k_scales"][page, h, off].double()[:, None], v * s["v_scales"][page, h, off].double()[:, None]
    p = torch.softmax((s["q"][b, h * group:(h + 1) * group].double() @ k.T) * s["scale"], 1)
    return p @ v


def _prefix_exact(c, s):
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    group = c["q_heads"] // c["kv_heads"]
    for b, n in enumerate(s["lengths"].tolist()):
        t = torch.arange(n, device=DEV)
        page, off = s["tables"][b, t // c["page"]].long(), t % c["page"]
        for h in range(c["kv_heads"] if n else 0):
            out[b, h * group:(h + 1) * group] = _attend(c, s, b, h, page, off)
    return {"out": out}


def _blocks_exact(c, s):
    ps, n, group = c["page"], c["budget"], c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    bounds = s["bounds"].double()
    for b, length in enumerate(s["lengths"].tolist()):
        if length == 0:
            continue
        have = -(-length // ps)
        table = s["tables"][b, :have].long()
        k = s["k"][table[-1]].double()
        if c["dtype"] == "int8":
            k = (s["k"][table[-1]].float() * s["k_scales"][table[-1]][..., None]).to(BF16).double()
        k = k[:, : (length - 1) % ps + 1]
        bounds[table[-1]] = torch.stack([k.amin(1), k.amax(1)], 1)
        for h in range(c["kv_heads"]):
            kept = list(range(have))
            if have > n:
                q = s["q"][b, h * group:(h + 1) * group].double()
                low, high = bounds[table, h, 0], bounds[table, h, 1]
                best = torch.maximum(q[:, None] * low, q[:, None] * high).sum(-1).amax(0).float().cpu().numpy()
                best[: s["first"]] = best[have - s["recent"]:] = np.inf
                kept = np.sort(np.lexsort((np.arange(have), -best))[:n]).tolist()
            page = table[torch.tensor(kept, device=DEV)].repeat_interleave(ps)
            tokens = length - max(0, have - n) * ps
            off = torch.arange(ps, device=DEV).repeat(len(kept))
            out[b, h * group:(h + 1) * group] = _attend(c, s, b, h, page[:tokens], off[:tokens])
    return {"out": out, "bounds": bounds, "picked": None, "picked_lengths": None}
