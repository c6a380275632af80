"""Performance cases of the paged key-value cache and the operators on it.

A scene that grows keeps the keys and values of its views' tokens in pages. One pass is one operator
call on device buffers, in the plain form (elementary torch operations in 32 bits, the selection's
scores in 64) or, with `own`, through the library's kernel entry points. `exact` restates every
operator from its definition in 64 bits, one sequence at a time.

Layout: key and value pools [pages, kv_heads, page_size, 64]; position p of sequence i lies in row
p % page_size of page table[i, p // page_size]; its slot is page * page_size + row.
"""
import math
import os
import random
import sys

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"
VIEW = 1037          # tokens of a 518x392 view: 37 x 28 patches and the class token
SCENE = 24889        # 24 such views and the scale token
BASE = 100.0         # rotation base of Depth Anything 3
EPS = 1e-5
_held = {}           # the library context that a program keeps


# --- the cases ----------------------------------------------------------------------------------

def listed():
    return [
        # 32 scenes, one new token each: what a serving loop does before every step. Latency.
        {"name": "tables_step", "kind": "tables", "n": 32, "max_past": SCENE - 1, "add": "one", "ps": 16},
        # 64 scenes that get up to 24 views at once: a million slots.
        {"name": "tables_views", "kind": "tables", "n": 64, "max_past": 4 * VIEW, "add": "views", "ps": 64},
        # One token of each of 32 scenes, 12 heads (the 768-wide global blocks). Latency.
        {"name": "rope_step_bf16", "kind": "rope", "tokens": 32, "heads": 12, "kv": 12, "norm": "layer", "rope": "grid",
         "cache": True, "ps": 16, "dtype": "bf16"},
        # A DA3-Small view (27 x 36 patches and the camera token) in fp32, 6 heads.
        {"name": "rope_view_f32", "kind": "rope", "tokens": 973, "heads": 6, "kv": 6, "norm": "layer", "rope": "grid",
         "cache": True, "ps": 32, "dtype": "f32"},
        # All tokens of 24 views in f16, shared key heads, positions on a line: the cache's first fill.
        {"name": "rope_scene_f16", "kind": "rope", "tokens": SCENE, "heads": 24, "kv": 8, "norm": "rms", "rope": "line",
         "cache": True, "ps": 64, "dtype": "f16"},
        # The page of each scene's new token, after the step. Latency.
        {"name": "bounds_step_bf16", "kind": "bounds", "n": 32, "max_len": 8 * VIEW, "add": "one", "heads": 12, "kv": 12,
         "ps": 16, "dtype": "bf16"},
        # Every page of four scenes, after their first fill.
        {"name": "bounds_scenes_f16", "kind": "bounds", "n": 4, "max_len": SCENE, "add": "all", "heads": 24, "kv": 8, "ps": 64,
         "dtype": "f16"},
        # One token of a few thumbnails' scenes in fp32: a handful of keys. Latency.
        {"name": "paged_small_f32", "kind": "paged", "n": 3, "max_len": 188, "heads": 6, "kv": 6, "ps": 8, "dtype": "f32"},
        # The scale token against one scene of 24 views: few rows, a long axis.
        {"name": "paged_scene_bf16", "kind": "paged", "n": 1, "max_len": SCENE, "heads": 12, "kv": 12, "ps": 16, "dtype": "bf16"},
        # 48 scenes of all lengths, one of them empty, four query heads to a key head.
        {"name": "paged_batch_f16", "kind": "paged", "n": 48, "max_len": SCENE, "heads": 32, "kv": 8, "ps": 64, "dtype": "f16"},
        # One token against a scene of 100 views, an eighth of its pages.
        {"name": "sparse_scene_bf16", "kind": "sparse", "n": 1, "max_len": 100 * VIEW + 1, "heads": 12, "kv": 12, "ps": 32,
         "topk": 405, "dtype": "bf16"},
        # 16 scenes of all lengths, shared key heads, 64 pages each.
        {"name": "sparse_batch_f16", "kind": "sparse", "n": 16, "max_len": 4 * SCENE, "heads": 32, "kv": 8, "ps": 64, "topk": 64,
         "dtype": "f16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tables", "rope", "rope", "bounds", "paged", "paged", "paged", "sparse", "sparse"])
    ps = rng.choice([8, 16, 32, 64, 128])
    heads, kv = rng.choice([(6, 6), (12, 12), (16, 16), (24, 8), (20, 4), (8, 1), (32, 2), (32, 8)])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "tables":
        add = rng.choice(["one", "views"])
        return {"kind": kind, "n": _log_int(rng, 1, 64 if add == "views" else 1000), "max_past": _log_int(rng, 1, SCENE),
                "add": add, "ps": ps}
    if kind == "rope":
        if (heads, kv) == (32, 8):
            heads = 28
        most = SCENE if dtype != "f32" else SCENE // 2
        return {"kind": kind, "tokens": _log_int(rng, 1, most), "heads": heads, "kv": kv,
                "norm": rng.choice(["none", "layer", "rms"]), "rope": rng.choice(["none", "line", "grid"]),
                "cache": rng.random() < 0.7, "ps": ps, "dtype": dtype}
    most = (SCENE if kind != "sparse" else 4 * SCENE) // (2 if dtype == "f32" else 1)
    max_len = _log_int(rng, 1, most)
    n = _log_int(rng, 1, max(1, min(48, 48 * 8 * SCENE // (2 * max_len * kv))))
    c = {"kind": kind, "n": n, "max_len": max_len, "heads": heads, "kv": kv, "ps": ps, "dtype": dtype}
    if kind == "bounds":
        c["n"] = min(n, 4) if max_len > 4 * VIEW else n
        c["add"] = rng.choice(["one", "view", "all"])
    if kind == "sparse":
        c["n"] = min(n, 16)
        c["topk"] = _log_int(rng, 1, 256)
    return c


# --- sizes, which the case alone decides ----------------------------------------------------------

def _spread(n, most):
    """n lengths from 1 to `most`, spread over their logarithm in no order, the longest among them; from
    eight on one of them is 0 (a scene without views yet)."""
    out = [int(round(math.exp(((0.5 + 0.6180339887 * i) % 1.0) * math.log(max(most, 1))))) for i in range(n)]
    out[0] = most
    if n >= 8:
        out[3] = 0
    return [min(most, max(0, v)) for v in out]


def _lengths(c):
    """(past, add) of every sequence: `add` new positions behind `past`."""
    n = c["n"]
    if c["kind"] == "tables":
        past = _spread(n, c["max_past"])
        return past, [1] * n if c["add"] == "one" else [VIEW * (1 + (7 * i + 3) % 24) for i in range(n)]
    lens = _spread(n, c["max_len"])
    step = {"one": 1, "view": VIEW, "all": c["max_len"]}[c.get("add", "one")]
    add = [min(v, step) for v in lens]
    return [v - a for v, a in zip(lens, add)], add


def _width(c, past, add):
    return max(1, max(-(-(p + a) // c["ps"]) for p, a in zip(past, add)))


# --- what a program has in hand -----------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * scale


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(g, c, lens, width):
    """A table [n, width] of distinct pages in random order, -1 behind the last one; the number of pages."""
    used = [-(-v // c["ps"]) for v in lens]
    total = sum(used)
    pages = total + 3
    ids = torch.randperm(pages, device=DEV, generator=g)[:total].to(torch.int32)
    at = torch.arange(width, device=DEV)[None, :] < torch.tensor(used, device=DEV)[:, None]
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    table[at] = ids
    return table, pages


def _pool(g, pages, c, spread=1.0):
    """Keys or values: neighbouring tokens are alike (a page's tokens share a part)."""
    kv, ps, td = c["kv"], c["ps"], TORCH[c["dtype"]]
    out = torch.empty(pages, kv, ps, 64, dtype=td, device=DEV)
    step = max(1, (1 << 26) // (kv * ps * 64))
    for a in range(0, pages, step):
        m = min(step, pages - a)
        out[a:a + m] = (_randn(g, m, kv, ps, 64, scale=0.8) + _randn(g, m, kv, 1, 64, scale=0.6 * spread)).to(td)
    return out


def _bounds_of(k):
    return torch.stack([k.amin(2), k.amax(2)], 2).contiguous()


def prepare(case, seed):
    c, kind, g = case, case["kind"], _gen(seed)
    s = {"c": c}
    if kind == "rope":
        T, heads, kv, ps, td = c["tokens"], c["heads"], c["kv"], c["ps"], TORCH[c["dtype"]]
        s["qkv"] = (_randn(g, T, (heads + 2 * kv) * 64) + _randn(g, (heads + 2 * kv) * 64, scale=0.3)).to(td)
        for name in ("qw", "kw"):
            s[name] = 1 + _randn(g, 64, scale=0.1)
        for name in ("qb", "kb"):
            s[name] = _randn(g, 64, scale=0.1)
        if c["rope"] == "grid":   # rows and columns of patches, the camera token at the origin
            s["pos"] = torch.randint(0, 38, (T, 2), device=DEV, generator=g, dtype=torch.int32)
        else:
            s["pos"] = (torch.arange(T, device=DEV) + torch.randint(0, SCENE, (1,), device=DEV, generator=g)).to(torch.int32)
        s["q"] = torch.empty(T, heads * 64, dtype=td, device=DEV)
        if c["cache"]:
            pages = -(-T // ps) + 3
            s["slots"] = torch.randperm(pages, device=DEV, generator=g)[:-(-T // ps)].repeat_interleave(ps)[:T] * ps
            s["slots"] = (s["slots"] + torch.arange(T, device=DEV) % ps).to(torch.int32)
            s["k"] = torch.zeros(pages, kv, ps, 64, dtype=td, device=DEV)
            s["v"] = torch.zeros(pages, kv, ps, 64, dtype=td, device=DEV)
        else:
            s["kout"] = torch.empty(T, kv * 64, dtype=td, device=DEV)
    elif kind == "tables":
        past, add = _lengths(c)
        ps, n, width = c["ps"], c["n"], _width(c, past, add)
        s["past"], s["add"], s["width"], s["cap"] = _int(past), _int(add), width, sum(add)
        s["table"], have = _pages(g, c, past, width)
        need = sum(-(-(p + a) // ps) - -(-p // ps) for p, a in zip(past, add))
        s["pool"] = have + torch.randperm(need + 5, device=DEV, generator=g).to(torch.int32)
        s["used"] = _int([random.Random(seed).randint(0, 5)])
        for name, m in (("lens", n), ("starts", n + 1), ("slots", s["cap"]), ("positions", s["cap"]), ("used_out", 1), ("status", 1)):
            s[name] = torch.empty(m, dtype=torch.int32, device=DEV)
    else:
        past, add = _lengths(c)
        lens = [p + a for p, a in zip(past, add)]
        s["width"] = _width(c, past, add)
        s["lens"], s["add"] = _int(lens), _int(add)
        s["table"], s["pages"] = _pages(g, c, lens, s["width"])
        s["k"] = _pool(g, s["pages"], c)
        if kind == "bounds":
            s["bounds"] = torch.zeros(s["pages"], c["kv"], 2, 64, dtype=s["k"].dtype, device=DEV)
            s["v"] = s["k"]   # a call reads no values
        else:
            s["v"] = _pool(g, s["pages"], c)
            s["q"] = (_randn(g, c["n"], c["heads"] * 64) * 1.2).to(s["k"].dtype)
            s["out"] = torch.empty_like(s["q"])
            if kind == "sparse":
                s["bounds"] = _bounds_of(s["k"])
                s["selected"] = torch.empty(c["n"], c["kv"], c["topk"], dtype=torch.int32, device=DEV)
    s["ptr"] = {name: t.data_ptr() for name, t in s.items() if isinstance(t, torch.Tensor)}
    torch.cuda.synchronize()
    return s


# --- one pass -------------------------------------------------------------------------------------

def _library():
    """The package and the context on device 0 whose stream the calls go to."""
    if not _held:
        package = os.path.join(os.getcwd(), "splatting-rs_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import splathip
        _held["package"], _held["context"] = splathip, splathip.Context(0)
    return _held["package"], _held["context"]


def _cache(lib, s):
    """What a program keeps with its cache: its description and a workspace for the calls on it."""
    if "cache" not in s:
        c, p = s["c"], s["ptr"]
        s["cache"] = lib.KvCache(lib.DTYPES[c["dtype"]], p["k"], p["v"], s["k"].shape[0], c["ps"], c["kv"])
        size = 0
        if c["kind"] == "paged":
            size = lib.paged_attention_workspace(s["cache"], c["n"], c["heads"], c["max_len"])
        elif c["kind"] == "sparse":
            size = lib.sparse_attention_workspace(s["cache"], c["n"], c["heads"], c["max_len"], c["topk"])
        s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
        s["ptr"]["workspace"], s["bytes"] = s["workspace"].data_ptr(), size
    return s["cache"]


def _run_own(s):
    lib, ctx = _library()
    c, p, kind = s["c"], s["ptr"], s["c"]["kind"]
    if kind == "tables":
        ctx.kernel_block_tables(c["n"], p["past"], p["add"], c["ps"], p["pool"], s["pool"].numel(), p["used"], p["table"],
                                s["width"], p["lens"], p["starts"], p["slots"], p["positions"], s["cap"], p["used_out"],
                                p["status"])
        return {name: s[name] for name in ("table", "lens", "starts", "slots", "positions", "used_out", "status")}
    if kind == "rope":
        norm = {"none": lib.NORM_NONE, "layer": lib.NORM_LAYER, "rms": lib.NORM_RMS}[c["norm"]]
        rope = {"none": lib.ROPE_NONE, "line": lib.ROPE_LINE, "grid": lib.ROPE_GRID}[c["rope"]]
        bias = c["norm"] == "layer"
        total, d = (c["heads"] + 2 * c["kv"]) * 64, c["heads"] * 64
        ctx.kernel_qk_norm_rope(lib.DTYPES[c["dtype"]], p["qkv"], total, c["tokens"], c["heads"], c["kv"], norm,
                                p["qw"], p["qb"] if bias else 0, p["kw"], p["kb"] if bias else 0, EPS, rope, BASE,
                                p["pos"], p["q"], d, 0 if c["cache"] else p["kout"], 0 if c["cache"] else c["kv"] * 64,
                                _cache(lib, s) if c["cache"] else None, p["slots"] if c["cache"] else 0)
        return {name: s[name] for name in (("q", "k", "v") if c["cache"] else ("q", "kout"))}
    cache = _cache(lib, s)
    if kind == "bounds":
        ctx.kernel_page_bounds(cache, c["n"], p["table"], s["width"], p["lens"], p["add"],
                               {"one": 1, "view": VIEW, "all": c["max_len"]}[c["add"]], p["bounds"])
        return {"bounds": s["bounds"]}
    d = c["heads"] * 64
    if kind == "paged":
        ctx.kernel_paged_attention(cache, p["q"], d, c["n"], c["heads"], p["table"], s["width"], p["lens"], c["max_len"], 0.125,
                                   p["out"], d, p["workspace"], s["bytes"])
        return {"out": s["out"]}
    ctx.kernel_sparse_attention(cache, p["bounds"], p["q"], d, c["n"], c["heads"], p["table"], s["width"], p["lens"],
                                c["max_len"], c["topk"], 0.125, p["out"], d, p["selected"], p["workspace"], s["bytes"])
    return {"out": s["out"], "selected": s["selected"]}


def _tables_plain(s):
    ps, cap = s["c"]["ps"], s["cap"]
    past, add, used = s["past"].long(), s["add"].long(), s["used"].long()
    lens = past + add
    have, last = (past + ps - 1) // ps, (lens + ps - 1) // ps
    first = torch.cumsum(last - have, 0) - (last - have)
    ends = torch.cumsum(add, 0)
    starts = torch.cat([ends.new_zeros(1), ends])
    j = torch.arange(s["width"], device=DEV)[None, :]
    fresh = (j >= have[:, None]) & (j < last[:, None])
    at = (used + first[:, None] + j - have[:, None]).clamp(0, s["pool"].numel() - 1)
    table = torch.where(fresh, s["pool"][at], s["table"])
    t = torch.arange(cap, device=DEV)
    r = torch.searchsorted(ends, t, right=True)
    pos = past[r] + t - starts[r]
    slots = table[r, pos // ps].long() * ps + pos % ps
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return {"table": table, "lens": i32(lens), "starts": i32(starts), "slots": i32(slots), "positions": i32(pos),
            "used_out": i32(used + (last - have).sum()), "status": torch.zeros(1, dtype=torch.int32, device=DEV)}


def _angles(c, pos):
    """[tokens, 64] angles in 64 bits: channel c turns with its partner half a span away."""
    if c["rope"] == "line":
        f = BASE ** (-torch.arange(32, device=DEV, dtype=torch.float64) / 32)
        a = pos.double()[:, None] * f
        return torch.cat([a, a], 1)
    f = BASE ** (-torch.arange(16, device=DEV, dtype=torch.float64) / 16)
    a, b = pos[:, :1].double() * f, pos[:, 1:].double() * f
    return torch.cat([a, a, b, b], 1)


def _partner(x, rope):
    """-x[c + span / 2] below the middle of its span, x[c - span / 2] above."""
    if rope == "line":
        return torch.cat([-x[..., 32:], x[..., :32]], -1)
    return torch.cat([-x[..., 16:32], x[..., :16], -x[..., 48:], x[..., 32:48]], -1)


def _norm_rope(x, w, b, c, cos, sin):
    if c["norm"] == "layer":
        m = x.mean(-1, keepdim=True)
        d = x - m
        x = d / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS) * w + b
    elif c["norm"] == "rms":
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    return x if c["rope"] == "none" else x * cos + _partner(x, c["rope"]) * sin


def _rope_plain(s):
    c = s["c"]
    T, heads, kv, ps, td = c["tokens"], c["heads"], c["kv"], c["ps"], TORCH[c["dtype"]]
    x = s["qkv"].float().view(T, heads + 2 * kv, 64)
    cos = sin = None
    if c["rope"] != "none":
        a = _angles(c, s["pos"])
        cos, sin = torch.cos(a).float()[:, None, :], torch.sin(a).float()[:, None, :]
    q = _norm_rope(x[:, :heads], s["qw"], s["qb"], c, cos, sin).reshape(T, heads * 64).to(td)
    k = _norm_rope(x[:, heads:heads + kv], s["kw"], s["kb"], c, cos, sin).to(td)
    if not c["cache"]:
        return {"q": q, "kout": k.reshape(T, kv * 64)}
    slot = s["slots"].long()
    s["k"][slot // ps, :, slot % ps] = k
    s["v"][slot // ps, :, slot % ps] = x[:, heads + kv:].to(td)
    return {"q": q, "k": s["k"], "v": s["v"]}


def _bounds_plain(s):
    ps = s["c"]["ps"]
    lens, add = s["lens"].long()[:, None], s["add"].long()[:, None]
    j = torch.arange(s["width"], device=DEV)[None, :]
    i, j = ((j * ps < lens) & ((j + 1) * ps > lens - add) & (add > 0)).nonzero(as_tuple=True)
    page = s["table"][i, j].long()
    there = (j[:, None] * ps + torch.arange(ps, device=DEV) < lens[i])[:, None, :, None]
    k = s["k"][page].float()
    lo = torch.where(there, k, math.inf).amin(2)
    hi = torch.where(there, k, -math.inf).amax(2)
    s["bounds"][page] = torch.stack([lo, hi], 2).to(s["k"].dtype)
    return {"bounds": s["bounds"]}


def _attend(q, k, v, there):
    """q [.., G, 64], k and v [.., L, 64], there [.., 1, L]: zeros where no key is there."""
    x = torch.matmul(q, k.transpose(-1, -2)) * 0.125
    x = torch.where(there, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(m), 0.0, m))
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return torch.where(there.any(-1, keepdim=True), out, 0.0)


def _paged_plain(s):
    c = s["c"]
    n, heads, kv, ps = c["n"], c["heads"], c["kv"], c["ps"]
    page = s["table"].long().clamp(min=0)
    L = s["width"] * ps
    k = s["k"][page].permute(0, 2, 1, 3, 4).reshape(n, kv, L, 64).float()
    v = s["v"][page].permute(0, 2, 1, 3, 4).reshape(n, kv, L, 64).float()
    there = (torch.arange(L, device=DEV)[None, :] < s["lens"][:, None])[:, None, None, :]
    out = _attend(s["q"].float().view(n, kv, heads // kv, 64), k, v, there)
    return {"out": out.reshape(n, heads * 64).to(s["q"].dtype)}


def _sparse_plain(s):
    c = s["c"]
    n, heads, kv, ps, topk, width = c["n"], c["heads"], c["kv"], c["ps"], c["topk"], s["width"]
    page = s["table"].long().clamp(min=0)
    q = s["q"].view(n, kv, heads // kv, 64)
    up, down = q.double().clamp(min=0).sum(2), q.double().clamp(max=0).sum(2)
    b = s["bounds"][page].permute(0, 2, 1, 3, 4).double()      # [n, kv, width, 2, 64]
    score = (b[..., 0, :] * down[:, :, None] + b[..., 1, :] * up[:, :, None]).sum(-1)
    j = torch.arange(width, device=DEV)
    held = (s["lens"].long() + ps - 1) // ps
    score = torch.where(j == held[:, None, None] - 1, math.inf, score)
    score = torch.where(j < held[:, None, None], score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :topk]
    order = torch.where(order < held[:, None, None], order, width)          # behind every page
    if topk > width:
        order = torch.cat([order, order.new_full((n, kv, topk - width), width)], -1)
    sel = torch.sort(order, dim=-1).values
    real = sel < width
    at = torch.gather(page[:, None, :].expand(n, kv, width), 2, sel.clamp(max=width - 1))
    h = torch.arange(kv, device=DEV)[None, :, None]
    k = s["k"][at, h].reshape(n, kv, topk * ps, 64).float()
    v = s["v"][at, h].reshape(n, kv, topk * ps, 64).float()
    there = real[..., None] & (sel[..., None] * ps + torch.arange(ps, device=DEV) < s["lens"].long()[:, None, None, None])
    out = _attend(q.float(), k, v, there.reshape(n, kv, 1, topk * ps))
    return {"out": out.reshape(n, heads * 64).to(s["q"].dtype), "selected": torch.where(real, sel, -1).to(torch.int32)}


def run(s):
    if own:
        return _run_own(s)
    return {"tables": _tables_plain, "rope": _rope_plain, "bounds": _bounds_plain, "paged": _paged_plain,
            "sparse": _sparse_plain}[s["c"]["kind"]](s)


# --- bytes and operations ---------------------------------------------------------------------------

def work(case):
    c, kind = case, case["kind"]
    es = 4 if c.get("dtype") == "f32" else 2
    if kind == "rope":
        rows = c["tokens"] * (c["heads"] + 2 * c["kv"]) * 64
        if not c["cache"]:   # values stay where they are
            rows -= c["tokens"] * c["kv"] * 64
        by = 2.0 * rows * es + c["tokens"] * (4 * c["cache"] + {"none": 0, "line": 4, "grid": 8}[c["rope"]])
        return {"bytes": by, "flops": 12.0 * c["tokens"] * (c["heads"] + c["kv"]) * 64}
    past, add = _lengths(c)
    ps, lens = c["ps"], [p + a for p, a in zip(past, add)]
    if kind == "tables":
        fresh = sum(-(-v // ps) - -(-p // ps) for v, p in zip(lens, past))
        return {"bytes": 4.0 * (4 * c["n"] + 2 * fresh + 2 * sum(add)), "flops": 4.0 * sum(add)}
    row = c["kv"] * 64 * es
    if kind == "bounds":
        pages = [(p // ps, -(-v // ps)) for p, v, a in zip(past, lens, add) if a]
        rows = sum(min(v, b * ps) - f * ps for (f, b), v in zip(pages, [v for v, a in zip(lens, add) if a]))
        return {"bytes": float(row) * (rows + 2 * sum(b - f for f, b in pages)) + 12.0 * c["n"], "flops": 2.0 * rows * c["kv"] * 64}
    io = 2.0 * c["n"] * c["heads"] * 64 * es + 4.0 * c["n"]
    if kind == "paged":
        return {"bytes": 2.0 * row * sum(lens) + 4.0 * sum(-(-v // ps) for v in lens) + io,
                "flops": 4.0 * c["heads"] * 64 * sum(lens)}
    held = [-(-v // ps) for v in lens]
    keys = sum(min(v, c["topk"] * ps - (-v) % ps) for v in lens if v)
    return {"bytes": 2.0 * row * (sum(held) + keys) + 4.0 * sum(held) + 4.0 * c["n"] * c["kv"] * c["topk"] + io,
            "flops": 4.0 * c["heads"] * 64 * keys + 4.0 * c["kv"] * 64 * sum(held)}


# --- the same in 64 bits --------------------------------------------------------------------------

def _exact_rope(s):
    c = s["c"]
    T, heads, kv, ps = c["tokens"], c["heads"], c["kv"], c["ps"]
    x = s["qkv"].double().view(T, heads + 2 * kv, 64)

    def one(y, w, b):
        if c["norm"] == "layer":
            y = (y - y.mean(-1, keepdim=True)) / (y.var(-1, unbiased=False, keepdim=True) + EPS).sqrt() * w.double() + b.double()
        elif c["norm"] == "rms":
            y = y * (y.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
        if c["rope"] == "none":
            return y
        # as complex numbers: pair (c, c + h) of each span turns by one angle
        spans, h = (1, 32) if c["rope"] == "line" else (2, 16)
        p = s["pos"].double().view(T, spans)
        a = p[:, :, None] * torch.exp(-math.log(BASE) * torch.arange(h, device=DEV, dtype=torch.float64) / h)
        z = y.reshape(T, -1, spans, 2, h)
        z = torch.complex(z[:, :, :, 0], z[:, :, :, 1]) * torch.polar(torch.ones_like(a), a)[:, None]
        return torch.stack([z.real, z.imag], 3).reshape(T, -1, 64)

    q = one(x[:, :heads], s["qw"], s["qb"]).reshape(T, heads * 64)
    k = one(x[:, heads:heads + kv], s["kw"], s["kb"])
    if not c["cache"]:
        return {"q": q, "kout": k.reshape(T, kv * 64)}
    pools = []
    for rows in (k, x[:, heads + kv:]):
        flat = torch.zeros(s["k"].shape[0] * ps, kv, 64, dtype=torch.float64, device=DEV)
        flat[s["slots"].long()] = rows
        pools.append(flat.view(-1, ps, kv, 64).transpose(1, 2).contiguous())
    return {"q": q, "k": pools[0], "v": pools[1]}


def _keys(s, i, positions):
    """Keys and values of sequence i at `positions`, [kv, L, 64] in 64 bits."""
    ps = s["c"]["ps"]
    page = s["table"][i].long()[positions // ps]
    return s["k"][page, :, positions % ps].double().transpose(0, 1), s["v"][page, :, positions % ps].double().transpose(0, 1)


def _softmax_sum(q, k, v):
    """[G, 64] for q [G, 64], k and v [L, 64]."""
    return torch.softmax((q[:, None, :] * k[None]).sum(-1) / 8, -1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    c, kind = case, case["kind"]
    if kind == "rope":
        return _exact_rope(s)
    past, add = _lengths(c)
    lens, ps = [p + a for p, a in zip(past, add)], c["ps"]
    if kind == "tables":
        table, pool, at = s["table"].tolist(), s["pool"].tolist(), int(s["used"])
        slots, positions, starts = [], [], [0]
        for row, p, v in zip(table, past, lens):
            for j in range(-(-p // ps), -(-v // ps)):
                row[j] = pool[at]
                at += 1
            slots += [row[t // ps] * ps + t % ps for t in range(p, v)]
            positions += range(p, v)
            starts.append(len(slots))
        return {"table": _int(table), "lens": _int(lens), "starts": _int(starts), "slots": _int(slots),
                "positions": _int(positions), "used_out": _int([at]), "status": _int([0])}
    if kind == "bounds":
        want = torch.zeros(s["bounds"].shape, dtype=torch.float64, device=DEV)
        for i, (p, v) in enumerate(zip(past, lens)):
            first, last = p // ps, -(-v // ps) if v > p else 0
            full = v // ps
            if last > first:
                k = s["k"][s["table"][i, first:last].long()].double()
                both = torch.stack([k.min(2).values, k.max(2).values], 2)
                if full < last:
                    part = k[full - first, :, :v - full * ps]
                    both[full - first] = torch.stack([part.min(1).values, part.max(1).values], 1)
                want[s["table"][i, first:last].long()] = both
        return {"bounds": want}
    n, heads, kv = c["n"], c["heads"], c["kv"]
    q = s["q"].double().view(n, kv, heads // kv, 64)
    out = torch.zeros(n, kv, heads // kv, 64, dtype=torch.float64, device=DEV)
    chosen = torch.full((n, kv, c.get("topk", 1)), -1, dtype=torch.int32, device=DEV)
    for i, v in enumerate(lens):
        if v == 0:
            continue
        if kind == "paged":
            keys, values = _keys(s, i, torch.arange(v, device=DEV))
            for h in range(kv):
                out[i, h] = _softmax_sum(q[i, h], keys[h], values[h])
            continue
        held = -(-v // ps)
        lo, hi = s["bounds"][s["table"][i, :held].long()].double().unbind(2)
        for h in range(kv):
            # the most that any key between the bounds can give, summed over the group's heads
            score = torch.maximum(q[i, h][:, None, :] * lo[None, :, h], q[i, h][:, None, :] * hi[None, :, h]).sum((0, 2))
            score[held - 1] = math.inf
            sel = torch.sort(score, descending=True, stable=True).indices[:c["topk"]].sort().values
            chosen[i, h, :sel.numel()] = sel.to(torch.int32)
            at = (sel[:, None] * ps + torch.arange(ps, device=DEV)).flatten()
            at = at[at < v]
            page, row = s["table"][i].long()[at // ps], at % ps
            out[i, h] = _softmax_sum(q[i, h], s["k"][page, h, row].double(), s["v"][page, h, row].double())
    out = out.reshape(n, heads * 64)
    return {"out": out} if kind == "paged" else {"out": out, "selected": chosen}
