"""Performance cases of the paged cache's pages and of attention over a prefix that many tokens share.

A scene's views stay in the cache; questions about it fork its row of pages, go on by themselves and end,
the pages they leave are given back, and a pool with holes is compacted. The forks of a scene, or all tokens of a
view, attend to its positions at once. One pass is one operator call on device buffers, in the plain form
(elementary torch operations, in 32 bits) or, with `own`, through the library's kernel entry points. `exact` restates
every operator from its definition, row by row, in 64 bits.

Layout: key and value pools [pages, kv_heads, page_size, 64]; position p of row i of a table lies in row p % page_size
of page table[i, p // page_size]. The free pages are pool[used:]. Inputs of a call stay as they are where it has outputs
of their own, so that a pass can be made again.
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
_held = {}           # the library context that a program keeps


# --- the cases ----------------------------------------------------------------------------------

def listed():
    return [
        # 28 of 64 rows become forks of four scenes between two steps of a serving loop. Latency.
        {"name": "fork_step", "kind": "fork", "n": 64, "scenes": 4, "max_len": 8 * VIEW, "ps": 16},
        # A thousand questions about eight scenes of up to 24 views: over half a million table entries.
        {"name": "fork_scenes", "kind": "fork", "n": 1024, "scenes": 8, "max_len": SCENE, "ps": 16},
        # One in eight of 64 rows ends, some go back to an earlier length; the others share its pages or not. Latency.
        {"name": "free_step", "kind": "free", "n": 64, "scenes": 4, "max_len": 8 * VIEW, "max_own": 64, "ps": 16},
        # A thousand rows of eight scenes with a view each of their own.
        {"name": "free_scenes", "kind": "free", "n": 1024, "scenes": 8, "max_len": SCENE, "max_own": VIEW, "ps": 16},
        # A small pool, half of it free in no order. Latency.
        {"name": "compact_step", "kind": "compact", "n": 16, "scenes": 4, "max_len": 4 * VIEW, "max_own": 64, "ps": 32},
        # 512 rows with forks, a hundred thousand pages and as many holes.
        {"name": "compact_scenes", "kind": "compact", "n": 512, "scenes": 128, "max_len": SCENE, "max_own": 2 * VIEW, "ps": 8},
        # The begun pages of 32 forks in four layers of 12 heads, after a fork. Latency.
        {"name": "copy_tails_bf16", "kind": "copy", "pairs": 32, "layers": 4, "rows": "tails", "kv": 12, "ps": 16, "dtype": "bf16"},
        # 1000 pages of 64 KB that a compaction moves, in two layers, with their bounds.
        {"name": "copy_moves_f16", "kind": "copy", "pairs": 1000, "layers": 2, "rows": "all", "kv": 8, "ps": 64, "dtype": "f16"},
        # Six questions about two thumbnails' scenes in fp32. Latency.
        {"name": "prefix_small_f32", "kind": "prefix", "mode": "forks", "n": 6, "groups": 2, "max_shared": 188, "max_own": 20,
         "heads": 6, "kv": 6, "ps": 8, "dtype": "f32"},
        # 64 questions about one scene of 24 views, each with up to a view of its own.
        {"name": "prefix_forks_bf16", "kind": "prefix", "mode": "forks", "n": 64, "groups": 1, "max_shared": SCENE, "max_own": VIEW,
         "heads": 12, "kv": 12, "ps": 16, "dtype": "bf16"},
        # 48 questions about four scenes of different lengths, four query heads to a key head.
        {"name": "prefix_groups_f16", "kind": "prefix", "mode": "forks", "n": 48, "groups": 4, "max_shared": SCENE,
         "max_own": 2 * VIEW, "heads": 32, "kv": 8, "ps": 64, "dtype": "f16"},
        # All tokens of a view against a scene of 24 views: the matrix cores' case.
        {"name": "prefix_view_bf16", "kind": "prefix", "mode": "view", "n": VIEW, "groups": 1, "max_shared": SCENE, "max_own": 0,
         "heads": 12, "kv": 12, "ps": 16, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo))))))))


MOST_SCORES = VIEW * 12 * SCENE   # of the largest listed case


def draw(rng):
    kind = rng.choice(["fork", "free", "compact", "copy", "prefix", "prefix", "prefix", "prefix"])
    ps = rng.choice([8, 16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("fork", "free", "compact"):
        n = _log_int(rng, 2, 1024 if kind != "compact" else 512)
        c = {"kind": kind, "n": n, "scenes": _log_int(rng, 1, max(1, n // 4)), "max_len": _log_int(rng, 1, SCENE), "ps": ps}
        if kind != "fork":
            c["max_own"] = _log_int(rng, 1, VIEW)
        return c
    heads, kv = rng.choice([(6, 6), (12, 12), (16, 16), (24, 8), (20, 4), (8, 1), (32, 2), (32, 8)])
    if kind == "copy":
        page = kv * ps * 64 * (4 if dtype == "f32" else 2)
        layers = rng.choice([1, 2, 4, 8])
        return {"kind": kind, "pairs": _log_int(rng, 1, max(1, min(4000, 250000000 // (2 * page * layers)))), "layers": layers,
                "rows": rng.choice(["tails", "all"]), "kv": kv, "ps": ps, "dtype": dtype}
    mode = rng.choice(["forks", "forks", "view", "chunk"])
    shared = _log_int(rng, 1, SCENE)
    most = MOST_SCORES // (2 if dtype == "f32" else 1) // heads
    if mode == "forks":
        max_own = _log_int(rng, 1, 2 * VIEW)
        n = _log_int(rng, 1, min(96, max(1, most // (shared + max_own) // 2)))
        groups = _log_int(rng, 1, min(n, 8))
    else:
        max_own = 0
        n = _log_int(rng, 1, min(2 * VIEW, max(1, most // max(shared, VIEW))))
        groups = rng.choice([1, 1, 2, 3])
        if mode == "chunk":
            shared = max(shared, n)
    return {"kind": kind, "mode": mode, "n": n, "groups": groups, "max_shared": shared, "max_own": max_own, "heads": heads, "kv": kv,
            "ps": ps, "dtype": dtype}


# --- sizes, which the case alone decides ----------------------------------------------------------

def _spread(n, most):
    """n lengths from 1 to `most`, spread over their logarithm in no order, the longest among them; from
    eight on one of them is 0."""
    out = [int(round(math.exp(((0.5 + 0.6180339887 * i) % 1.0) * math.log(max(most, 1))))) for i in range(n)]
    if n:
        out[0] = most
    if n >= 8:
        out[3] = 0
    return [min(most, max(0, v)) for v in out]


def _even(i, most):
    """A length from 0 to `most`, spread evenly over i in no order."""
    return int(((0.25 + 0.7548776662 * i) % 1.0) * (most + 1))


def _rows(c):
    """Of every row of the table: (parent or -1, positions it has in common with it, its length). Rows up to
    c["scenes"] are scenes, the others forks of them; one in eight is empty."""
    out = [(-1, 0, v) for v in _spread(c["scenes"], c["max_len"])]
    for i in range(c["scenes"], c["n"]):
        if i % 8 == 5:
            out.append((-1, 0, 0))
            continue
        parent = (7 * i + i // 8) % c["scenes"]
        whole = out[parent][2]
        keep = whole if i % 3 else _even(i, whole)
        out.append((parent, keep, keep + (1 + _even(3 * i, c["max_own"] - 1) if "max_own" in c else 0)))
    return out


def _kept(c):
    """The new length of every row of a "free" case: some end, some go back, the others stay."""
    return [0 if i % 8 == 1 or i % 8 == 4 and c["n"] > 64 else _even(i, v) if i % 16 == 7 else v for i, (_, _, v) in enumerate(_rows(c))]


def _entries(c):
    """Per row: places of the table that are its parent's, and all of its places."""
    ps = c["ps"]
    return [(keep // ps if parent >= 0 else 0, -(-v // ps)) for parent, keep, v in _rows(c)]


def _members(c):
    """The first token of each group and their number: later groups are larger."""
    return [int(round(c["n"] * (g / c["groups"]) ** 1.3)) for g in range(c["groups"] + 1)]


def _lengths(c):
    """(shared positions of every group, length of every token)."""
    at = _members(c)
    shared = _spread(c["groups"], c["max_shared"])
    lens = []
    for g in range(c["groups"]):
        m = at[g + 1] - at[g]
        if c["mode"] == "chunk":
            shared[g] = max(shared[g], m)
        for t in range(m):
            lens.append(shared[g] - m + 1 + t if c["mode"] == "chunk" else shared[g] + (_even(at[g] + t, c["max_own"])))
    return shared, lens


# --- what a program has in hand -----------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * scale


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pool(g, pages, c):
    """Keys or values: neighbouring tokens are alike (a page's tokens share a part)."""
    kv, ps, td = c["kv"], c["ps"], TORCH[c["dtype"]]
    out = torch.empty(pages, kv, ps, 64, dtype=td, device=DEV)
    step = max(1, (1 << 26) // (kv * ps * 64))
    for a in range(0, pages, step):
        m = min(step, pages - a)
        out[a:a + m] = (_randn(g, m, kv, ps, 64, scale=0.8) + _randn(g, m, kv, 1, 64, scale=0.6)).to(td)
    return out


def _prepare_pages(c, seed, s):
    """A table of scenes and, but for "fork", their forks on pages in random order, and what is free."""
    g, kind, ps, n = _gen(seed), c["kind"], c["ps"], c["n"]
    rows, places = _rows(c), _entries(c)
    width = max(1, max(have for _, have in places)) + 1
    there = [(0 if parent >= 0 else have) if kind == "fork" else have for (parent, _, _), (_, have) in zip(rows, places)]
    fresh = [0 if kind == "fork" and parent >= 0 else have - first for (parent, _, _), (first, have) in zip(rows, places)]
    total = sum(fresh)
    more = {"fork": n + 7, "free": total // 16 + 5, "compact": total + 9}[kind]
    pages = total + more
    ids = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    j = torch.arange(width, device=DEV)[None, :]
    first = _int([a if t else 0 for t, (a, _) in zip(there, places)])[:, None]
    begin = _int([sum(fresh[:i]) for i in range(n)] if n < 64 else torch.tensor([0] + fresh[:-1]).cumsum(0).tolist())[:, None]
    own_page = ids[(begin + j - first).clamp(0, max(total - 1, 0))]
    parent = _int([p for p, _, _ in rows]).long().clamp(min=0)
    table = torch.where(j < first, own_page[parent], own_page)
    s["table"] = torch.where(j < _int(there)[:, None], table, -1).to(torch.int32).contiguous()
    s["pages"], s["width"] = pages, width
    s["pool"], s["used"] = ids, _int([total])
    s["parents"] = _int([p for p, _, _ in rows])
    s["lens"] = _int([0 if kind == "fork" and p >= 0 else v for p, _, v in rows])
    s["keep"] = _int([k for _, k, _ in rows] if kind == "fork" else _kept(c) if kind == "free" else [0] * n)
    s["cap"] = pages // 2 + 1
    for name, m in (("lens_out", n), ("used_out", 1), ("status", 1), ("count", 1)):
        s[name] = torch.empty(m, dtype=torch.int32, device=DEV)
    m = n if kind == "fork" else s["cap"] if kind == "compact" else 1
    for name in ("src", "dst", "rows"):
        s[name] = torch.empty(m, dtype=torch.int32, device=DEV)
    s["table_out"], s["pool_out"] = torch.empty_like(s["table"]), s["pool"].clone()


def _prepare_copy(c, seed, s):
    g, pairs, ps = _gen(seed), c["pairs"], c["ps"]
    pages = 2 * pairs + 3
    ids = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    s["src"], s["dst"] = ids[:pairs].contiguous(), ids[pairs:2 * pairs].contiguous()
    s["count"] = _int([pairs])
    if c["rows"] == "tails":
        s["rows"] = _int([1 + _even(i, ps - 2) for i in range(pairs)])
    for layer in range(c["layers"]):
        s["k%d" % layer], s["v%d" % layer] = _pool(g, pages, c), _pool(g, pages, c)
        if c["rows"] == "all":
            k = s["k%d" % layer]
            s["b%d" % layer] = torch.stack([k.amin(2), k.amax(2)], 2).contiguous()


def _prepare_prefix(c, seed, s):
    g, ps, n, groups, at = _gen(seed), c["ps"], c["n"], c["groups"], _members(c)
    shared, lens = _lengths(c)
    forks = c["mode"] == "forks"
    common = [v // ps for v in shared]                       # full pages that the forks have in common
    held = [-(-v // ps) for v in shared]
    s["prefix_width"] = max(1, max(held))
    group_of = [k for k in range(groups) for _ in range(at[k + 1] - at[k])]
    mine = [max(0, -(-v // ps) - common[k]) if v > shared[k] else 0 for v, k in zip(lens, group_of)] if forks else []
    total = sum(held) + sum(mine)
    s["pages"] = total + 3
    ids = torch.randperm(s["pages"], device=DEV, generator=g).to(torch.int32)
    j = torch.arange(s["prefix_width"], device=DEV)[None, :]
    begin = _int([sum(held[:k]) for k in range(groups)])[:, None]
    s["prefix"] = torch.where(j < _int(held)[:, None], ids[(begin + j).clamp(max=s["pages"] - 1)], -1).contiguous()
    s["shared"], s["starts"] = _int(shared), _int(at)
    s["width"] = 0
    if forks:   # a fork's row: the common full pages, then pages of its own
        s["width"] = width = max(1, max(-(-v // ps) for v in lens))
        j = torch.arange(width, device=DEV)[None, :]
        k = _int(group_of).long()
        first = _int(common)[k][:, None]
        begin = _int([sum(held) + sum(mine[:i]) for i in range(n)])[:, None]
        old = s["prefix"][k][:, :width]
        old = torch.nn.functional.pad(old, (0, width - old.shape[1]), value=-1)
        row = torch.where(j < first, old, ids[(begin + j - first).clamp(0, s["pages"] - 1)])
        s["table"] = torch.where(j < _int([-(-v // ps) for v in lens])[:, None], row, -1).to(torch.int32).contiguous()
    if c["mode"] != "view":
        s["lens"] = _int(lens)
    s["k"], s["v"] = _pool(g, s["pages"], c), _pool(g, s["pages"], c)
    if forks and any(v % ps for v in shared):   # the begun page of the prefix was copied into each fork's own
        i = [x for x in range(n) if mine[x] and shared[group_of[x]] % ps]
        if i:
            a = torch.tensor([group_of[x] for x in i], device=DEV)
            f = _int(common).long()[a]
            src, dst = s["prefix"][a, f].long(), s["table"][torch.tensor(i, device=DEV), f].long()
            there = (torch.arange(ps, device=DEV)[None, :] < (_int(shared).long()[a] % ps)[:, None])[:, None, :, None]
            for pool in (s["k"], s["v"]):
                pool[dst] = torch.where(there, pool[src], pool[dst])
    s["q"] = (_randn(g, n, c["heads"] * 64) * 1.2).to(s["k"].dtype)
    s["out"] = torch.empty_like(s["q"])


def prepare(case, seed):
    s = {"c": case}
    {"copy": _prepare_copy, "prefix": _prepare_prefix}.get(case["kind"], _prepare_pages)(case, seed, s)
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


def _workspace(lib, s):
    """What a program keeps with its cache: its description and a workspace for the calls on it."""
    if "workspace" not in s:
        c, p, kind = s["c"], s["ptr"], s["c"]["kind"]
        size = 0
        if kind in ("free", "compact"):
            size = lib.pages_workspace(s["pages"])
        elif kind == "copy":
            s["caches"] = lib.layers(lib.KvCache(lib.DTYPES[c["dtype"]], p["k%d" % i], p["v%d" % i], s["k0"].shape[0], c["ps"], c["kv"])
                                     for i in range(c["layers"]))
            s["bounds"] = lib.pointers(p["b%d" % i] for i in range(c["layers"])) if c["rows"] == "all" else None
        elif kind == "prefix":
            s["cache"] = lib.KvCache(lib.DTYPES[c["dtype"]], p["k"], p["v"], s["pages"], c["ps"], c["kv"])
            size = lib.prefix_attention_workspace(s["cache"], c["n"], c["heads"], c["groups"], c["max_shared"], c["max_own"])
        s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
        p["workspace"], s["bytes"] = s["workspace"].data_ptr(), size
    return s["bytes"]


def _run_own(s):
    lib, ctx = _library()
    size = _workspace(lib, s)
    c, p, kind = s["c"], s["ptr"], s["c"]["kind"]
    if kind == "fork":
        ctx.kernel_fork_pages(c["n"], p["parents"], p["keep"], p["lens"], c["ps"], s["pages"], p["pool"], s["pool"].numel(), p["used"],
                              p["table"], s["width"], p["lens_out"], p["src"], p["dst"], p["rows"], p["used_out"], p["status"])
        return {name: s[name] for name in ("table", "lens_out", "src", "dst", "rows", "used_out", "status")}
    if kind == "free":
        ctx.kernel_free_pages(c["n"], p["keep"], p["lens"], c["ps"], s["pages"], p["pool"], s["pool"].numel(), p["used"], p["table"],
                              s["width"], p["lens_out"], p["used_out"], p["status"], p["workspace"], size)
        return {name: s[name] for name in ("lens_out", "pool", "used_out", "status")}
    if kind == "compact":
        ctx.kernel_compact_pages(c["n"], p["lens"], c["ps"], s["pages"], p["pool"], s["pool"].numel(), p["used"], p["table"], s["width"],
                                 p["table_out"], p["pool_out"], p["src"], p["dst"], s["cap"], p["count"], p["status"], p["workspace"], size)
        return {name: s[name] for name in ("table_out", "pool_out", "src", "dst", "count", "status")}
    if kind == "copy":
        ctx.kernel_copy_pages(s["caches"], s["bounds"], c["pairs"], p["src"], p["dst"], p.get("rows", 0), p["count"])
        return {name: s[name] for name in _pools(c)}
    d = c["heads"] * 64
    ctx.kernel_prefix_attention(s["cache"], p["q"], d, c["n"], c["heads"], p["starts"], c["groups"], p["prefix"], s["prefix_width"],
                                p["shared"], c["max_shared"], p.get("table", 0), s["width"], p.get("lens", 0), c["max_own"], 0.125,
                                p["out"], d, p["workspace"], size)
    return {"out": s["out"]}


def _pools(c):
    return [x + str(i) for x in ("kvb" if c["rows"] == "all" else "kv") for i in range(c["layers"])]


def _i32(x):
    return x.to(torch.int32)


def _fork_plain(s):
    ps, lens, keep, parent = s["c"]["ps"], s["lens"].long(), s["keep"].long(), s["parents"].long()
    fork, at = parent >= 0, parent.clamp(min=0)
    full, tail = keep // ps, keep % ps
    old = s["table"][at]
    page = torch.gather(old, 1, full.clamp(max=s["width"] - 1)[:, None])[:, 0].long()
    takes = fork & (tail > 0) & (page >= 0) & (page < s["pages"])
    rank = torch.cumsum(takes, 0) - takes.long()
    new = s["pool"][(s["used"].long() + rank).clamp(0, s["pool"].numel() - 1)].long()
    j = torch.arange(s["width"], device=DEV)[None, :]
    table = torch.where(fork[:, None] & (j < full[:, None]), old, s["table"])
    table = torch.where((fork & (tail > 0))[:, None] & (j == full[:, None]), torch.where(takes, new, page)[:, None], table.long())
    return {"table": _i32(table), "lens_out": _i32(torch.where(fork, keep, lens)), "src": _i32(torch.where(takes, page, -1)),
            "dst": _i32(torch.where(takes, new, -1)), "rows": _i32(torch.where(takes, tail, 0)), "used_out": _i32(s["used"] + takes.sum()),
            "status": torch.zeros(1, dtype=torch.int32, device=DEV)}


def _mark(pages, table, there):
    """Flags of the pages that the table names where `there` says so."""
    flags = torch.zeros(pages + 1, dtype=torch.bool, device=DEV)
    at = torch.where(there & (table >= 0) & (table < pages), table.long(), pages)
    flags[at.reshape(-1)] = True
    return flags[:pages]


def _free_plain(s):
    ps, pages, size, used = s["c"]["ps"], s["pages"], s["pool"].numel(), s["used"].long()
    j = torch.arange(s["width"], device=DEV)[None, :]
    stays, was = ((s["keep"].long() + ps - 1) // ps)[:, None], ((s["lens"].long() + ps - 1) // ps)[:, None]
    held = _mark(pages, s["table"], j < stays) | _mark(pages, s["pool"], torch.arange(size, device=DEV) >= used)
    gone = _mark(pages, s["table"], (j >= stays) & (j < was)) & ~held
    rank, count = torch.cumsum(gone, 0) - 1, gone.sum()
    pool = torch.cat([s["pool"], s["pool"][:1]])
    pool[torch.where(gone, used - count + rank, size)] = torch.arange(pages, device=DEV, dtype=torch.int32)
    return {"lens_out": s["keep"].clone(), "pool": pool[:size], "used_out": _i32(used - count),
            "status": torch.zeros(1, dtype=torch.int32, device=DEV)}


def _compact_plain(s):
    ps, pages, size, cap, used = s["c"]["ps"], s["pages"], s["pool"].numel(), s["cap"], s["used"].long()
    there = torch.arange(s["width"], device=DEV)[None, :] < ((s["lens"].long() + ps - 1) // ps)[:, None]
    live, free = _mark(pages, s["table"], there), _mark(pages, s["pool"], torch.arange(size, device=DEV) >= used)
    both = live | free
    rank, count = torch.cumsum(both, 0) - both.long(), live.sum()
    moves, hole, ids = live & (rank >= count), free & (rank < count), torch.arange(pages, device=DEV, dtype=torch.int32)
    src = torch.full((cap + 1,), -1, dtype=torch.int32, device=DEV)
    dst = src.clone()
    at = torch.cumsum(moves, 0) - 1
    src[torch.where(moves, at, cap)] = ids
    dst[torch.where(hole, torch.cumsum(hole, 0) - 1, cap)] = ids
    now = torch.where(moves, dst[at.clamp(0, cap)], ids)
    ok = there & (s["table"] >= 0) & (s["table"] < pages)
    pool = torch.cat([s["pool"], s["pool"][:1]])
    pool[torch.where(both & (rank >= count), used + rank - count, size)] = ids
    return {"table_out": torch.where(ok, now[s["table"].long().clamp(0, pages - 1)], s["table"]), "pool_out": pool[:size], "src": src[:cap],
            "dst": dst[:cap], "count": _i32(moves.sum().reshape(1)), "status": torch.zeros(1, dtype=torch.int32, device=DEV)}


def _copy_plain(s):
    c, src, dst = s["c"], s["src"].long(), s["dst"].long()
    there = None
    if c["rows"] == "tails":
        there = (torch.arange(c["ps"], device=DEV)[None, :] < s["rows"][:, None])[:, None, :, None]
    for name in _pools(c):
        s[name][dst] = s[name][src] if there is None else torch.where(there, s[name][src], s[name][dst])
    return {name: s[name] for name in _pools(c)}


def _part(q, k, v, there):
    """The largest score, the sum of weights and the weighted values of q [.., R, 64] over k and v [.., L, 64] where `there`."""
    x = torch.where(there, torch.matmul(q, k.transpose(-1, -2)) * 0.125, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(m), 0.0, m))
    return m, p.sum(-1, keepdim=True), torch.matmul(p, v)


def _prefix_plain(s):
    c = s["c"]
    n, heads, kv, ps, groups = c["n"], c["heads"], c["kv"], c["ps"], c["groups"]
    G, starts, shared = heads // kv, s["starts"].long(), s["shared"].long()
    i = torch.arange(n, device=DEV)
    g = torch.searchsorted(starts[1:], i, right=True)
    most = max(b - a for a, b in zip(_members(c), _members(c)[1:]))
    t = i - starts[g]
    q = s["q"].float().view(n, kv, G, 64)
    lens = s["lens"].long() if "lens" in s else shared[g]
    # the prefix of each group, for all its tokens at once
    L = s["prefix_width"] * ps
    page = s["prefix"].long().clamp(min=0)
    k = s["k"][page].permute(0, 2, 1, 3, 4).reshape(groups, kv, L, 64).float()
    v = s["v"][page].permute(0, 2, 1, 3, 4).reshape(groups, kv, L, 64).float()
    rows = torch.zeros(groups, most, kv, G, 64, device=DEV)
    rows[g, t] = q
    sees = torch.zeros(groups, most, dtype=torch.long, device=DEV)
    sees[g, t] = torch.minimum(lens, shared[g])
    there = (torch.arange(L, device=DEV) < sees[:, None, :, None, None]).expand(groups, 1, most, G, L).reshape(groups, 1, most * G, L)
    m, l, o = (x.view(groups, kv, most, G, -1)[g, :, t] for x in _part(rows.transpose(1, 2).reshape(groups, kv, most * G, 64), k, v, there))
    if "table" in s:
        # then each token's own positions
        L = c["max_own"] + 2 * ps
        p0 = shared[g] // ps * ps
        at = p0[:, None] + torch.arange(0, L // ps * ps, ps, device=DEV)
        page = torch.gather(s["table"].long(), 1, (at // ps).clamp(max=s["width"] - 1)).clamp(min=0)
        L = page.shape[1] * ps
        k = s["k"][page].permute(0, 2, 1, 3, 4).reshape(n, kv, L, 64).float()
        v = s["v"][page].permute(0, 2, 1, 3, 4).reshape(n, kv, L, 64).float()
        pos = p0[:, None] + torch.arange(L, device=DEV)
        there = ((pos >= shared[g][:, None]) & (pos < lens[:, None]))[:, None, None, :]
        m2, l2, o2 = _part(q, k, v, there)
        top = torch.maximum(m, m2)
        ref = torch.where(torch.isinf(top), 0.0, top)
        a, b = torch.exp(m - ref), torch.exp(m2 - ref)
        l, o = l * a + l2 * b, o * a + o2 * b
    out = torch.where(l > 0, o / l, 0.0)
    return {"out": out.reshape(n, heads * 64).to(s["q"].dtype)}


def run(s):
    if own:
        return _run_own(s)
    return {"fork": _fork_plain, "free": _free_plain, "compact": _compact_plain, "copy": _copy_plain, "prefix": _prefix_plain}[s["c"]["kind"]](s)


# --- bytes and operations ---------------------------------------------------------------------------

def work(case):
    c, kind = case, case["kind"]
    es = 4 if c.get("dtype") == "f32" else 2
    if kind == "fork":
        full = sum(first for first, _ in _entries(c))
        return {"bytes": 8.0 * full + 32.0 * c["n"], "flops": float(full)}
    if kind == "free":
        held = sum(have for _, have in _entries(c))
        return {"bytes": 4.0 * held + 12.0 * c["n"], "flops": float(held)}
    if kind == "compact":
        held = sum(have for _, have in _entries(c))
        fresh = sum(have - first for first, have in _entries(c))
        return {"bytes": 8.0 * held + 8.0 * fresh + 4.0 * c["n"], "flops": float(held)}
    if kind == "copy":
        rows = c["pairs"] * c["ps"] if c["rows"] == "all" else sum(1 + _even(i, c["ps"] - 2) for i in range(c["pairs"]))
        by = 4.0 * rows * c["kv"] * 64 * es * c["layers"]
        if c["rows"] == "all":
            by += 2.0 * c["pairs"] * c["kv"] * 128 * es * c["layers"]
        return {"bytes": by + 12.0 * c["pairs"], "flops": 0.0}
    shared, lens = _lengths(c)
    at = _members(c)
    group_of = [k for k in range(c["groups"]) for _ in range(at[k + 1] - at[k])]
    mine = sum(max(0, v - shared[k]) for v, k in zip(lens, group_of))
    there = sum(v for k, v in enumerate(shared) if at[k + 1] > at[k])
    return {"bytes": 2.0 * c["kv"] * 64 * es * (there + mine) + 4.0 * (there + mine) / c["ps"] + 2.0 * c["n"] * c["heads"] * 64 * es,
            "flops": 4.0 * c["heads"] * 64 * sum(lens)}


# --- the same from the definitions ------------------------------------------------------------------

def _exact_pages(c, s):
    ps, pages, n = c["ps"], s["pages"], c["n"]
    table, pool, used, lens, keep = s["table"].tolist(), s["pool"].tolist(), int(s["used"]), s["lens"].tolist(), s["keep"].tolist()
    if c["kind"] == "fork":
        src, dst, part = [-1] * n, [-1] * n, [0] * n
        for i, p in enumerate(s["parents"].tolist()):
            if p < 0:
                continue
            lens[i] = keep[i]
            for j in range(-(-keep[i] // ps)):
                table[i][j] = table[p][j]
            j = keep[i] // ps
            if keep[i] % ps and 0 <= table[p][j] < pages:   # a page of its own for what the parent has begun
                src[i], dst[i], part[i] = table[p][j], pool[used], keep[i] % ps
                table[i][j] = pool[used]
                used += 1
        return {"table": _int(table), "lens_out": _int(lens), "src": _int(src), "dst": _int(dst), "rows": _int(part), "used_out": _int([used]),
                "status": _int([0])}
    if c["kind"] == "free":
        held, gone = set(pool[used:]), set()
        for row, v in zip(table, keep):
            held.update(row[:-(-v // ps)])
        for row, v, w in zip(table, keep, lens):
            gone.update(x for x in row[-(-v // ps):-(-w // ps)] if 0 <= x < pages and x not in held)
        pool[used - len(gone):used] = sorted(gone)
        return {"lens_out": _int(keep), "pool": _int(pool), "used_out": _int([used - len(gone)]), "status": _int([0])}
    live = {x for row, v in zip(table, lens) for x in row[:-(-v // ps)] if 0 <= x < pages}
    both = sorted(live | set(pool[used:]))
    low, high = both[:len(live)], both[len(live):]
    to = dict(zip((x for x in high if x in live), (x for x in low if x not in live)))
    for row, v in zip(table, lens):
        m = -(-v // ps)
        row[:m] = [to.get(x, x) for x in row[:m]]
    pool[used:] = high
    src = list(to) + [-1] * (s["cap"] - len(to))
    dst = list(to.values()) + [-1] * (s["cap"] - len(to))
    return {"table_out": _int(table), "pool_out": _int(pool), "src": _int(src), "dst": _int(dst), "count": _int([len(to)]), "status": _int([0])}


def _rows_of(s, row, first, end):
    """Keys and values of the positions from `first` to `end` of a table's row, [kv, L, 64] in 64 bits."""
    ps = s["c"]["ps"]
    at = torch.arange(first, end, device=DEV)
    page = row.long()[at // ps]
    return s["k"][page, :, at % ps].double().transpose(0, 1), s["v"][page, :, at % ps].double().transpose(0, 1)


def exact(case, seed):
    c, kind = case, case["kind"]
    s = prepare(case, seed)
    if kind in ("fork", "free", "compact"):
        return _exact_pages(c, s)
    if kind == "copy":
        want = {}
        rows = s["rows"].tolist() if "rows" in s else [c["ps"]] * c["pairs"]
        for name in _pools(c):
            x = s[name]
            want[name] = x.double()
            for a, b, m in zip(s["src"].tolist(), s["dst"].tolist(), rows):
                want[name][b][:, :m] = x[a][:, :m].double()
        return want
    n, heads, kv, at = c["n"], c["heads"], c["kv"], _members(c)
    shared, lens = _lengths(c)
    q = s["q"].double().view(n, kv, heads // kv, 64)
    out = torch.zeros(n, kv, heads // kv, 64, dtype=torch.float64, device=DEV)
    for g in range(c["groups"]):
        pk, pv = _rows_of(s, s["prefix"][g], 0, shared[g])
        if c["mode"] != "forks":   # tokens of one request, a few at a time: those that see other lengths get their own mask
            for a in range(at[g], at[g + 1], 64):
                b = min(a + 64, at[g + 1])
                sees = torch.tensor(lens[a:b], device=DEV)[:, None, None]
                for h in range(kv):
                    x = torch.matmul(q[a:b, h], pk[h].t().contiguous()) / 8
                    x.masked_fill_(torch.arange(shared[g], device=DEV) >= sees, -math.inf)
                    out[a:b, h] = torch.softmax(x, -1) @ pv[h]
            continue
        for i in range(at[g], at[g + 1]):
            if lens[i] == 0:
                continue
            ok, ov = _rows_of(s, s["table"][i], shared[g], lens[i])
            k, v = torch.cat([pk, ok], 1), torch.cat([pv, ov], 1)
            out[i] = torch.softmax((q[i] @ k.transpose(1, 2)) / 8, -1) @ v
    return {"out": out.reshape(n, heads * 64)}
