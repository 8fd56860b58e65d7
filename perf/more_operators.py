"""Decoding with drafted tokens on the paged cache as measured workloads:
appending rows with the position rotation applied on the way, attention of
trees of drafted tokens over the pages, and keeping the rows of the path that
was accepted (PagedCache of the package).

A case is a dict of plain values; "kind" says what one pass is:

  rotate   PagedCache.append_rotary: q and k of the new rows normed per head
           (some cases) and rotated at their positions, k and v into the pages
  attend   PagedCache.tree, then per layer PagedCache.attend_tree: the drafted
           tokens of every sequence over its pages and their own ancestors
  accept   PagedCache.tree, PagedCache.follow and PagedCache.keep: the path that
           the target's choices take through the tree, its rows moved to their
           places in every layer, the other rows' pages released
  step     all of it: the tree, per layer append_rotary and attend_tree, then
           follow and keep

Lengths, page numbers, tables and trees follow from the case alone; the seed
gives the contents.  Head shapes, rotary factor and base are those of the
attention mixer's workloads (perf/cases.py) and its tests.
"""
import importlib.util
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
own = False


def _pkg():
    if "qmoe_amd" not in sys.modules:
        d = os.path.join(ROOT, "qwen3.8-flash-next_amd")
        spec = importlib.util.spec_from_file_location("qmoe_amd", os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["qmoe_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["qmoe_amd"]


# heads, kv heads, head dim
HEADS = [(16, 2, 128), (4, 1, 256), (4, 2, 64), (8, 8, 128), (6, 2, 192)]
THETA, EPS = 1e7, 1e-6


def listed():
    return [
        # the smallest call: the new row of one conversation, a quarter of the head rotated, q and k normed
        dict(name="rotate_token", kind="rotate", shape=0, bf16=True, wide=False, page=16, seqs=1, nodes=1, even=True, depth=1,
             ctx_lo=333, ctx_hi=333, rot=32, inter=False, norm=True, tree=False, mix=1),
        # drafted trees of 64 conversations far into their contexts, f32 rows into bf16 pages
        dict(name="rotate_drafts_64", kind="rotate", shape=0, bf16=True, wide=True, page=16, seqs=64, nodes=24, even=False, depth=6,
             ctx_lo=500, ctx_hi=900000, rot=32, inter=False, norm=True, tree=True, mix=2),
        # prompts of a large batch, f32 as the framework's own caches, whole heads rotated in neighbouring pairs
        dict(name="rotate_prompts_f32", kind="rotate", shape=0, bf16=False, wide=False, page=64, seqs=5, nodes=4000, even=False,
             depth=1, ctx_lo=1, ctx_hi=2000, rot=128, inter=True, norm=False, tree=False, mix=3),
        # eight drafted tokens of one conversation
        dict(name="tree_one", kind="attend", shape=0, bf16=True, page=16, seqs=1, nodes=8, even=True, depth=4, ctx_lo=700, ctx_hi=700,
             window=0, sinks=0, grouped=False, layers=1, mix=4),
        # a decode batch: up to 16 drafted tokens for each of 64 conversations of very different lengths
        dict(name="tree_decode_64", kind="attend", shape=0, bf16=True, page=16, seqs=64, nodes=16, even=False, depth=6, ctx_lo=64,
             ctx_hi=32768, window=0, sinks=0, grouped=False, layers=2, mix=5),
        # wide trees over long contexts: 256 nodes each
        dict(name="tree_wide_8", kind="attend", shape=0, bf16=True, page=64, seqs=8, nodes=256, even=True, depth=9, ctx_lo=8000,
             ctx_hi=24000, window=0, sinks=0, grouped=True, layers=1, mix=6),
        # f32 pages, trees of 5 to 40 nodes
        dict(name="tree_f32_16", kind="attend", shape=0, bf16=False, page=24, seqs=16, nodes=40, even=False, depth=7, ctx_lo=300,
             ctx_hi=9000, window=0, sinks=0, grouped=False, layers=1, mix=7),
        # chains of five drafts under a window of 512 with 16 sinks, head dim 256
        dict(name="tree_window_32", kind="attend", shape=1, bf16=True, page=16, seqs=32, nodes=6, even=True, depth=6, ctx_lo=1000,
             ctx_hi=20000, window=512, sinks=16, grouped=True, layers=1, mix=8),
        # one conversation, one layer
        dict(name="accept_one", kind="accept", shape=0, bf16=True, page=16, seqs=1, nodes=12, even=True, depth=4, ctx_lo=300,
             ctx_hi=300, layers=1, mix=9),
        # 256 conversations, twelve attention layers
        dict(name="accept_256", kind="accept", shape=0, bf16=True, page=32, seqs=256, nodes=32, even=False, depth=7, ctx_lo=100,
             ctx_hi=3000, layers=12, mix=10),
        # a whole verify pass of four conversations
        dict(name="step_4", kind="step", shape=0, bf16=True, wide=False, page=16, seqs=4, nodes=10, even=True, depth=5, ctx_lo=200,
             ctx_hi=2000, rot=32, inter=False, norm=True, window=0, sinks=0, grouped=False, layers=3, mix=11),
        # and of 48, f32 rows into bf16 pages
        dict(name="step_48", kind="step", shape=0, bf16=True, wide=True, page=32, seqs=48, nodes=20, even=False, depth=6, ctx_lo=200,
             ctx_hi=8000, rot=32, inter=False, norm=True, window=0, sinks=0, grouped=False, layers=3, mix=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "attend", "attend", "attend", "accept", "step"])
    shape, bf16, mix = rng.choice([0, 0, 0, 1, 2, 3, 4]), rng.random() < 0.6, rng.randrange(1 << 20)
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    h, kvh, hd = HEADS[shape]
    c = dict(kind=kind, shape=shape, bf16=bf16, page=page, even=rng.random() < 0.3, mix=mix)
    row = 2 * kvh * hd * (2 if bf16 else 4)  # bytes of k and v
    if kind in ("rotate", "step"):
        c.update(wide=bf16 and rng.random() < 0.5, rot=rng.choice([hd // 4, hd // 4, hd, hd // 2, 20, 2 * rng.randint(1, hd // 2)]),
                 inter=rng.random() < 0.4, norm=rng.random() < 0.6)
    if kind == "rotate":
        tree = rng.random() < 0.5
        seqs = _log_int(rng, 1, 100)
        nodes = _log_int(rng, 1, 64) if tree else _log_int(rng, 1, max(2, 8000 // seqs))
        c.update(seqs=seqs, nodes=nodes, depth=rng.randint(1, 9) if tree else 1, ctx_lo=1, ctx_hi=_log_int(rng, 16, 1000000), tree=tree)
        return c
    if kind == "accept":
        c.update(seqs=_log_int(rng, 1, 256), nodes=_log_int(rng, 2, 64), depth=rng.randint(1, 8), ctx_lo=1,
                 ctx_hi=_log_int(rng, 16, 2000), layers=rng.randint(1, 6 if row <= 4096 else 2))
        return c
    window = rng.choice([0, 0, _log_int(rng, 4, 4096)])
    seqs = _log_int(rng, 1, 64 if kind == "attend" else 32)
    nodes = _log_int(rng, 1, 256 if seqs <= 8 else 48)
    if kind == "attend":
        hi = _log_int(rng, 16, min(32768, (300 << 20) // (seqs * row), (1 << 22) // (seqs * nodes) + 500))
    else:
        hi = _log_int(rng, 16, min(8000, (1 << 20) // (seqs * nodes) + 300))
    c.update(seqs=seqs, nodes=nodes, depth=rng.choice([1, 4, 6, 12, 300]), ctx_lo=max(1, hi // rng.choice([1, 8, 100])), ctx_hi=hi,
             window=window, sinks=rng.choice([0, 1, 4, 37]) if window else 0, grouped=rng.random() < 0.5,
             layers=rng.randint(1, 2) if kind == "attend" else rng.randint(1, 3))
    return c


# ------------------------------------------------------ what follows from a case

def _log_pick(r, lo, hi):
    return lo if hi <= lo else max(lo, min(hi, int(math.exp(r.uniform(math.log(max(lo, 1)), math.log(hi))))))


def _lengths(case):
    """(new rows, rows with the new ones) of every sequence; the first has the most new ones"""
    r = random.Random(case["mix"])
    seqs = []
    for i in range(case["seqs"]):
        ctx = _log_pick(r, case["ctx_lo"], case["ctx_hi"])
        new = case["nodes"] if case["even"] or i == 0 else r.randint(max(1, case["nodes"] // 8), case["nodes"])
        seqs.append((new, ctx + new))
    r.shuffle(seqs)
    return seqs


def _trees(case):
    """parents and depths of every sequence, in order of depth; depth as large as the nodes: some chains"""
    r = random.Random(case["mix"] + 7)
    out = []
    for new, _ in _lengths(case):
        depth = [0]
        chain = case["depth"] >= new or r.random() < 0.1
        for _ in range(1, new):
            at = r.randrange(len(depth))
            depth.append(len(depth) if chain else min(depth[at], case["depth"] - 2) + 1 if case["depth"] > 1 else 1)
        depth = [0] + sorted(depth[1:])
        parents = [-1]
        for t in range(1, new):
            above = [a for a in range(t) if depth[a] == depth[t] - 1]
            if not above:  # a level that nobody drew: one below the last row's
                depth[t] = depth[t - 1] + 1
                above = [a for a in range(t) if depth[a] == depth[t] - 1]
            parents.append(r.choice(above))
        out.append((parents, depth))
    return out


def _paths(case):
    """the rows that the target's choices accept, from row 0 on.  A row that
    moves is never where another one goes: a pass may then be run again on what
    it left."""
    r = random.Random(case["mix"] + 13)
    out = []
    for parents, _ in _trees(case):
        path = [0]
        while r.random() < 0.85:
            kids = [t for t in range(len(parents)) if parents[t] == path[-1]]
            if not kids:
                break
            path.append(r.choice(kids))
        while any(x in range(1, len(path)) and x != path.index(x) for x in path):
            path.pop()
        out.append(path)
    return out


def _pages_of(rows, page):
    return (rows + page - 1) // page


def _tables(spans, page, spare, rnd, pad):
    """distinct random pages for rows [first, len) of every sequence, -1 for
    the pages before (released behind a window): table rows, the pool's size"""
    need = [(lo // page, _pages_of(n, page)) for lo, n in spans]
    total = sum(b - a for a, b in need) + spare
    ids = list(range(total))
    rnd.shuffle(ids)
    width = max(b for _, b in need) + pad
    rows, at = [], 0
    for a, b in need:
        rows.append([-1] * a + ids[at:at + b - a] + [-1] * (width - b))
        at += b - a
    return rows, total


def _visible(ctx, depths, parents, window, sinks):
    """(query, key) pairs seen, and keys that any query sees"""
    pairs, seen, low = 0, set(), ctx
    for t, d in enumerate(depths):
        p = ctx + d
        lo = max(0, p - window + 1) if window else 0
        pairs += max(0, ctx - lo) + min(sinks, lo, ctx)
        low = min(low, lo)
        a = t
        while a >= 0:
            if not window or d - depths[a] < window or ctx + depths[a] < sinks:
                pairs += 1
                seen.add(a)
            a = parents[a]
    return pairs, ctx - low + min(sinks, low, ctx) + len(seen)


def _attend_work(case):
    h, kvh, hd = HEADS[case["shape"]]
    es = 2 if case["bf16"] else 4
    rows = pairs = keys = 0
    for (new, total), (parents, depths) in zip(_lengths(case), _trees(case)):
        p, k = _visible(total - new, depths, parents, case["window"], case["sinks"])
        rows, pairs, keys = rows + new, pairs + p, keys + k
    return rows, 2 * rows * h * hd * es + 2 * keys * kvh * hd * es, 4 * pairs * h * hd


def _moved(case):
    return sum(1 for path in _paths(case) for i, x in enumerate(path) if i != x)


def work(case):
    h, kvh, hd = HEADS[case["shape"]]
    es = 2 if case["bf16"] else 4
    rows = sum(new for new, _ in _lengths(case))
    total = dict(bytes=0, flops=0)
    if case["kind"] in ("rotate", "step"):
        layers = case.get("layers", 1)
        src = 4 if case["wide"] else es
        total["bytes"] += layers * rows * hd * (h + 2 * kvh) * (src + es)
        total["flops"] += layers * rows * (h + kvh) * (3 * case["rot"] + (4 * hd if case["norm"] else 0))
    if case["kind"] in ("attend", "step"):
        _, b, f = _attend_work(case)
        total["bytes"] += case["layers"] * b + 4 * rows
        total["flops"] += case["layers"] * f
    if case["kind"] in ("accept", "step"):
        total["bytes"] += 2 * 2 * case["layers"] * _moved(case) * kvh * hd * es + 16 * rows
    return total


# ------------------------------------------------------------------ inputs

class _Gen:
    def __init__(self, seed, stream):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed((seed * 1000003 + stream * 7919 + 31) % (1 << 62))

    def normal(self, shape, dtype):
        """drawn in slabs, so that a large pool needs no f32 copy of itself"""
        t = torch.empty(shape, dtype=dtype, device=DEV)
        flat = t.view(-1)
        for i in range(0, flat.numel(), 1 << 26):
            part = flat[i:i + (1 << 26)]
            part.copy_(torch.randn(part.shape, generator=self.g, device=DEV))
        return t

    def ints(self, n, top):
        return torch.randint(0, top, (n,), generator=self.g, device=DEV, dtype=torch.int32)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _drafts(s, case, seed):
    """drafted tokens, and the target's choice after each of them: the next
    token of the path on its rows, on its last row one that no child has; rows
    beside the path have a child chosen too, now and then"""
    g, starts = _Gen(seed, 11), s["host_starts"]
    tokens, chosen = g.ints(starts[-1], 50000), g.ints(starts[-1], 50000) + 50000
    r = random.Random(case["mix"] + 17)
    at, to, on = [], [], []
    for i, (path, (parents, _)) in enumerate(zip(_paths(case), _trees(case))):
        pairs = list(zip(path, path[1:]))
        on += [starts[i] + b for _, b in pairs]
        taken = set(path)
        for t, p in enumerate(parents):
            if p >= 0 and p not in taken and r.random() < 0.5:
                taken.add(p)
                pairs.append((p, t))
        at += [starts[i] + a for a, _ in pairs]
        to += [starts[i] + b for _, b in pairs]
    if on:  # a sibling of the path never holds the path's token
        tokens[torch.tensor(on, device=DEV)] += 100000
    if at:
        chosen[torch.tensor(at, device=DEV)] = tokens[torch.tensor(to, device=DEV)]
    s.update(tokens=tokens, chosen=chosen)


def prepare(case, seed):
    """pages with the contents of running sequences, tables, lengths and
    reference counts, the trees' parents and the inputs of the call"""
    h, kvh, hd = HEADS[case["shape"]]
    dtype = torch.bfloat16 if case["bf16"] else torch.float32
    page, kind = case["page"], case["kind"]
    s = dict(kind=kind, case=case)
    seqs = _lengths(case)
    lens = [n for _, n in seqs]
    # rotate: far positions behind a window, only the new rows have pages
    spans = [(n - new if kind == "rotate" else 0, n) for new, n in seqs]
    rows, n_pages = _tables(spans, page, 3, random.Random(case["mix"] + 1), 2)
    layers, starts = case.get("layers", 1), [0]
    for new, _ in seqs:
        starts.append(starts[-1] + new)
    n = starts[-1]
    refs = [0] * n_pages
    for x in rows:
        for p in x:
            if p >= 0:
                refs[p] += 1
    shape = (layers, n_pages, page, kvh, hd)
    s.update(starts=_i32(starts), host_starts=starts, host_lens=lens, most=max(new for new, _ in seqs),
             k=_Gen(seed, 4).normal(shape, dtype), v=_Gen(seed, 5).normal(shape, dtype), table=_i32(rows), lens=_i32(lens),
             refs=_i32(refs))
    if kind != "rotate" or case["tree"]:
        trees = _trees(case)
        s.update(parents=_i32([p for t, _ in trees for p in t]), levels=max(max(d) for _, d in trees) + 1)
    if kind in ("rotate", "step"):
        src = torch.float32 if case["wide"] else dtype
        s.update(q=_Gen(seed, 1).normal((layers, n, h, hd), src), k_new=_Gen(seed, 2).normal((layers, n, kvh, hd), src),
                 v_new=_Gen(seed, 3).normal((layers, n, kvh, hd), src),
                 q_rot=torch.empty((layers, n, h, hd), dtype=dtype, device=DEV))
        i = torch.arange(case["rot"] // 2, dtype=torch.float64, device=DEV)
        s["freqs"] = (THETA ** (-2.0 * i / case["rot"])).float()
        if case["norm"]:
            s["q_norm"], s["k_norm"] = (1.0 + 0.1 * _Gen(seed, x).normal((hd,), torch.float32) for x in (6, 7))
    if kind == "attend":
        s["q"] = _Gen(seed, 1).normal((layers, n, h, hd), dtype)
    if kind in ("attend", "step"):
        s["out"] = torch.empty((layers, n, h, hd), dtype=dtype, device=DEV)
    if kind in ("accept", "step"):
        _drafts(s, case, seed)
        s.update(table0=s["table"].clone(), lens0=s["lens"].clone(), refs0=s["refs"].clone())
    if own:
        s["cache"] = _pkg().PagedCache(s["k"], s["v"], s["table"], s["lens"], s["refs"])
    return s


# ------------------------------------------------------------------ a pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _back(s):
    """every pass starts from the drafted rows still counted: lengths and tables are put back"""
    for x in ("table", "lens", "refs"):
        s[x].copy_(s[x + "0"])


def _run_own(s):
    kind, case, c = s["kind"], s["case"], s["cache"]
    if kind in ("accept", "step"):
        _back(s)
    tree = c.tree(s["parents"], s["starts"], most=s["most"]) if "parents" in s else None
    for l in range(case.get("layers", 1)):
        q = s["q"][l] if "q" in s else None
        if kind in ("rotate", "step"):
            q = c.append_rotary(l, s["k_new"][l], s["v_new"][l], s["starts"], s["freqs"], q=q, tree=tree, q_norm=s.get("q_norm"),
                                k_norm=s.get("k_norm"), eps=EPS, interleaved=case["inter"], out=s["q_rot"][l])
        if kind in ("attend", "step"):
            c.attend_tree(l, q, tree, window=case["window"], sinks=case["sinks"], grouped=case["grouped"], out=s["out"][l])
    if kind == "rotate":
        return s["q_rot"], s["k"], s["v"]
    if kind == "attend":
        return s["out"]
    rows, counts, token = c.follow(tree, s["tokens"], s["chosen"])
    status = c.keep(rows, counts, s["starts"])
    return _kept(s, rows, counts, token, status)


def _kept(s, rows, counts, token, status):
    got = (rows, counts, token, status, s["table"], s["lens"], s["refs"], s["k"], s["v"])
    return (s["q_rot"], s["out"]) + got if s["kind"] == "step" else got


# --------------------------------------------------------------- plain forms

def _run_plain(s):
    kind, case = s["kind"], s["case"]
    if kind in ("accept", "step"):
        _back(s)
    starts, n = s["starts"].long(), s["host_starts"][-1]
    t = torch.arange(n, device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    first = s["lens"].long()[seq] - (starts[seq + 1] - starts[seq])  # rows before the new ones
    pos = first + t - starts[seq]                                    # where a row lies
    depth = None
    if "parents" in s:
        parents = s["parents"].long()
        up = torch.where(parents >= 0, parents + starts[seq], -1)
        depth, cur = torch.zeros_like(t), up
        for _ in range(s["levels"] - 1):
            depth = depth + (cur >= 0)
            cur = torch.where(cur >= 0, up[cur.clamp(min=0)], -1)
    for l in range(case.get("layers", 1)):
        q = s["q"][l] if "q" in s else None
        if kind in ("rotate", "step"):
            _rotary(s, l, seq, pos, pos if depth is None else first + depth)
            q = s["q_rot"][l]
        if kind in ("attend", "step"):
            _attend(s, l, q, up, depth)
    if kind == "rotate":
        return s["q_rot"], s["k"], s["v"]
    if kind == "attend":
        return s["out"]
    rows, counts, token = _follow(s, seq, starts, parents, depth)
    return _kept(s, rows, counts, token, _keep(s, seq, starts, first, rows, counts))


def _turn(x, cos, sin, rot, inter):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, d = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((c, d), -1).flatten(-2) if inter else torch.cat((c, d), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _rotary(s, l, seq, pos, at):
    """q and k normed and rotated at positions `at`, k and v to rows `pos`; angles in 64 bits"""
    case, page = s["case"], s["k"].shape[2]
    angle = at.double()[:, None, None] * s["freqs"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def rows(x, w):
        x = x.float()
        if w is not None:
            x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w
        return _turn(x, cos, sin, case["rot"], case["inter"]).to(s["k"].dtype)

    s["q_rot"][l] = rows(s["q"][l], s.get("q_norm"))
    ids = s["table"][seq, pos // page].long()
    s["k"][l, ids, pos % page] = rows(s["k_new"][l], s.get("k_norm"))
    s["v"][l, ids, pos % page] = s["v_new"][l].to(s["v"].dtype)


def _attend(s, l, q, up, depth):
    case, out, page = s["case"], s["out"][l], s["k"].shape[2]
    h, kvh, hd = HEADS[case["shape"]]
    window, sinks = case["window"], case["sinks"]
    hh = torch.arange(h, device=DEV)
    kv_of = hh // (h // kvh) if case["grouped"] else hh % kvh
    for i, n in enumerate(s["host_lens"]):
        a, b = s["host_starts"][i], s["host_starts"][i + 1]
        c, first = b - a, n - (b - a)
        ids = s["table"][i, :_pages_of(n, page)].long()
        k, v = (s[x][l, ids].reshape(-1, kvh, hd)[:n].float().transpose(0, 1)[kv_of] for x in "kv")
        t = torch.arange(c, device=DEV)
        mine = torch.zeros((c, c), dtype=torch.bool, device=DEV)
        cur = t
        for _ in range(s["levels"]):
            mine[t[cur >= 0], cur[cur >= 0]] = True
            cur = torch.where(cur >= 0, up[a + cur.clamp(min=0)] - a, -1)
            cur = cur.clamp(min=-1)
        d = depth[a:b]
        j = torch.arange(first, device=DEV)
        ctx = torch.ones((c, first), dtype=torch.bool, device=DEV)
        if window:
            ctx = ((first + d)[:, None] - j[None] < window) | (j < sinks)[None]
            mine = mine & ((d[:, None] - d[None] < window) | (first + d < sinks)[None])
        see = torch.cat((ctx, mine), 1)
        sc = torch.matmul(q[a:b].float().transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) / math.sqrt(hd)
        sc = torch.where(see[None], sc, -math.inf)
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = torch.matmul(p, v.contiguous()) / p.sum(-1, keepdim=True)
        out[a:b] = o.transpose(0, 1).to(out.dtype)


def _follow(s, seq, starts, parents, depth):
    m, n = starts.shape[0] - 1, parents.shape[0]
    t = torch.arange(n, device=DEV)
    index = t - starts[seq]
    fits = (parents >= 0) & (s["tokens"] == s["chosen"][(starts[seq] + parents).clamp(min=0)])
    cur = torch.zeros(m, dtype=torch.long, device=DEV)
    rows = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    rows[starts[:-1]] = 0
    counts, going = torch.ones(m, dtype=torch.int32, device=DEV), torch.ones(m, dtype=torch.bool, device=DEV)
    for step in range(1, s["levels"]):
        kid = torch.where(fits & (parents == cur[seq]) & going[seq], index, n)
        best = torch.full((m,), n, dtype=torch.long, device=DEV).scatter_reduce(0, seq, kid, "amin")
        going = best < n
        cur = torch.where(going, best, cur)
        counts += going.int()
        place = starts[:-1] + step
        rows[place[going]] = best[going].int()
    return rows, counts, s["chosen"][starts[:-1] + cur]


def _keep(s, seq, starts, first, rows, counts):
    page, table, refs = s["k"].shape[2], s["table"], s["refs"]
    t = torch.arange(rows.shape[0], device=DEV)
    place = t - starts[seq]
    kept = place < counts[seq]
    src, dst = (first + rows)[kept], (first + place)[kept]
    sq = seq[kept]
    si, di = table[sq, src // page].long(), table[sq, dst // page].long()
    s["k"][:, di, dst % page], s["v"][:, di, dst % page] = s["k"][:, si, src % page], s["v"][:, si, src % page]
    lens = first[starts[:-1]] + counts
    gone = torch.arange(table.shape[1], device=DEV)[None] >= ((lens + page - 1) // page)[:, None]
    held = torch.where(gone, table, -1).reshape(-1).long()
    refs.index_add_(0, held.clamp(min=0), -(held >= 0).int())
    table.copy_(torch.where(gone, -1, table))
    s["lens"].copy_(lens)
    return torch.zeros(1, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------ in 64 bits

def exact(case, seed):
    was, globals()["own"] = own, False
    try:
        s = prepare(case, seed)
    finally:
        globals()["own"] = was
    kind, starts = case["kind"], s["host_starts"]
    trees = _trees(case) if "parents" in s else None
    firsts = [n - (starts[i + 1] - starts[i]) for i, n in enumerate(s["host_lens"])]
    table = s["table"].tolist()
    k, v = s["k"].double(), s["v"].double()
    q_rot = out = None
    if kind in ("rotate", "step"):
        q_rot = _exact_rotary(case, s, k, v, trees, firsts, table)
    if kind == "rotate":
        return q_rot, k, v
    if kind in ("attend", "step"):
        out = _exact_attend(case, s, q_rot if kind == "step" else s["q"].double(), k, v, trees, firsts)
    if kind == "attend":
        return out
    rows, counts, token, lens, refs = [], [], [], [], s["refs"].tolist()
    chosen, page = s["chosen"].tolist(), case["page"]
    moved = []
    for i, path in enumerate(_paths(case)):
        rows += path + [-1] * (starts[i + 1] - starts[i] - len(path))
        counts.append(len(path))
        token.append(chosen[starts[i] + path[-1]])
        lens.append(firsts[i] + len(path))
        for to, x in enumerate(path):
            a, b = firsts[i] + x, firsts[i] + to
            moved.append((table[i][a // page], a % page, table[i][b // page], b % page))
        for e in range(_pages_of(lens[i], page), len(table[i])):
            if table[i][e] >= 0:
                refs[table[i][e]] -= 1
                table[i][e] = -1
    m = torch.tensor(moved, device=DEV)
    k[:, m[:, 2], m[:, 3]], v[:, m[:, 2], m[:, 3]] = k[:, m[:, 0], m[:, 1]], v[:, m[:, 0], m[:, 1]]
    got = (_i32(rows), _i32(counts), _i32(token), _i32([0]), _i32(table), _i32(lens), _i32(refs), k, v)
    return (q_rot, out) + got if kind == "step" else got


def _exact_rotary(case, s, k, v, trees, firsts, table):
    """as complex numbers: the pair (a, b) is a + ib, turned by e^(i angle)"""
    rot, page, starts = case["rot"], case["page"], s["host_starts"]
    at, where = [], []
    for i, f in enumerate(firsts):
        for t in range(starts[i + 1] - starts[i]):
            at.append(f + (trees[i][1][t] if trees else t))
            where.append((table[i][(f + t) // page], (f + t) % page))
    angle = torch.tensor(at, dtype=torch.float64, device=DEV)[:, None, None] * s["freqs"].double()
    turn = torch.polar(torch.ones_like(angle), angle)

    def rows(x, w):
        x = x.double()
        if w is not None:
            x = x * w.double() * (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).rsqrt()
        y = x.clone()
        ia = slice(0, rot, 2) if case["inter"] else slice(0, rot // 2)
        ib = slice(1, rot, 2) if case["inter"] else slice(rot // 2, rot)
        z = torch.complex(x[..., ia].contiguous(), x[..., ib].contiguous()) * turn
        y[..., ia], y[..., ib] = z.real, z.imag
        return y

    w = torch.tensor(where, device=DEV)
    q = torch.stack([rows(x, s.get("q_norm")) for x in s["q"]])
    for l in range(k.shape[0]):
        k[l, w[:, 0], w[:, 1]] = rows(s["k_new"][l], s.get("k_norm"))
        v[l, w[:, 0], w[:, 1]] = s["v_new"][l].double()
    return q


def _exact_attend(case, s, q, k, v, trees, firsts):
    h, kvh, hd = HEADS[case["shape"]]
    window, sinks, page, starts = case["window"], case["sinks"], case["page"], s["host_starts"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for i, f in enumerate(firsts):
        parents, depths = trees[i]
        c = len(parents)
        hide = torch.ones((c, f + c), dtype=torch.bool)
        j = torch.arange(f)
        for t in range(c):
            p, a = f + depths[t], t
            hide[t, :f] = (p - j >= window) & (j >= sinks) if window else False
            while a >= 0:
                if not window or p - (f + depths[a]) < window or f + depths[a] < sinks:
                    hide[t, f + a] = False
                a = parents[a]
        hide = hide.to(DEV)
        slot = torch.arange(f + c, device=DEV)
        pg = s["table"][i].long()[slot // page]
        for l in range(q.shape[0]):
            for g in range(kvh):
                kk, vv = k[l, pg, slot % page, g], v[l, pg, slot % page, g]
                for hh in range(h):
                    if (hh // (h // kvh) if case["grouped"] else hh % kvh) == g:
                        z = (q[l, starts[i]:starts[i + 1], hh] @ kk.T) * hd ** -0.5
                        out[l, starts[i]:starts[i + 1], hh] = torch.softmax(z.masked_fill(hide, -math.inf), -1) @ vv
    return out
