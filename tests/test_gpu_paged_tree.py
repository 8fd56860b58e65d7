"""Decoding with drafted tokens on the paged cache (PagedCache.append_rotary,
tree, attend_tree, follow, keep) on the GPU against plain restatements in 64
bits and Python integers.

Bar of attention: test_gpu_paged's, whose sums these are under another mask.

Bar of the rotation, in steps u = 2^-24 of fp32.  A normed element: the sum
of squares is 8 products in a chain and a tree of at most 5 sums (13 u), the
division by head_dim and the sum with eps 2 u, halved by the root, 2 u for the
root and 1 / x, 2 u for the two products: at most 12 u of it.  cos and sin: the
angle's rest, at most 1/8 turn, is rounded to fp32 (0.8 u of the angle), the
series' coefficients and sums are off by less than 4 u: 6 u together.  An
output a cos - b sin has two products and a sum more: (12 + 6 + 2) u (|a| +
|b|), taken as 24 u.  Not normed and not rotated elements are exact.  The
output's own rounding is 2^-8 (bf16) or 2^-24 (f32) of it.
"""
import random

import numpy as np
import pytest
import torch

from conftest import load_pkg
from test_gpu_paged import HEADS, Setup, U, check, i32, reference, tables  # noqa: F401

pytestmark = pytest.mark.gpu

DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])


@pytest.fixture(scope="module")
def dev(gpu):
    return gpu


def cuts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(int).tolist()


def grow(r, c, kind="tree", dead=0.0):
    """parents of a tree of c rows: drawn, a chain, a star, several roots; some rows no nodes"""
    up = []
    for t in range(c):
        if t == 0 or (kind == "roots" and r.random() < 0.3):
            p = -1
        elif kind == "chain":
            p = t - 1
        elif kind == "star":
            p = 0
        elif kind == "braid":
            p = max(t - 2, 0)
        else:
            p = r.randrange(max(0, t - 12), t)
        if r.random() < dead:
            p = r.choice([t, t + 3, -2, 10 ** 9, -2 ** 31])
        up.append(p)
    return up


def plan(up, limit=1024):
    """depth (-1: no node) and ancestors with itself of every row"""
    depth, kin = [], []
    for t, p in enumerate(up):
        ok = t < limit and (p == -1 or (0 <= p < t and depth[p] >= 0))
        depth.append(-1 if not ok else 0 if p == -1 else depth[p] + 1)
        kin.append(set() if not ok else {t} | (set() if p == -1 else kin[p]))
    return depth, kin


def sight(first, depth, kin, window, sinks):
    """[c, first + c]: what each row sees"""
    c = len(depth)
    see = torch.zeros(c, first + c, dtype=torch.bool)
    j = torch.arange(first)
    for t in range(c):
        if depth[t] < 0:
            continue
        p = first + depth[t]
        see[t, :first] = (p - j < window) | (j < sinks) if window else True
        for a in kin[t]:
            see[t, first + a] = not window or depth[t] - max(depth[a], 0) < window or first + max(depth[a], 0) < sinks
    return see


def masked(q, k, v, see, grouped, scale=None):
    """attention under a mask in 64 bits -> (out, A, B) of test_gpu_paged's bar; rows that see nothing are zero"""
    c, h, hd = q.shape
    kvh = k.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    out, A, B = (torch.zeros(c, h, hd, dtype=torch.float64) for _ in range(3))
    some = see.any(-1)
    for hh in range(h):
        g = hh // (h // kvh) if grouped else hh % kvh
        s = torch.where(see, (q[:, hh] @ k[:, g].T) * scale, -torch.inf)
        e = torch.where(see, torch.exp(s - torch.where(some, s.amax(-1), 0.0)[:, None]), 0.0)
        pr = e / torch.where(some, e.sum(-1), 1.0)[:, None]
        out[:, hh], A[:, hh] = pr @ v[:, g], pr @ v[:, g].abs()
        B[:, hh] = torch.where(see, (q[:, hh].abs() @ k[:, g].abs().T) * abs(scale), 0.0).amax(-1)[:, None]
    return out, A, B


def run_trees(s, ups, window=0, sinks=0, grouped=False, scale=None, slots=None, words=None, out=None):
    counts = [len(u) for u in ups]
    q, starts = s.queries(counts)
    st = i32(starts, s.dev)
    tree = s.cache.tree(i32([p for u in ups for p in u], s.dev), st, most=words and 32 * words)
    got = s.cache.attend_tree(0, q.to(s.dev), tree, None if slots is None else i32(slots, s.dev), window=window, sinks=sinks,
                              grouped=grouped, scale=scale, out=out)
    for i, up in enumerate(ups):
        sl = i if slots is None else slots[i]
        c, T = len(up), s.lens[sl]
        if c == 0:
            continue
        see = sight(T - c, *plan(up, 32 * words if words else 1024), window, sinks)
        want, A, B = masked(q[starts[i]:starts[i + 1]], s.hk[sl], s.hv[sl], see, grouped, scale)
        mine = got[starts[i]:starts[i + 1]]
        check(mine, want, A, B, s.hd, T, s.dtype, (i, c, T))
        assert (mine[~see.any(-1).to(s.dev)] == 0).all()
    return q, tree, got


# ---------------------------------------------------------------- trees

@pytest.mark.parametrize("kind", ["tree", "chain", "star", "roots", "braid"])
@pytest.mark.parametrize("dead", [0.0, 0.1])
def test_depths_and_ancestors(dev, kind, dead):
    r = random.Random(hash((kind, dead)) % 1000)
    cache = Setup(dev, HEADS[2], torch.float32, 8, [3]).cache
    counts = [1, 0, 2, 31, 32, 33, 64, 65, 100, 300, 1023, 1024, 1025, 1500, 7]
    ups = [grow(r, c, kind, dead) for c in counts]
    starts = cuts(counts)
    for most in (None, 64, 33, 0):
        tree = cache.tree(i32([p for u in ups for p in u], dev), i32(starts, dev), most=most)
        words = 32 if most is None else max(1, -(-most // 32))
        assert tree.seen.shape[1] == words
        depth, seen = tree.depths.cpu().numpy(), tree.seen.cpu().numpy().view(np.uint32)
        for i, up in enumerate(ups):
            d, kin = plan(up, 32 * words)
            assert depth[starts[i]:starts[i + 1]].tolist() == d
            for t in range(len(up)):
                bits = int.from_bytes(seen[starts[i] + t].astype("<u4").tobytes(), "little")
                assert bits == sum(1 << a for a in kin[t]), (i, t)


def test_trees_of_wrong_starts_stay_inside(dev):
    """rows of no sequence are left alone, starts out of range or order touch nothing outside the call"""
    pkg = load_pkg()
    parents, n = i32([-1, 0, 0, 1, -1, 0, 1, 2], dev), 8
    depths, seen = torch.full((n + 2,), 77, dtype=torch.int32, device=dev), torch.full((n + 2, 1), 77, dtype=torch.int32, device=dev)
    t, e = pkg.DraftTree(parents, None, depths[1:], seen[1:]), pkg.QmoeErr()
    import ctypes
    for starts, touched in (([2, 4, 6], range(2, 6)), ([-5, 3, 99], range(0, 8)), ([6, 2, 7], range(2, 7)), ([8, 8, 9], [])):
        depths.fill_(77)
        seen.fill_(77)
        st = i32(starts, dev)
        assert pkg.lib().qmoe_paged_tree_build(parents.data_ptr(), st.data_ptr(), n, 2, t._p, None, ctypes.byref(e)) == 0
        torch.cuda.synchronize()
        assert [x for x in range(-1, n + 1) if depths[x + 1] != 77] == list(touched), starts
        assert [x for x in range(-1, n + 1) if seen[x + 1] != 77] == list(touched), starts


# ---------------------------------------------------------------- attention

@pytest.mark.usefixtures("tables")
@DTYPES
@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("shape", range(len(HEADS)))
def test_ragged_trees(dev, shape, page, dtype):
    r = random.Random(shape * 10 + page)
    counts = [1, 2, 0, 8, 31, 1, 32, 5, 64, 33, 9, 70, 3, 40]
    lens = [1, 2, 0, 8, 40, 33, 95, 64, 65, 127, 128, 200, 300, 513]
    s = Setup(dev, HEADS[shape], dtype, page, lens, seed=shape * 100 + page)
    run_trees(s, [grow(r, c, r.choice(["tree", "tree", "roots", "chain", "star"])) for c in counts], grouped=shape % 2 == 1)
    # drafts of a few rows each, the usual step
    run_trees(s, [grow(r, min(c, 6)) for c in counts], grouped=shape % 2 == 0)


@pytest.mark.usefixtures("tables")
@DTYPES
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (2, 0), (3, 40), (5, 1), (32, 0), (33, 4), (100, 7), (2 ** 31 - 1, 9)])
def test_windows_and_sinks(dev, window, sinks, dtype):
    """windows shorter and longer than the trees are deep, sinks that reach into the drafts of short sequences"""
    r = random.Random(window % 1000 + sinks)
    lens, counts = [1, 12, 38, 90, 200, 333, 513, 64], [1, 12, 30, 40, 3, 100, 1, 64]
    for shape, page in ((0, 16), (2, 7), (1, 64)):
        s = Setup(dev, HEADS[shape], dtype, page, lens, seed=window % 1000 + shape)
        run_trees(s, [grow(r, c, k) for c, k in zip(counts, ["tree", "chain", "tree", "braid", "chain", "tree", "tree", "roots"])],
                  window=window, sinks=sinks, grouped=shape == 1)


@pytest.mark.usefixtures("tables")
@DTYPES
@pytest.mark.parametrize("lens,counts", [([4000, 10], [9, 10]), ([3000] * 3, [2, 130, 600]), ([9000], [256]),
                                         ([1500, 1100], [1024, 1000]), ([70] * 200, [6] * 200), ([50] * 700, [3, 0] * 350),
                                         ([20 + 97 * i % 2500 for i in range(90)], [5 + i % 13 for i in range(90)]),
                                         ([40, 33, 7] * 400, [20, 33, 0] * 400)],
                         ids=["long", "chunks", "wide", "largest", "many", "more_than_512", "indexed", "more_than_1024"])
def test_longer_trees(dev, lens, counts, dtype):
    r = random.Random(len(lens))
    s = Setup(dev, HEADS[0 if len(lens) < 100 else 2], dtype, 32, lens, seed=len(lens))
    ups = [grow(r, c) for c in counts]
    run_trees(s, ups)
    run_trees(s, ups, window=300, sinks=2)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("lens,counts", [([6500] * 9, [1024] * 9), ([4000, 900, 12000, 300], [1000, 800, 1024, 256])], ids=["even", "uneven"])
def test_more_units_than_run_at_once(dev, lens, counts):
    """tasks that do not fit the card's units: parts in two turns, where the table is long enough for them"""
    r = random.Random(50)
    s = Setup(dev, HEADS[2], torch.bfloat16, 16, lens, seed=51)
    run_trees(s, [grow(r, c) for c in counts])


@DTYPES
@pytest.mark.parametrize("shape", [(16, 2, 128), (4, 1, 256), (6, 2, 192), (8, 2, 64), (40, 1, 128)], ids=str)
def test_trees_of_many_sequences(dev, shape, dtype):
    """4, 8 and 16 drafts of 16 sequences on thousands of rows: units of 16, 32 and 128 rows, parts that are joined"""
    r = random.Random(3)
    s = Setup(dev, shape, dtype, 16, [r.randrange(500, 5000) for _ in range(16)], seed=4)
    for c in (4, 8, 16):
        run_trees(s, [grow(r, c) for _ in range(16)], grouped=True)


@pytest.mark.usefixtures("tables")
@DTYPES
def test_rows_that_are_no_node_give_zeros(dev, dtype):
    r = random.Random(5)
    lens, counts = [40, 300, 90, 5], [12, 50, 64, 5]
    s = Setup(dev, HEADS[0], dtype, 16, lens, seed=6)
    run_trees(s, [grow(r, c, "tree", 0.2) for c in counts])
    run_trees(s, [grow(r, c, "tree", 0.2) for c in counts], window=6, sinks=2)
    run_trees(s, [grow(r, c) for c in counts], words=1)  # rows past the first 32
    run_trees(s, [[5] * c for c in counts])  # not one node


@DTYPES
def test_chains_are_causal_order(dev, dtype):
    """a chain of drafts is attend()'s own order"""
    lens, counts = [300, 77, 1200], [5, 77, 130]
    s = Setup(dev, HEADS[0], dtype, 16, lens, seed=7)
    for window, sinks in ((0, 0), (20, 3)):
        q, starts = s.queries(counts)
        st = i32(starts, dev)
        tree = s.cache.tree(i32([t - 1 for c in counts for t in range(c)], dev), st)
        a = s.cache.attend(0, q.to(dev), st, window=window, sinks=sinks)
        b = s.cache.attend_tree(0, q.to(dev), tree, window=window, sinks=sinks)
        for i, c in enumerate(counts):
            want, A, B = reference(q[starts[i]:starts[i + 1]], s.hk[i], s.hv[i], c, window, sinks, False)
            for x in (a, b):
                check(x[starts[i]:starts[i + 1]], want, A, B, s.hd, lens[i], dtype, i)


@pytest.mark.usefixtures("tables")
@DTYPES
def test_masks_of_the_callers_own(dev, dtype):
    """bits and depths of no tree: any earlier rows, rows whose bits are empty, bits past the own row, which do not count"""
    pkg = load_pkg()
    r = random.Random(8)
    lens, counts = [30, 80, 45], [30, 41, 45]  # two of them without a row before the drafts
    s = Setup(dev, HEADS[0], dtype, 16, lens, seed=9)
    q, starts = s.queries(counts)
    depth, kin, words = [], [], []
    for c in counts:
        for t in range(c):
            depth.append(r.choice([0, 1, t // 3, t, 10 ** 6, -1]))
            w = r.choice([0, r.getrandbits(64), 2 ** 64 - 1])
            kin.append({a for a in range(t + 1) if w >> a & 1})
            words.append([w & 0xFFFFFFFF, w >> 32])
    seen = torch.from_numpy(np.array(words, dtype=np.uint32).view(np.int32)).to(dev)
    tree = pkg.DraftTree(None, i32(starts, dev), i32(depth, dev), seen)
    for window, sinks in ((0, 0), (4, 0), (3, 33)):
        out = s.cache.attend_tree(0, q.to(dev), tree, window=window, sinks=sinks)
        for i, c in enumerate(counts):
            a, b = starts[i], starts[i + 1]
            d = [min(x, t) for t, x in enumerate(depth[a:b])]
            see = sight(lens[i] - c, d, kin[a:b], window, sinks)
            want, A, B = masked(q[a:b], s.hk[i], s.hv[i], see, False)
            check(out[a:b], want, A, B, s.hd, lens[i], dtype, (i, window))
            assert (out[a:b][~see.any(-1).to(dev)] == 0).all()


@pytest.mark.usefixtures("tables")
@DTYPES
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -3e38])
@pytest.mark.parametrize("counts", [[8, 4, 1], [33, 80, 64]], ids=["drafts", "wide"])
def test_what_unseen_rows_hold_does_not_matter(dev, counts, junk, dtype):
    """drafts of other branches, unused rows of pages, free pages"""
    r = random.Random(10)
    lens = [45, 100, 97]
    s = Setup(dev, HEADS[0], dtype, 16, lens, seed=11, junk=junk)
    ups = [grow(r, c) for c in counts]
    run_trees(s, ups)
    q, starts = s.queries(counts)
    tree = s.cache.tree(i32([p for u in ups for p in u], dev), i32(starts, dev))
    for i, (n, c) in enumerate(zip(lens, counts)):  # the k and v of a row in the middle
        j = n - c + c // 2
        s.k[0, s.rows[i][j // 16], j % 16] = junk
        s.v[0, s.rows[i][j // 16], j % 16] = junk
    out = s.cache.attend_tree(0, q.to(dev), tree)
    for i, (n, c) in enumerate(zip(lens, counts)):
        see = sight(n - c, *plan(ups[i]), 0, 0)
        blind = ~see[:, n - c + c // 2]
        want, A, B = masked(q[starts[i]:starts[i + 1]], s.hk[i], s.hv[i], see, False)
        check(out[starts[i]:starts[i + 1]][blind.to(dev)], want[blind], A[blind], B[blind], 128, n, dtype, (i, "other branches"))
        if junk != junk:
            assert torch.isnan(out[starts[i]:starts[i + 1]][(~blind).to(dev)]).all()


@pytest.mark.usefixtures("tables")
@DTYPES
def test_more_drafts_than_rows_and_bad_lengths(dev, dtype):
    """lens below the new rows: the first of them are no rows of the cache; nothing outside the call is touched"""
    s = Setup(dev, HEADS[0], dtype, 8, [5, 30, 16], seed=12)
    ups = [[-1, 0, 1, 1, 2, 3, 0, 6], [-1, 0, 0], [-1]]
    q, starts = s.queries([8, 3, 1])
    tree = s.cache.tree(i32([p for u in ups for p in u], dev), i32(starts, dev))
    guard = torch.full((14, s.h, s.hd), 7.0, dtype=dtype, device=dev)
    s.cache.attend_tree(0, q.to(dev), tree, out=guard[1:13])
    # first = -3: row t of the sequence is cached row t - 3, positions are depth - 3
    depth, kin = plan(ups[0])
    see = torch.zeros(8, 5, dtype=torch.bool)
    for t in range(8):
        for a in kin[t]:
            if a >= 3:
                see[t, a - 3] = True
    want, A, B = masked(q[:8], s.hk[0], s.hv[0], see, False)
    check(guard[1:9], want, A, B, s.hd, 5, dtype, "short")
    for i in (1, 2):
        see = sight(s.lens[i] - len(ups[i]), *plan(ups[i]), 0, 0)
        want, A, B = masked(q[starts[i]:starts[i + 1]], s.hk[i], s.hv[i], see, False)
        check(guard[1 + starts[i]:1 + starts[i + 1]], want, A, B, s.hd, 30, dtype, i)
    assert (guard[0] == 7).all() and (guard[13] == 7).all()
    s.len_t.copy_(i32([10 ** 9, -7, 16], dev))
    s.cache.attend_tree(0, q.to(dev), tree, out=guard[1:13])
    assert (guard[9:12] == 0).all() and (guard[0] == 7).all() and (guard[13] == 7).all()
    # slots out of range, a batch that is refused
    guard.fill_(7)
    s.cache.attend_tree(0, q.to(dev), tree, slots=i32([-1, 99, -2 ** 31], dev), out=guard[1:13])
    assert (guard[0] == 7).all() and (guard[13] == 7).all() and torch.isfinite(guard.float()).all()
    guard.fill_(7)
    s.cache.attend_tree(0, q.to(dev), tree, out=guard[1:13], status=i32([4], dev))
    assert (guard == 7).all()


@pytest.mark.usefixtures("tables")
@DTYPES
@pytest.mark.parametrize("n", [90, 400])
def test_starts_in_no_order_stay_inside(dev, n, dtype):
    """sequences that have more rows together than the call: nothing outside it is touched, by any of the calls"""
    s = Setup(dev, HEADS[0], dtype, 16, [900] * 100, seed=19)
    starts = i32([0 if i % 2 else n for i in range(99)] + [0, n], dev)
    q = torch.randn(n, s.h, s.hd, generator=s.g).to(dtype).to(dev)
    parents = i32([t - 1 if t % 7 else max(t - 2, -1) for t in range(n)], dev)
    for st in (starts, starts.flip(0).contiguous(), starts[:40].contiguous()):
        tree = s.cache.tree(parents, st)
        guard = torch.full((n + 2, s.h, s.hd), 7.0, dtype=dtype, device=dev)
        s.cache.attend_tree(0, q, tree, out=guard[1:n + 1])
        assert (guard[0] == 7).all() and (guard[n + 1] == 7).all()
        before = s.refs.clone(), s.full.clone(), s.len_t.clone()
        rows, cnt, last = s.cache.follow(tree, torch.zeros_like(parents), torch.zeros_like(parents))
        assert (cnt >= 0).all() and (cnt <= n).all()
        assert int(s.cache.keep(rows, cnt, st)) == -1
        for a, b in zip(before, (s.refs, s.full, s.len_t)):
            assert torch.equal(a, b)
    # the last sequence has rows 0 .. n in any case
    kv = torch.randn(n, s.kvh, s.hd, generator=s.g).to(dtype).to(dev)
    s.cache.append_rotary(0, kv, kv, starts, torch.rand(4, device=dev), q=q, tree=tree)
    torch.cuda.synchronize()


@pytest.mark.usefixtures("tables")
@DTYPES
def test_released_pages_and_shared_slots(dev, dtype):
    s = Setup(dev, HEADS[0], dtype, 16, [100, 130, 90], seed=13)
    r = random.Random(14)
    ups = [grow(r, c) for c in (20, 33, 9)]
    s.rows[0][2] = -1
    s.rows[1] = [-5, 2 ** 31 - 1] + s.rows[1][2:]
    s.rows[2][5] = s.k.shape[1]  # the page of the last drafts
    s.table.copy_(i32(s.rows, dev))
    q, starts = s.queries([20, 33, 9])
    tree = s.cache.tree(i32([p for u in ups for p in u], dev), i32(starts, dev))
    out = s.cache.attend_tree(0, q.to(dev), tree)
    for i, (a, b) in enumerate([(32, 48), (0, 32), (80, 96)]):
        c = len(ups[i])
        see = sight(s.lens[i] - c, *plan(ups[i]), 0, 0)
        see[:, a:b] = False
        want, A, B = masked(q[starts[i]:starts[i + 1]], s.hk[i], s.hv[i], see, False)
        check(out[starts[i]:starts[i + 1]], want, A, B, s.hd, 130, dtype, i)
    t = Setup(dev, HEADS[2], dtype, 8, [60, 33], seed=15)
    run_trees(t, [grow(r, 5), grow(r, 12), grow(r, 5)], slots=[1, 0, 1], scale=-0.7)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("hd", [64, 128, 192, 256])
def test_weights_of_small_trees_have_16_bits(dev, hd):
    """up to 128 rows a sequence: bf16 outputs within the weights' 16 bits (2^-16 of A twice: a half step of the second
    part, and of the sum that leaves it out) and their own rounding, far below one bf16 part's 2^-8"""
    r = random.Random(hd)
    lens, counts = [2000, 1500, 900], [16, 5, 11]
    s = Setup(dev, (8, 1, hd), torch.bfloat16, 16, lens, seed=hd)
    ups = [grow(r, c) for c in counts]
    q, starts = s.queries(counts)
    tree = s.cache.tree(i32([p for u in ups for p in u], dev), i32(starts, dev))
    out = s.cache.attend_tree(0, q.to(dev), tree).double().cpu()
    for i, up in enumerate(ups):
        see = sight(lens[i] - counts[i], *plan(up), 0, 0)
        want, A, B = masked(q[starts[i]:starts[i + 1]], s.hk[i], s.hv[i], see, False)
        T = lens[i]
        tol = A * (2 * (hd + 24) * U * (B + 1) + 2 * (T + 64) * U + 2 * 2.0 ** -16)
        tol = tol + (want.abs() + tol) * 2.0 ** -8
        err = (out[starts[i]:starts[i + 1]] - want).abs()
        assert (err <= tol).all(), (i, float((err / tol).max()))


@DTYPES
def test_strides_and_repeats(dev, dtype):
    s = Setup(dev, HEADS[0], dtype, 16, [100, 33, 2000], seed=16, order="heads")
    r = random.Random(17)
    ups = [grow(r, c) for c in (30, 1, 20)]
    q, tree, got = run_trees(s, ups)
    qt = q.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    big = torch.full((16, 60, 3, 128), 9.0, dtype=dtype, device=dev)
    out = big[:, 4:55, 1].transpose(0, 1)
    s.cache.attend_tree(0, qt, tree, out=out)
    assert torch.equal(out, got)
    assert (big[:, :4] == 9).all() and (big[:, 55:] == 9).all() and (big[:, :, 0] == 9).all() and (big[:, :, 2] == 9).all()
    for _ in range(3):
        assert torch.equal(s.cache.attend_tree(0, q.to(dev), tree), got)


# ---------------------------------------------------------------- rotation

def turned(x, pos, freqs, inter, w, eps):
    """rows x [n, heads, hd] in 64 bits at positions pos: (rotated, |a| + |b| of the bar)"""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    rot = 2 * freqs.shape[0]
    ang = (pos.double()[:, None] * freqs.double()[None])[:, None]
    cos, sin = torch.from_numpy(np.cos(ang.numpy())), torch.from_numpy(np.sin(ang.numpy()))
    ia = slice(0, rot, 2) if inter else slice(0, rot // 2)
    ib = slice(1, rot, 2) if inter else slice(rot // 2, rot)
    a, b, y, mag = x[..., ia], x[..., ib], x.clone(), x.abs() * (w is not None)
    y[..., ia], y[..., ib] = a * cos - b * sin, a * sin + b * cos
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag


def near(got, want, mag, dtype, what):
    tol = 24 * U * mag
    tol = tol + (want.abs() + tol) * (2.0 ** -8 if dtype == torch.bfloat16 else U) * (1 if dtype == torch.bfloat16 else (mag > 0)) + 1e-38
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), (what, float((err / tol).max()))


PAIRS = pytest.mark.parametrize("src,dst", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                            (torch.float32, torch.bfloat16)], ids=["bf16", "f32", "f32_to_bf16"])


def new_rows(s, counts, src):
    n = sum(counts)
    q, k, v = (torch.randn(n, m, s.hd, generator=s.g).to(src) for m in (s.h, s.kvh, s.kvh))
    return q, k, v


def rows_of(s, pages, i, a, b):
    return torch.stack([pages[-1, s.rows[i][j // s.page], j % s.page] for j in range(a, b)]).cpu() if b > a else \
        torch.zeros(0, s.kvh, s.hd)


def check_append(s, counts, starts, q, k, v, got, at, freqs, inter, qn, kn, eps, dst, live=None):
    for i, c in enumerate(counts):
        a, b = starts[i], starts[i + 1]
        on = torch.ones(c, dtype=torch.bool) if live is None else live[a:b]
        if not on.any():
            continue
        want, mag = turned(k[a:b], at[a:b], freqs, inter, kn, eps)
        near(rows_of(s, s.k, i, s.lens[i] - c, s.lens[i])[on], want[on], mag[on], dst, (i, "k"))
        assert torch.equal(rows_of(s, s.v, i, s.lens[i] - c, s.lens[i])[on], v[a:b].to(dst)[on])
        if got is not None:
            want, mag = turned(q[a:b], at[a:b], freqs, inter, qn, eps)
            near(got[a:b][on.to(s.dev)], want[on], mag[on], dst, (i, "q"))


@PAIRS
@pytest.mark.parametrize("inter", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("shape", range(len(HEADS)))
def test_append_rotary(dev, shape, inter, src, dst):
    lens, counts = [1, 40, 0, 33, 200, 17, 9], [1, 40, 0, 1, 90, 2, 3]
    hd = HEADS[shape][2]
    for rot, norm, page in ((hd // 4, True, 16), (hd, False, 5), (2, True, 1), (20, False, 21), (hd // 2 + 6, True, 64)):
        s = Setup(dev, HEADS[shape], dst, page, lens, seed=rot + shape, junk=5.0)
        freqs = torch.rand(rot // 2, generator=s.g) ** 4
        qn, kn = (torch.randn(hd, generator=s.g) if norm else None for _ in range(2))
        eps = 0.3 if rot == 2 else 1e-6
        q, k, v = new_rows(s, counts, src)
        starts = cuts(counts)
        before = [x.clone() for x in (s.k, s.v)]
        put = lambda x: None if x is None else x.to(dev)
        got = s.cache.append_rotary(0, put(k), put(v), i32(starts, dev), put(freqs), q=put(q), q_norm=put(qn), k_norm=put(kn),
                                    eps=eps, interleaved=inter)
        at = torch.cat([torch.arange(n - c, n) for n, c in zip(lens, counts)])
        check_append(s, counts, starts, q, k, v, got, at, freqs, inter, qn, kn, eps, dst)
        # no other row of the pool is written
        for x, y in zip((s.k, s.v), before):
            for i, (n, c) in enumerate(zip(lens, counts)):
                for j in range(n - c, n):
                    y[0, s.rows[i][j // page], j % page] = x[0, s.rows[i][j // page], j % page]
            assert torch.equal(x, y)
        # k alone writes the same
        for x in (s.k, s.v):
            x.fill_(5.0)
        assert s.cache.append_rotary(0, put(k), put(v), i32(starts, dev), put(freqs), k_norm=put(kn), eps=eps,
                                     interleaved=inter) is None
        check_append(s, counts, starts, q, k, v, None, at, freqs, inter, qn, kn, eps, dst)


def test_rotary_of_far_positions(dev):
    """angles in 64 bits: positions up to 2^29, where position * freq has 53 bits; windows behind which all is released"""
    pkg = load_pkg()
    kvh, hd, page, h = 2, 64, 4096, 3
    lens = [2 ** 29, 2 ** 29 - 1, 1000003, 2 ** 24 + 1, 65537, 3]
    width = 2 ** 29 // page
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=dev)
    for i, n in enumerate(lens):
        table[i, (n - 1) // page] = i
    k, v = (torch.zeros(1, len(lens), page, kvh, hd, device=dev) for _ in range(2))
    cache = pkg.PagedCache(k, v, table, i32(lens, dev), torch.ones(len(lens), dtype=torch.int32, device=dev))
    g = torch.Generator().manual_seed(21)
    n = len(lens)
    for freqs in (torch.tensor([1.0, 0.1, 1e-3, 1e-7, 0.999999, 0.25, 3.0, 0.0, 2.0 ** -30, 0.7071]),
                  torch.rand(32, generator=g), 1e7 ** (-torch.arange(16) / 16.0), -torch.rand(5, generator=g)):
        freqs = freqs.float()
        q, kn, vn = (torch.randn(n, m, hd, generator=g) for m in (h, kvh, kvh))
        got = cache.append_rotary(0, kn.to(dev), vn.to(dev), i32(list(range(n + 1)), dev), freqs.to(dev), q=q.to(dev))
        at = torch.tensor(lens) - 1
        want, mag = turned(q, at, freqs, False, None, 0)
        near(got, want, mag, torch.float32, "q")
        want, mag = turned(kn, at, freqs, False, None, 0)
        near(torch.stack([k[0, i, (x - 1) % page] for i, x in enumerate(lens)]), want, mag, torch.float32, "k")


@PAIRS
def test_rotary_of_trees_and_rows_that_are_not_written(dev, src, dst):
    """positions by depth; rows that are no node, of no sequence, before the first, without a page, of a slot out of
    range or of a refused batch stay as they are"""
    r = random.Random(22)
    lens, counts = [50, 9, 100, 70, 20], [20, 9, 33, 40, 5]
    ups = [grow(r, c, "tree", 0.1) for c in counts]
    s = Setup(dev, HEADS[0], dst, 16, lens, seed=23, junk=5.0)
    starts = cuts([2] + counts + [3])
    n = starts[-1]
    st = i32(starts[1:-1], dev)
    parents = [-1] * 2 + [p for u in ups for p in u] + [-1] * 3
    tree = s.cache.tree(i32(parents, dev), st)
    q, k, v = (torch.randn(n, m, s.hd, generator=s.g).to(src) for m in (s.h, s.kvh, s.kvh))
    freqs = torch.rand(16, generator=s.g)
    s.k.fill_(5.0)
    s.v.fill_(5.0)
    out = torch.full((n, s.h, s.hd), 5.0, dtype=dst, device=dev)
    rows3 = s.rows[3][2]
    s.table[3, 2] = -1  # rows 32 .. 47 of sequence 3 have no page: k and v go nowhere, q is rotated
    slots = i32([0, 1, 2, 3, 77], dev)
    call = lambda status: s.cache.append_rotary(0, k.to(dev), v.to(dev), st, freqs.to(dev), q=q.to(dev), slots=slots, tree=tree,
                                                out=out, status=status)
    call(i32([3], dev))
    assert (out == 5).all() and (s.k == 5).all() and (s.v == 5).all()
    assert call(i32([0], dev)) is out
    assert (out[:2] == 5).all() and (out[starts[5]:] == 5).all() and (s.k[0, rows3] == 5).all()
    for i in range(4):
        a, b = starts[i + 1], starts[i + 2]
        depth, _ = plan(ups[i])
        live = torch.tensor(depth) >= 0
        at = torch.tensor([lens[i] - counts[i] + max(d, 0) for d in depth])
        want, mag = turned(q[a:b], at, freqs, False, None, 0)
        near(out[a:b][live.to(dev)], want[live], mag[live], dst, (i, "q"))
        assert (out[a:b][~live.to(dev)] == 5).all()
        want, mag = turned(k[a:b], at, freqs, False, None, 0)
        got, gv = (rows_of(s, x, i, lens[i] - counts[i], lens[i]) for x in (s.k, s.v))
        page = torch.tensor([not (i == 3 and 32 <= j < 48) for j in range(lens[i] - counts[i], lens[i])])
        near(got[live & page], want[live & page], mag[live & page], dst, (i, "k"))
        assert torch.equal(gv[live & page], v[a:b].to(dst)[live & page])
        assert (got[~(live & page)] == 5).all() and (gv[~(live & page)] == 5).all()
    # more new rows than cached ones: the first have no position
    s.len_t.copy_(i32([50, 4, 100, 70, 20], dev))
    out.fill_(5.0)
    s.cache.append_rotary(0, k.to(dev), v.to(dev), st, freqs.to(dev), q=q.to(dev), out=out)
    a = starts[2]
    assert (out[a:a + 5] == 5).all()
    want, mag = turned(q[a + 5:a + 9], torch.arange(4), freqs, False, None, 0)
    near(out[a + 5:a + 9], want, mag, dst, "short")


@DTYPES
def test_rotary_strides_in_place_and_infinities(dev, dtype):
    s = Setup(dev, HEADS[0], dtype, 16, [40, 33], seed=24, order="heads")
    counts, starts = [30, 5], [0, 30, 35]
    q, k, v = (x.to(dev) for x in new_rows(s, counts, dtype))
    w, freqs = torch.randn(129, generator=s.g).to(dev), torch.rand(23, generator=s.g).to(dev)
    st = i32(starts, dev)
    for inter in (False, True):
        kw = dict(interleaved=inter, q_norm=w[1:], k_norm=w[:128])  # weights that start at 4 bytes
        want = s.cache.append_rotary(0, k, v, st, freqs, q=q, **kw)
        pages = s.k.clone(), s.v.clone()
        big = torch.full((16, 60, 3, 128), 9.0, dtype=dtype, device=dev)
        qt = big[:, 4:39, 1].transpose(0, 1)
        qt.copy_(q)
        kv = torch.stack([k, v], 1)
        assert s.cache.append_rotary(0, kv[:, 0], kv[:, 1], st, freqs, q=qt, out=qt, **kw) is qt
        assert torch.equal(qt, want) and torch.equal(s.k, pages[0]) and torch.equal(s.v, pages[1])
        assert (big[:, :4] == 9).all() and (big[:, 39:] == 9).all() and (big[:, :, 0] == 9).all() and (big[:, :, 2] == 9).all()
    # an infinity or NaN stays with its head
    bad = q.clone()
    bad[3, 2, 7], bad[8, 1, 100] = float("inf"), float("nan")
    got = s.cache.append_rotary(0, k, v, st, freqs, q=bad, **kw)
    same = torch.ones(35, 16, dtype=torch.bool, device=dev)
    same[3, 2] = same[8, 1] = False
    assert torch.equal(got[same], want[same]) and torch.isnan(got[8, 1]).all()
    # nothing but zeros: the norm's eps
    assert (s.cache.append_rotary(0, k, v, st, freqs, q=torch.zeros_like(q), **kw) == 0).all()


@DTYPES
def test_offsets_past_32_bits(dev, dtype):
    """a pool of more than 2^31 elements: rows appended, attended, moved at both ends of it"""
    kvh, hd, page, h = 2, 128, 64, 4
    n_pages = (2 ** 31 + 2 ** 28) // (page * kvh * hd)
    k, v = (torch.empty(1, n_pages, page, kvh, hd, dtype=dtype, device=dev) for _ in range(2))
    ids = [n_pages - 1, 0, n_pages - 2, n_pages // 2]
    g = torch.Generator().manual_seed(25)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
    refs[torch.tensor(ids, device=dev)] = 1
    T, c = 250, 130
    cache = load_pkg().PagedCache(k, v, i32([ids], dev), i32([T], dev), refs)
    hk, hv = (torch.randn(T, kvh, hd, generator=g).to(dtype) for _ in range(2))
    cache.append(0, hk.to(dev), hv.to(dev), i32([0, T], dev))
    q = torch.randn(c, h, hd, generator=g).to(dtype)
    up = grow(random.Random(26), c)
    tree = cache.tree(i32(up, dev), i32([0, c], dev))
    out = cache.attend_tree(0, q.to(dev), tree)
    want, A, B = masked(q, hk, hv, sight(T - c, *plan(up), 0, 0), False)
    check(out, want, A, B, hd, T, dtype, "tree")
    freqs = torch.tensor([0.5, 0.01])
    got = cache.append_rotary(0, hk[T - c:].to(dev), hv[T - c:].to(dev), i32([0, c], dev), freqs.to(dev), q=q.to(dev), tree=tree)
    at = torch.tensor([T - c + d for d in plan(up)[0]])
    want, mag = turned(q, at, freqs, False, None, 0)
    near(got, want, mag, dtype, "q")
    want, mag = turned(hk[T - c:], at, freqs, False, None, 0)
    place = lambda j: (0, ids[j // page], j % page)
    near(torch.stack([k[place(j)] for j in range(T - c, T)]), want, mag, dtype, "k")
    moved = [k[place(j)].clone() for j in (T - c, T - c + 70, T - 1)]
    rows = i32([0, 70, c - 1] + [-1] * (c - 3), dev)
    assert int(cache.keep(rows, i32([3], dev), i32([0, c], dev))) == 0
    for x, j in zip(moved, range(T - c, T - c + 3)):
        assert torch.equal(k[place(j)], x)
    assert cache.lens.tolist() == [T - c + 3] and cache.table.tolist() == [ids[:2] + [-1, -1]]
    assert refs[torch.tensor(ids, device=dev)].tolist() == [1, 1, 0, 0]


# ---------------------------------------------------------------- follow and keep

def walk(up, depth, tokens, chosen):
    path = [0] if up and depth[0] >= 0 else []
    while path:
        kids = [t for t in range(len(up)) if up[t] == path[-1] and depth[t] >= 0 and tokens[t] == chosen[path[-1]]]
        if not kids:
            break
        path.append(kids[0])
    return path


@pytest.mark.parametrize("vocab", [1, 2, 5, 1000])
@pytest.mark.parametrize("most", [None, 64])
def test_follow(dev, vocab, most):
    """few tokens, so that siblings share them: the lowest is taken"""
    r = random.Random(vocab)
    cache = Setup(dev, HEADS[2], torch.float32, 8, [3]).cache
    counts = [1, 0, 2, 5, 33, 64, 65, 100, 700, 1024, 1100, 16] + [r.randrange(0, 40) for _ in range(80)]
    ups = [grow(r, c, r.choice(["tree", "chain", "star", "roots"]), r.choice([0.0, 0.05])) for c in counts]
    starts = cuts(counts)
    n = starts[-1]
    tokens, chosen = ([r.choice([-1, 0, 2 ** 31 - 1, -2 ** 31] if x % 97 == 0 else range(vocab)) for x in range(n)] for _ in range(2))
    tree = cache.tree(i32([p for u in ups for p in u], dev), i32(starts, dev), most=most)
    rows, cnt, nxt = (x.tolist() for x in cache.follow(tree, i32(tokens, dev), i32(chosen, dev)))
    for i, up in enumerate(ups):
        a, b = starts[i], starts[i + 1]
        path = walk(up, plan(up, most or 1024)[0], tokens[a:b], chosen[a:b])
        assert rows[a:b] == path + [-1] * (b - a - len(path)), i
        assert cnt[i] == len(path) and nxt[i] == (chosen[a + path[-1]] if path else -1), i


class Kept:
    """a cache of several layers, every row's contents its own, and the model of keep on it"""

    def __init__(self, dev, dtype, page, lens, layers=3, shape=(4, 2, 64), order="rows", seed=0):
        self.s = Setup(dev, shape, dtype, page, lens, seed=seed, layers=layers, order=order)
        self.dev, self.page, self.lens = dev, page, list(lens)
        self.cache = self.s.cache
        for x in (self.s.k, self.s.v):
            x.copy_(torch.randn(x.shape, generator=self.s.g).to(dtype))

    def state(self):
        return [x.clone() for x in (self.s.k, self.s.v, self.s.full, self.s.len_t, self.s.refs)]

    def check(self, counts, paths, slots=None, status=None):
        """keep() against moving the rows one by one"""
        s, page = self.s, self.page
        k, v, table, lens, refs = self.state()
        starts = cuts(counts)
        rows = i32([x for p, c in zip(paths, counts) for x in p + [-1] * (c - len(p))], self.dev)
        got = self.cache.keep(rows, i32([len(p) for p in paths], self.dev), i32(starts, self.dev),
                              None if slots is None else i32(slots, self.dev), status=status)
        assert int(got) == 0
        ids = table.tolist()
        for i, (path, c) in enumerate(zip(paths, counts)):
            sl = i if slots is None else slots[i]
            first = int(lens[sl]) - c
            for to, x in enumerate(path):
                a, b = first + x, first + to
                if a != b:
                    for t in (k, v):
                        t[:, ids[sl][b // page], b % page] = t[:, ids[sl][a // page], a % page]
            lens[sl] = first + len(path)
            for e in range(-(-int(lens[sl]) // page), table.shape[1]):
                if table[sl, e] >= 0:
                    refs[table[sl, e]] -= 1
                    table[sl, e] = -1
        for a, b in zip((k, v, table, lens, refs), (s.k, s.v, s.full, s.len_t, s.refs)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("order", ["rows", "heads"])
@DTYPES
@pytest.mark.parametrize("page", [1, 4, 7, 16, 64])
def test_keep(dev, page, dtype, order):
    r = random.Random(page)
    counts = [1, 5, 0, 12, 40, 7, 64, 3, 100, 9]
    lens = [c + x for c, x in zip(counts, [0, 3, 10, 0, 65, 16, 64, 1, 33, 200])]
    x = Kept(dev, dtype, page, lens, order=order, seed=page)
    paths = [sorted(r.sample(range(c), r.randint(0, c))) for c in counts]
    paths[4] = list(range(1, 40))  # every row one place on
    paths[8] = list(range(0, 100, 3))
    x.check(counts, paths)


@DTYPES
def test_keep_some_slots(dev, dtype):
    """slots in any order, the whole batch kept, nothing of it kept, one sequence, many layers, wide heads"""
    x = Kept(dev, dtype, 8, [30, 40, 50, 60], seed=31)
    x.check([7, 20, 1], [[0, 3, 6], list(range(20)), []], slots=[3, 0, 2])
    x.check([10, 10], [[9], []], slots=[0, 1], status=i32([0], dev))
    x = Kept(dev, dtype, 16, [33], layers=17, shape=(8, 8, 128), seed=32)
    x.check([20], [[0, 1, 2, 5, 9, 17, 18, 19]])
    x = Kept(dev, dtype, 3, [200, 210], layers=1, shape=(4, 1, 256), seed=33)
    x.check([180, 210], [list(range(0, 180, 2)), list(range(5, 205))])


@DTYPES
def test_keep_of_small_batches(dev, dtype):
    """one workgroup's and two launches' sizes: sequences, rows and layers around the limits"""
    r = random.Random(37)
    for n, rows, layers, page in ((1, 3, 1, 16), (3, 40, 2, 5), (16, 64, 1, 16), (16, 65, 1, 16), (17, 5, 1, 8), (2, 512, 4, 32), (16, 4, 9, 4)):
        counts = [r.randint(1, rows) for _ in range(n - 1)] + [rows]
        x = Kept(dev, dtype, page, [c + r.randrange(40) for c in counts], layers=layers, seed=n)
        slots = r.sample(range(n), n)
        counts = [counts[sl] for sl in slots]
        x.check(counts, [sorted(r.sample(range(c), r.randint(0, c))) for c in counts], slots=slots)


def test_keep_of_many_sequences(dev):
    r = random.Random(34)
    counts = [r.randrange(0, 6) for _ in range(1024)]
    x = Kept(dev, torch.float32, 4, [c + r.randrange(0, 9) for c in counts], layers=1, seed=35)
    x.check(counts, [sorted(r.sample(range(c), r.randint(0, c))) for c in counts])


def test_keep_refusals_change_nothing(dev):
    x = Kept(dev, torch.float32, 8, [20, 30, 16, 40], seed=36)
    s, c = x.s, x.cache
    before = x.state()

    def refused(rows, counts, starts, slots=None, want=-1, status=None):
        got = c.keep(i32(rows, dev), i32(counts, dev), i32(starts, dev), None if slots is None else i32(slots, dev), status=status)
        assert int(got) == want
        for a, b in zip(before, (s.k, s.v, s.full, s.len_t, s.refs)):
            assert torch.equal(a, b)

    good = [0, 2, -1, -1, 1, 3, -1, -1]
    refused(good, [2, 2], [0, 4, 8], [0, 0])                 # a slot twice
    refused(good, [2, 2], [0, 4, 8], [0, 4])                 # out of range
    refused(good, [2, 2], [0, 4, 8], [-1, 1])
    refused(good, [2, 5], [0, 4, 8])                         # more than the rows
    refused(good, [2, -1], [0, 4, 8])
    refused(good, [3, 2], [0, 4, 8])                         # -1 is no row
    refused([0, 2, 2, -1, 1, 3, -1, -1], [3, 2], [0, 4, 8])  # not ascending
    refused([0, 2, 1, -1, 1, 3, -1, -1], [3, 2], [0, 4, 8])
    refused([0, 4, -1, -1, 1, 3, -1, -1], [2, 2], [0, 4, 8])  # past the sequence
    refused([2 ** 31 - 1] * 8, [1, 1], [0, 4, 8])
    refused(good, [2, 2], [0, 4, 9])                         # starts past the call
    refused(good, [2, 2], [0, 4, 3])
    refused(good, [2, 2], [-1, 4, 8])
    refused(good, [2, 2], [0, 4, 8], want=7, status=i32([7], dev))
    refused([], [], [0], want=7, status=i32([7], dev))
    assert int(c.keep(i32([], dev), i32([], dev), i32([0], dev))) == 0
    refused(list(range(20)) + [-1], [20], [0, 21], [0])      # more new rows than cached ones
    for bad in (-3, 10 ** 6):
        s.len_t[1] = bad
        before = x.state()
        refused(good, [2, 2], [0, 4, 8])
    s.len_t[1] = 30
    s.full[1, 3] = -1  # rows 24 .. 31
    before = x.state()
    refused(good, [2, 2], [0, 4, 8])
    s.full[1, 3] = s.rows[1][3]
    s.refs[s.rows[1][3]] = 2  # another slot holds the page that row 1 would move within
    before = x.state()
    refused(good, [2, 2], [0, 4, 8])
    x.check([4, 4], [[0, 2], [0, 1]])  # rows that stay where they are do not write


# ---------------------------------------------------------------- together

def drafts(r, counts):
    ups = [grow(r, c) for c in counts]
    return ups, [p for u in ups for p in u]


@DTYPES
def test_decoding_with_drafts(dev, dtype):
    """reserve, tree, append_rotary and attend_tree, follow, keep, over many steps with forks, a window and releases:
    outputs against 64 bits over each sequence's own history, the cache against the rows that were accepted"""
    pkg = load_pkg()
    h, kvh, hd, page, layers, n, window, sinks = 8, 2, 64, 8, 2, 4, 60, 5
    c = pkg.PagedCache.allocate(layers, 160, page, kvh, hd, 6, 40, dtype, dev)
    c.k.fill_(float("nan"))
    c.v.fill_(float("nan"))
    g, r = torch.Generator().manual_seed(41), random.Random(42)
    freqs = 1e4 ** (-torch.arange(8) / 8.0)
    qn, kn = torch.rand(hd, generator=g) + 0.5, torch.rand(hd, generator=g) + 0.5
    dq, dk, df = qn.to(dev), kn.to(dev), freqs.to(dev)
    hist = {s: [[torch.zeros(0, kvh, hd, dtype=dtype)] * 2 for _ in range(layers)] for s in range(6)}

    def inputs(m):
        return [[torch.randn(m, x, hd, generator=g).to(dtype) for x in (h, kvh, kvh)] for _ in range(layers)]

    def rotated(x, at, w):
        return turned(x, at, freqs, False, w, 1e-6)

    def step(slots, counts, prompt=False):
        ups = [grow(r, m, "chain" if prompt else "tree") for m in counts]
        starts, sl = cuts(counts), i32(slots, dev)
        st = i32(starts, dev)
        firsts = [hist[s][0][0].shape[0] for s in slots]
        status = c.reserve(i32(counts, dev), sl)
        tree = c.tree(i32([p for u in ups for p in u], dev), st, most=max(counts))
        at = torch.tensor([f + d for f, u in zip(firsts, ups) for d in plan(u)[0]])
        new = []
        for l, (q, k, v) in enumerate(inputs(starts[-1])):
            qr = c.append_rotary(l, k.to(dev), v.to(dev), st, df, q=q.to(dev), slots=sl, tree=tree, q_norm=dq, k_norm=dk, status=status)
            out = c.attend_tree(l, qr, tree, sl, window=window, sinks=sinks, status=status)
            want, mag = rotated(q, at, qn)
            near(qr, want, mag, dtype, "q")
            kr = torch.cat([torch.stack([c.k[l, c.table[s, j // page], j % page] for j in range(f, f + m)])
                            for s, f, m in zip(slots, firsts, counts)]).cpu()
            want, mag = rotated(k, at, kn)
            near(kr, want, mag, dtype, "k")
            new.append((kr, v))
            table = c.table.tolist()
            for i, s in enumerate(slots):
                a, b = starts[i], starts[i + 1]
                kk, vv = torch.cat([hist[s][l][0], kr[a:b]]), torch.cat([hist[s][l][1], v[a:b]])
                see = sight(firsts[i], *plan(ups[i]), window, sinks)
                for e, p in enumerate(table[s]):
                    if p < 0:
                        see[:, e * page:(e + 1) * page] = False
                want, A, B = masked(qr[a:b].cpu(), kk, vv, see, False)
                check(out[a:b], want, A, B, hd, kk.shape[0], dtype, (l, s))
        assert int(status) == 0
        m = starts[-1]
        tokens, chosen = ([r.randrange(3) for _ in range(m)] for _ in range(2))
        if prompt:
            tokens = chosen = [1] * m
        rows, cnt, last = c.follow(tree, i32(tokens, dev), i32(chosen, dev))
        assert int(c.keep(rows, cnt, st, sl, status=status)) == 0
        for i, s in enumerate(slots):
            a, b = starts[i], starts[i + 1]
            path = walk(ups[i], plan(ups[i])[0], tokens[a:b], chosen[a:b])
            assert int(cnt[i]) == len(path) and int(last[i]) == chosen[a + path[-1]]
            for l in range(layers):
                hist[s][l] = [torch.cat([old, x[a:b][path]]) for old, x in zip(hist[s][l], new[l])]
        same()
        c.evict(window, sinks, sl)

    def same():
        table, lens = c.table.tolist(), c.lens.tolist()
        for s in range(6):
            assert lens[s] == hist[s][0][0].shape[0]
            for l in range(layers):
                for pages, mine in ((c.k, hist[s][l][0]), (c.v, hist[s][l][1])):
                    for e, p in enumerate(table[s]):
                        if p >= 0:
                            rows = mine[e * page:(e + 1) * page]
                            assert torch.equal(pages[l, p, :rows.shape[0]].cpu(), rows)
        assert (c.refs >= 0).all() and int(c.refs.sum()) == int((c.table >= 0).sum())

    step([0, 1], [37, 20], prompt=True)
    for _ in range(3):
        step([1, 0], [9, 14])
    assert int(c.fork(i32([0, 0, 1], dev), i32([2, 3, 4], dev))) == 0
    for a, b in ((2, 0), (3, 0), (4, 1)):
        hist[a] = [list(x) for x in hist[b]]
    for _ in range(8):
        step([4, 0, 2, 3, 1], [8, 1, 12, 30, 5])
    c.compact()
    step([2, 3], [40, 2])


@DTYPES
def test_a_captured_step_of_drafts(dev, dtype):
    """one graph of a whole step, replayed as the sequences grow, against eager calls on a second cache, with eager work
    between; a second graph of the same cache takes turns"""
    pkg = load_pkg()
    h, kvh, hd, n, layers = 16, 2, 128, 5, 2
    r = random.Random(43)
    counts = [7, 12, 1, 5, 9]
    ups, flat = drafts(r, counts)
    starts, parents, add = i32(cuts(counts), dev), i32(flat, dev), i32(counts, dev)
    m = sum(counts)
    g = torch.Generator(device=dev).manual_seed(44)
    caches = [pkg.PagedCache.allocate(layers, 300, 8, kvh, hd, n, 60, dtype, dev) for _ in range(3)]
    first = [3, 40, 1, 17, 8]
    s0 = i32(cuts(first), dev)
    k0, v0 = (torch.randn(sum(first), kvh, hd, generator=g, device=dev).to(dtype) for _ in range(2))
    for c in caches:
        c.k.zero_()
        c.v.zero_()
        assert int(c.reserve(i32(first, dev))) == 0
        for l in range(layers):
            c.append(l, k0, v0, s0)
    q, k, v = (torch.randn(m, x, hd, generator=g, device=dev).to(dtype) for x in (h, kvh, kvh))
    freqs, w = torch.rand(16, device=dev), torch.rand(hd, device=dev)
    tokens, chosen = (torch.randint(0, 2, (m,), generator=g, device=dev, dtype=torch.int32) for _ in range(2))

    def step(c):
        status = c.reserve(add)
        tree = c.tree(parents, starts, most=12)
        outs = []
        for l in range(layers):
            qr = c.append_rotary(l, k, v, starts, freqs, q=q, tree=tree, q_norm=w, k_norm=w, status=status)
            outs += [qr, c.attend_tree(l, qr, tree, window=40, sinks=2, status=status)]
        rows, cnt, last = c.follow(tree, tokens, chosen)
        kept = c.keep(rows, cnt, starts, status=status)
        c.evict(40, 2)
        return [status, rows, cnt, last, kept] + outs

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[2])
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            results.append(step(caches[0]))
        graphs.append(gr)
    for i in range(10):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=dev))
        for t in (tokens, chosen):
            t.copy_(torch.randint(0, 2, (m,), generator=g, device=dev))
        graphs[i % 2].replay()
        eager = step(caches[1])
        torch.cuda.synchronize()
        assert int(eager[0]) == 0 and int(eager[4]) == 0
        for a, b in zip(results[i % 2], eager):
            assert torch.equal(a, b), i
        for a, b in zip((caches[0].table, caches[0].lens, caches[0].refs, caches[0].k, caches[0].v),
                        (caches[1].table, caches[1].lens, caches[1].refs, caches[1].k, caches[1].v)):
            assert torch.equal(a, b)


def test_a_refused_step_of_drafts_writes_nothing(dev):
    """the pool is full: with the reserve's status the step leaves all as it was"""
    pkg = load_pkg()
    c = pkg.PagedCache.allocate(2, 6, 8, 2, 64, 2, 10, torch.bfloat16, dev)
    c.k.zero_()
    c.v.zero_()
    assert int(c.reserve(i32([24, 20], dev))) == 0
    before = [t.clone() for t in (c.k, c.v, c.table, c.lens, c.refs)]
    starts, n = i32([0, 9, 15], dev), 15
    q, k, v = (torch.randn(n, m, 64, device=dev).bfloat16() for m in (4, 2, 2))
    out = torch.full_like(q, 5.0)
    status = c.reserve(i32([9, 6], dev))
    tree = c.tree(i32([-1] + [0] * 8 + [-1] + [0] * 5, dev), starts)
    for l in range(2):
        c.append_rotary(l, k, v, starts, torch.rand(8, device=dev), q=q, tree=tree, out=out, status=status)
        c.attend_tree(l, q, tree, out=out, status=status)
    tokens = torch.zeros(n, dtype=torch.int32, device=dev)
    rows, cnt, _ = c.follow(tree, tokens, tokens)
    kept = c.keep(rows, cnt, starts, status=status)
    assert int(status) > 0 and int(kept) == int(status) and (out == 5).all()
    for a, b in zip(before, (c.k, c.v, c.table, c.lens, c.refs)):
        assert torch.equal(a, b)


def test_other_streams(dev):
    s = Setup(dev, HEADS[0], torch.bfloat16, 16, [2000, 60, 900], seed=45)
    r = random.Random(46)
    ups, flat = drafts(r, [9, 4, 20])
    q, starts = s.queries([9, 4, 20])
    q, st, parents = q.to(dev), i32(starts, dev), i32(flat, dev)
    tree = s.cache.tree(parents, st)
    a = s.cache.attend_tree(0, q, tree)
    torch.cuda.synchronize()
    s1, s2, outs = torch.cuda.Stream(), torch.cuda.Stream(), []
    for _ in range(5):
        t1 = s.cache.tree(parents, st, stream=s1)
        outs.append((s.cache.attend_tree(0, q, t1, stream=s1), t1))
        with torch.cuda.stream(s2):
            t2 = s.cache.tree(parents, st)
            outs.append((s.cache.attend_tree(0, q, t2), t2))
    torch.cuda.synchronize()
    for o, _ in outs:
        assert torch.equal(o, a)


def test_other_arguments_are_refused(dev):
    pkg = load_pkg()
    s = Setup(dev, HEADS[2], torch.bfloat16, 8, [20, 30], seed=47)
    c = s.cache
    st = i32([0, 3, 5], dev)
    parents = i32([-1, 0, 0, -1, 0], dev)
    tree = c.tree(parents, st)
    q, k = (torch.zeros(5, m, 64, dtype=torch.bfloat16, device=dev) for m in (4, 2))
    f = torch.rand(8, device=dev)
    ints = torch.zeros(5, dtype=torch.int32, device=dev)
    bad = [
        (lambda: c.tree(None, st), "parents"), (lambda: c.tree(parents, None), "parents"), (lambda: c.tree(parents.long(), st), "int32"),
        (lambda: c.tree(parents.cpu(), st), "int32"), (lambda: c.tree(parents, st[::2]), "contiguous"),
        (lambda: c.tree(parents, st, most=-1), "most"), (lambda: c.tree(parents, st, most=2 ** 31), "most"),
        (lambda: c.attend_tree(0, q, None), "tree"), (lambda: c.attend_tree(0, q[:4], tree), "rows"),
        (lambda: c.attend_tree(1, q, tree), "layer"), (lambda: c.attend_tree(2 ** 32, q, tree), "layer"),
        (lambda: c.attend_tree(0, q.float(), tree), "q must"), (lambda: c.attend_tree(0, q, tree, window=2 ** 31), "window"),
        (lambda: c.attend_tree(0, q, tree, scale=0.0), "scale"), (lambda: c.attend_tree(0, q, tree, out=q[:3]), "out"),
        (lambda: c.append_rotary(0, k, k, st, f[:0]), "freqs"), (lambda: c.append_rotary(0, k, k, st, None), "freqs"),
        (lambda: c.append_rotary(0, k, k, st, torch.rand(33, device=dev)), "freqs"),
        (lambda: c.append_rotary(0, k, k, st, f.double()), "freqs"), (lambda: c.append_rotary(0, k, k, st, f.cpu()), "freqs"),
        (lambda: c.append_rotary(0, k, k[:4], st, f), "same rows"), (lambda: c.append_rotary(0, k, k.float(), st, f), "same rows"),
        (lambda: c.append_rotary(0, k, k, st, f, q=q.float()), "q must"), (lambda: c.append_rotary(0, k, k, st, f, q=q[:3]), "q has"),
        (lambda: c.append_rotary(0, k, k, st, f, out=q), "without q"), (lambda: c.append_rotary(0, k, k, st, f, q_norm=f), "without q"),
        (lambda: c.append_rotary(0, k, k, st, f, k_norm=f), "k_norm"), (lambda: c.append_rotary(0, k, k, st, f, eps=-1.0), "eps"),
        (lambda: c.append_rotary(0, k, k, st, f, q=q, out=q[:2]), "out has"), (lambda: c.append_rotary(7, k, k, st, f), "layer"),
        (lambda: c.append_rotary(0, k[:4], k[:4], st, f, tree=tree), "rows"),
        (lambda: c.append_rotary(0, k, k, st, f, slots=ints[:1]), "slots"),
        (lambda: c.follow(tree, None, ints), "tokens"), (lambda: c.follow(tree, ints, ints[:3]), "chosen"),
        (lambda: c.follow(tree, ints.long(), ints), "tokens"), (lambda: c.keep(None, ints[:2], st), "rows"),
        (lambda: c.keep(ints, None, st), "counts"), (lambda: c.keep(ints, ints, st), "counts"),
        (lambda: c.keep(ints, ints[:2], st, slots=ints), "slots"), (lambda: c.keep(ints, ints[:2], None), "starts"),
        (lambda: c.keep(ints, ints[:2], st, status=ints), "status"),
    ]
    for i, (call, msg) in enumerate(bad):
        with pytest.raises(pkg.QmoeError, match=msg):
            call()
            pytest.fail(f"call {i} ({msg}) was not refused")
    # nothing to do
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    t = c.tree(none, i32([0, 0, 0], dev))
    assert c.attend_tree(0, q[:0], t).shape == (0, 4, 64)
    rows, cnt, last = c.follow(t, none, none)
    assert rows.shape == (0,) and cnt.tolist() == [0, 0] and last.tolist() == [-1, -1]
    assert int(c.keep(rows, cnt, i32([0, 0, 0], dev))) == 0
