"""The paged cache (qmoe_paged_*, PagedCache) on the GPU against plain
restatements: attention in 64 bits over each sequence's rows, the pages'
bookkeeping in Python integers.

Bar of attention.  With A = sum_j p_j |v_j| / sum p (64 bits) and B = the
row's largest scale * sum_i |q_i k_i|:
  * scores: each fp32 dot of hd products is off by at most (hd + 8) 2^-24 B
    (also when computed from parts of at least 24 bits), the log2 argument
    and exp2 by a few 2^-24 of it, so p / sum p is off by a factor of at most
    1 + 2 (hd + 24) 2^-24 (B + 1): slack S on A;
  * sums over T keys and the rescalings: 2 (T + 64) 2^-24 of A;
  * bf16 only: each weight p_j becomes p_j (1 + e_j), |e_j| <= 2^-8 (half a
    step), in the product with v and in the sum alike.  With w_j = p_j / sum p
    and D = sum_j w_j e_j, |D| <= 2^-8, the result is off by
    sum_j w_j e_j (v_j - out) / (1 + D), at most 2^-8 (A + |out|) / (1 - 2^-8).
    The output is rounded: 2^-8 of it.
  f32 output rounding: 2^-24 of it.
"""
import numpy as np
import pytest
import torch

from conftest import load_pkg

pytestmark = pytest.mark.gpu

HEADS = [(16, 2, 128), (4, 1, 256), (4, 2, 64), (8, 8, 128), (6, 2, 192), (5, 1, 64), (40, 1, 128)]
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev(gpu):
    return gpu


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Setup:
    """a cache with random pages for sequences of given lengths; the pages'
    unused rows and the free pages hold `junk`.  The table has room for
    `table_rows` rows at the least: short calls on short tables run on units
    of few rows, whatever the calls' own."""
    table_rows = 0

    def __init__(self, dev, shape, dtype, page, lens, seed=0, layers=1, spare=4, junk=0.0, order="rows", slots=None):
        self.h, self.kvh, self.hd = shape
        self.page, self.lens, self.dev, self.dtype = page, list(lens), dev, dtype
        g = torch.Generator().manual_seed(seed)
        n_slots = slots or len(lens)
        need = [-(-n // page) for n in lens] + [0] * (n_slots - len(lens))
        n_pages = sum(need) + spare
        ids = torch.randperm(n_pages, generator=g).tolist()
        width = max(max(need), 1) + 2
        self.rows, at = [], 0
        for c in need:
            self.rows.append(ids[at:at + c] + [-1] * (width - c))
            at += c
        refs = [0] * n_pages
        for r in self.rows:
            for p in r:
                if p >= 0:
                    refs[p] += 1
        dims = {"rows": (layers, n_pages, page, self.kvh, self.hd), "heads": (layers, n_pages, self.kvh, page, self.hd)}[order]
        perm = (0, 1, 2, 3, 4) if order == "rows" else (0, 1, 3, 2, 4)
        self.k, self.v = (torch.full(dims, junk, dtype=dtype, device=dev).permute(perm) for _ in range(2))
        self.hk, self.hv = [], []
        for s, n in enumerate(lens):
            kk, vv = (torch.randn(n, self.kvh, self.hd, generator=g).to(dtype) for _ in range(2))
            self.hk.append(kk)
            self.hv.append(vv)
            for j0 in range(0, n, page):
                m = min(page, n - j0)
                self.k[layers - 1, self.rows[s][j0 // page], :m] = kk[j0:j0 + m].to(dev)
                self.v[layers - 1, self.rows[s][j0 // page], :m] = vv[j0:j0 + m].to(dev)
        self.full = torch.full((n_slots, max(width, -(-self.table_rows // page))), -1, dtype=torch.int32, device=dev)
        self.table, self.refs = self.full[:, :width], i32(refs, dev)
        self.table.copy_(i32(self.rows, dev))
        self.len_t = i32(list(lens) + [0] * (n_slots - len(lens)), dev)
        self.cache = load_pkg().PagedCache(self.k, self.v, self.full, self.len_t, self.refs)
        self.g = g

    def queries(self, counts):
        starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
        q = torch.randn(starts[-1], self.h, self.hd, generator=self.g).to(self.dtype)
        return q, starts


@pytest.fixture(params=[0, 1 << 20], ids=["short", "long"])
def tables(request, monkeypatch):
    monkeypatch.setattr(Setup, "table_rows", request.param)


def reference(q, k, v, n_new, window, sinks, grouped, scale=None, hidden=()):
    """one sequence in 64 bits: q [c, h, hd], k, v [len, kvh, hd] -> (out, A, B) ; rows without keys are zero"""
    c, h, hd = q.shape
    T, kvh = k.shape[0], k.shape[1]
    scale = hd ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    p = torch.arange(T - n_new, T)[:, None]
    j = torch.arange(T)[None]
    see = j <= p
    if window:
        see = see & ((p - j < window) | (j < sinks))
    for a, b in hidden:
        see = see & ~((j >= a) & (j < b))
    out, A, B = (torch.zeros(c, h, hd, dtype=torch.float64) for _ in range(3))
    if T == 0:
        return out, A, B
    for hh in range(h):
        g = hh // (h // kvh) if grouped else hh % kvh
        kk, vv = torch.where(torch.isfinite(k[:, g]), k[:, g], 0.0), v[:, g]
        s = (q[:, hh] @ k[:, g].T) * scale
        mag = (q[:, hh].abs() @ kk.abs().T) * abs(scale)
        s = torch.where(see, s, -torch.inf)
        m = s.amax(-1, keepdim=True)
        e = torch.where(see, torch.exp(s - m), 0.0)
        pr = torch.where(see.any(-1)[:, None], e / e.sum(-1, keepdim=True), 0.0)
        B[:, hh] = torch.where(see, mag, 0.0).amax(-1)[:, None]
        if torch.isfinite(vv).all():
            out[:, hh], A[:, hh] = pr @ vv, pr @ vv.abs()
            continue
        for r in range(c):  # only seen rows are multiplied: what others hold never counts
            idx = see[r].nonzero()[:, 0]
            out[r, hh], A[r, hh] = pr[r, idx] @ vv[idx], pr[r, idx] @ vv[idx].abs()
    return out, A, B


def bound(out, A, B, hd, T, dtype):
    tol = A * (2 * (hd + 24) * U * (B + 1) + 2 * (T + 64) * U)
    if dtype == torch.bfloat16:
        return tol + (A + out.abs()) / 255 + out.abs() * 2.0 ** -8 + 1e-38
    return tol + out.abs() * U + 1e-38


def check(got, want, A, B, hd, T, dtype, what):
    got = got.double().cpu()
    err = (got - want).abs()
    tol = bound(want, A, B, hd, max(T, 1), dtype)
    bad = ~(err <= tol)
    assert not bad.any(), (what, "worst", float((err / tol).nan_to_num(9e9).max()), int(bad.sum()))


def run_batch(s, counts, window=0, sinks=0, grouped=False, scale=None, slots=None, layer=0, hidden=None):
    q, starts = s.queries(counts)
    out = s.cache.attend(layer, q.to(s.dev), i32(starts, s.dev), None if slots is None else i32(slots, s.dev), window=window,
                         sinks=sinks, grouped=grouped, scale=scale)
    for i, c in enumerate(counts):
        sl = i if slots is None else slots[i]
        if c == 0:
            continue
        T = s.lens[sl]
        qi = q[starts[i]:starts[i] + c]
        blind = max(0, c - T)  # more queries than rows: the first see nothing
        want, A, B = reference(qi[blind:], s.hk[sl], s.hv[sl], c - blind, window, sinks, grouped, scale,
                               (hidden or {}).get(sl, ()))
        got = out[starts[i]:starts[i] + c]
        assert (got[:blind] == 0).all()
        check(got[blind:], want, A, B, s.hd, T, s.dtype, (i, c, T))
    return q, starts, out


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 100])
@pytest.mark.parametrize("shape", range(len(HEADS)))
def test_ragged_batches(dev, shape, page, dtype):
    lens = [1, 2, 0, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 7, 260, 40]
    counts = [1, 1, 0, 1, 3, 1, 0, 5, 1, 1, 128, 17, 1, 7, 4, 41]
    s = Setup(dev, HEADS[shape], dtype, page, lens, seed=shape * 100 + page)
    run_batch(s, counts, grouped=shape % 2 == 1)
    # one token each, the decode step
    run_batch(s, [1 if n else 0 for n in lens], grouped=shape % 2 == 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (32, 0), (33, 40), (64, 4), (100, 0), (1000, 5), (2 ** 31 - 1, 9)])
def test_windows_and_sinks(dev, window, sinks, dtype):
    lens, counts = [1, 5, 90, 200, 333, 513, 700, 64], [1, 5, 90, 3, 100, 1, 37, 0]
    for shape, page in ((0, 16), (2, 7), (1, 64)):
        s = Setup(dev, HEADS[shape], dtype, page, lens, seed=window % 1000 + shape)
        run_batch(s, counts, window=window, sinks=sinks, grouped=shape == 1)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("lens,counts", [([2500], [2500]), ([4000, 10], [1, 10]), ([3000] * 3, [2, 130, 600]),
                                         ([9000], [64]), ([70] * 200, [1] * 200), ([50] * 700, [1, 0] * 350)],
                         ids=["prompt", "long", "chunks", "chunk_of_long", "many", "more_than_512"])
def test_longer_batches(dev, lens, counts, dtype):
    s = Setup(dev, HEADS[0 if len(lens) < 100 else 2], dtype, 32, lens, seed=len(lens))
    run_batch(s, counts)
    run_batch(s, counts, window=300, sinks=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape,n", [((40, 1, 128), 16), ((48, 2, 64), 8)], ids=["128", "64"])
def test_many_units(dev, shape, n, dtype):
    """calls of more units than fill the card several times over, runs of more than 512 keys among them"""
    lens = [300 + 37 * i % 500 for i in range(2 * n)]
    counts = [min(m, 260) if i % 3 else min(m, 300) for i, m in enumerate(lens)]
    s = Setup(dev, shape, dtype, 24, lens, seed=21)
    assert sum(counts) * shape[0] // 128 >= 1000
    run_batch(s, counts)
    run_batch(s, counts, window=130, sinks=70, grouped=True)
    s.rows[3][5] = -1
    s.table.copy_(i32(s.rows, dev))
    s.v[0, s.rows[4][4], 4] = float("nan")  # key 100: its unit is computed one row at a time beside the others
    s.hv[4][100] = float("nan")
    q, starts = s.queries(counts)
    for window, sinks in ((0, 0), (130, 70)):
        out = s.cache.attend(0, q.to(dev), i32(starts, dev), window=window, sinks=sinks)
        for i in (3, 4, 5):
            c, a = counts[i], starts[i]
            want, A, B = reference(q[a:a + c], s.hk[i], s.hv[i], c, window, sinks, False, hidden=[(120, 144)] if i == 3 else ())
            pos = torch.arange(lens[i] - c, lens[i])
            sees = (pos >= 100) & ((pos < 230) | (window == 0)) & (i == 4)
            assert torch.isnan(out[a:a + c].cpu()[sees]).all()
            check(out[a:a + c].cpu()[~sees], want[~sees], A[~sees], B[~sees], s.hd, lens[i], dtype, (i, window))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape,window,sinks", [((64, 1, 64), 32, 0), ((64, 1, 64), 33, 40), ((32, 1, 128), 64, 4),
                                                ((32, 1, 192), 100, 0), ((32, 1, 256), 130, 9)], ids=str)
def test_windows_of_long_prompts(dev, shape, window, sinks, dtype):
    """small windows on units of many rows"""
    lens, counts = [713, 513, 900, 20, 0], [700, 513, 900, 1, 0]
    s = Setup(dev, shape, dtype, 20, lens, seed=25)
    run_batch(s, counts, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128, 192, 256])
def test_a_few_tokens_per_sequence(dev, hd, dtype, monkeypatch):
    """17 to 32 rows a sequence on long tables"""
    monkeypatch.setattr(Setup, "table_rows", 1 << 18)
    lens = [7000, 300, 3, 33, 64, 65, 700, 1, 90, 128, 513, 2, 40, 800, 77, 1000]
    counts = [min(m, 2 + i % 4) for i, m in enumerate(lens)]
    s = Setup(dev, (8, 1, hd), dtype, 16, lens, seed=26)
    run_batch(s, counts)
    run_batch(s, counts, window=6500, sinks=5)
    s.rows[6][3] = s.rows[0][100] = -1
    s.table.copy_(i32(s.rows, dev))
    run_batch(s, counts, hidden={6: [(48, 64)], 0: [(1600, 1616)]})


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(16, 2, 128), (4, 1, 256), (6, 2, 192), (8, 2, 64)], ids=str)
def test_many_short_prompts(dev, shape, dtype):
    """more sequences than a wave has lanes, of more rows than single tokens; parts that are joined"""
    lens = [40 + (29 * i) % 90 for i in range(100)] + [2000, 0, 1]
    counts = [20 + i % 21 for i in range(100)] + [70, 0, 1]
    s = Setup(dev, shape, dtype, 16, lens, seed=22)
    run_batch(s, counts)


@pytest.mark.parametrize("n", [64, 65, 1024, 1025, 5000])
def test_numbers_of_sequences(dev, n):
    """single tokens of n sequences of a few rows, a long one among them, some without new rows"""
    lens = [i % 7 for i in range(n)]
    lens[n // 3] = 1500
    s = Setup(dev, (4, 2, 64), torch.bfloat16, 4, lens, seed=n)
    run_batch(s, [1 if m and i % 11 else 0 for i, m in enumerate(lens)])
    run_batch(s, [min(m, 70) for m in lens], grouped=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape", [(16, 2, 128), (4, 1, 256), (6, 2, 192), (8, 2, 64), (40, 1, 128)], ids=str)
@pytest.mark.parametrize("lens,counts", [([15000], [1]), ([15000, 3], [2, 0]), ([5000, 300, 2, 4100] * 4, [1, 1, 1, 1] * 4),
                                         ([6000, 2500, 40, 0], [4, 1, 3, 1])], ids=["one", "one_of_two", "sixteen", "ragged"])
def test_single_tokens_of_long_sequences(dev, shape, lens, counts, dtype):
    s = Setup(dev, shape, dtype, 32, lens, seed=23)
    run_batch(s, counts)
    run_batch(s, counts, window=2100, sinks=3)


def test_the_largest_number_of_units(dev):
    """16 776 960 workgroups: single tokens of 65535 sequences with one row, on 256 kv heads; one more is refused"""
    pkg = load_pkg()
    n, kvh, hd = 65536, 256, 64
    k, v = (torch.randn(1, 2, 1, kvh, hd, device=dev).bfloat16() for _ in range(2))
    cache = pkg.PagedCache(k, v, (torch.arange(n, device=dev).int() % 2)[:, None].contiguous(), torch.ones(n, dtype=torch.int32, device=dev),
                           i32([n // 2] * 2, dev))
    q = torch.ones(1, kvh, hd, dtype=torch.bfloat16, device=dev).expand(n, kvh, hd)
    starts = torch.arange(n + 1, device=dev).int()
    with pytest.raises(pkg.QmoeError, match="more work"):
        cache.attend(0, q, starts)
    out = cache.attend(0, q[:-1], starts[:-1])
    assert torch.equal(out[0::2], v[0, 0].expand(n // 2, kvh, hd)) and torch.equal(out[1::2], v[0, 1].expand(n // 2 - 1, kvh, hd))


def test_forks_of_large_tables(dev):
    """tables of 60 x 250 entries: sources shared, swapped and cut, refusals, against the tables before"""
    pkg = load_pkg()
    slots, width, page = 60, 250, 4
    c = pkg.PagedCache.allocate(1, 6000, page, 1, 64, slots, width, torch.bfloat16, dev)
    rng = np.random.RandomState(24)
    lens = rng.randint(0, 300, slots).tolist()
    assert int(c.reserve(i32(lens, dev))) == 0
    t, n = c.table.cpu(), c.lens.cpu()
    dst = rng.permutation(slots).tolist()
    src = rng.randint(0, slots, slots).tolist()
    rows = rng.randint(-1, 400, slots).tolist()
    for bad in ([dst[1]] + dst[1:], [-1] + dst[1:], [slots] + dst[1:]):
        assert int(c.fork(i32(src, dev), i32(bad, dev))) == -1
    assert int(c.fork(i32([slots] + src[1:], dev), i32(dst, dev))) == -1
    assert torch.equal(c.table.cpu(), t) and torch.equal(c.lens.cpu(), n)
    assert int(c.fork(i32(src, dev), i32(dst, dev), i32(rows, dev))) == 0
    for a, b, r in zip(src, dst, rows):
        m = min(max(r, 0), int(n[a]))
        e = -(-m // page)
        assert int(c.lens[b]) == m
        assert torch.equal(c.table[b].cpu(), torch.cat([t[a, :e], torch.full((width - e,), -1, dtype=torch.int32)]))
    held = c.table.cpu()[c.table.cpu() >= 0].long()
    assert torch.equal(c.refs.cpu().long(), torch.bincount(held, minlength=6000))


def test_numbers_that_c_would_read_differently_are_refused(dev):
    s = Setup(dev, HEADS[2], torch.float32, 8, [20])
    q, starts = s.queries([2])
    q, starts, error = q.to(dev), i32(starts, dev), load_pkg().QmoeError
    with pytest.raises(error, match="scale"):
        s.cache.attend(0, q, starts, scale=0.0)
    for kw in (dict(window=2 ** 32 + 5), dict(window=-1), dict(window=4, sinks=2 ** 32)):
        with pytest.raises(error, match="window"):
            s.cache.attend(0, q, starts, **kw)
    with pytest.raises(error, match="window"):
        s.cache.evict(2 ** 32 + 5)
    assert s.table.tolist() == s.rows


def test_layers_and_rows_that_c_would_cut_off_are_refused(dev):
    s = Setup(dev, HEADS[2], torch.float32, 8, [20], layers=2)
    q, starts = s.queries([2])
    q, starts, error = q.to(dev), i32(starts, dev), load_pkg().QmoeError
    new = torch.zeros(2, 2, 64, device=dev)
    before = s.k.clone()
    for layer in (2 ** 32, 2 ** 32 + 1, -2 ** 32, -1, 2):
        with pytest.raises(error, match="layer"):
            s.cache.attend(layer, q, starts)
        with pytest.raises(error, match="layer"):
            s.cache.append(layer, new, new, starts)
    # broadcast rows, which take no memory: 2^32 + 2 of them would be read as 2
    with pytest.raises(error, match="below 2\\^31"):
        s.cache.append(0, new[:1].expand(2 ** 32 + 2, 2, 64), new[:1].expand(2 ** 32 + 2, 2, 64), starts)
    with pytest.raises(error, match="below 2\\^31"):
        s.cache.attend(0, q[:1].expand(2 ** 32 + 2, 4, 64), starts, out=q)
    assert torch.equal(s.k, before)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n", [90, 400])
def test_starts_in_no_order_stay_inside(dev, n, dtype):
    """100 sequences whose starts descend, overlap and leave [0, n), slots out of range, lengths past the table:
    only rows that some sequence claims are written"""
    s = Setup(dev, HEADS[0], dtype, 16, [int(x) for x in np.random.RandomState(n).randint(0, 700, 20)], seed=n)
    rng = np.random.RandomState(n + 1)
    for _ in range(3):
        starts = rng.randint(-50, n + 50, 101)
        slots = rng.randint(-2, 23, 100).tolist()
        s.len_t.copy_(i32(rng.randint(-100, 3000, 20).tolist(), dev))
        claimed = np.zeros(n, dtype=bool)
        for a, b in zip(starts[:-1], starts[1:]):
            claimed[max(a, 0):max(min(b, n), 0)] = True
        guard = torch.full((n + 64, s.h, s.hd), 7.0, dtype=dtype, device=dev)
        q = torch.randn(n, s.h, s.hd, generator=s.g).to(dtype).to(dev)
        s.cache.attend(0, q, i32(starts.tolist(), dev), i32(slots, dev), out=guard[32:32 + n])
        assert (guard[:32] == 7).all() and (guard[32 + n:] == 7).all()
        assert (guard[32:32 + n].cpu()[~torch.from_numpy(claimed)] == 7).all()


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_tiny_scales(dev, dtype):
    """the smallest that f32 holds weigh all visible rows alike; smaller ones are refused, not taken for the default"""
    s = Setup(dev, HEADS[0], dtype, 16, [300, 77], seed=31)
    for counts in ([1, 2], [200, 70]):
        run_batch(s, counts, scale=2.0 ** -149)
        run_batch(s, counts, scale=-2.0 ** -148, window=33, sinks=2)
        q, starts = s.queries(counts)
        for bad in (1e-46, -1e-46, 1e-300):
            with pytest.raises(load_pkg().QmoeError, match="scale"):
                s.cache.attend(0, q.to(dev), i32(starts, dev), scale=bad)


@pytest.mark.parametrize("hd", [64, 128, 192, 256])
def test_weights_of_few_rows_have_16_bits(dev, hd, monkeypatch):
    """bf16 calls of 16 and 32 rows a unit.  A weight is taken as bf16(w) + bf16(w - bf16(w)): the first is off by
    2^-8 w at the most, the second by 2^-8 of that, so the sum of w v is off by 2^-16 A beside the fp32 terms of the
    bar above.  A small scale keeps those small (B is below 1), and sums that nearly cancel show the weights' error,
    which rounding the weights to bf16 makes 2^-9 A / sqrt(keys) and more."""
    for table_rows, counts in ((0, [1, 1, 1]), (1 << 18, [3, 4, 3])):
        monkeypatch.setattr(Setup, "table_rows", table_rows)
        s = Setup(dev, (8, 1, hd), torch.bfloat16, 16, [20, 33, 60], seed=33)
        q, starts = s.queries(counts)
        out = s.cache.attend(0, q.to(dev), i32(starts, dev), scale=0.02 * hd ** -0.5).double().cpu()
        for i, c in enumerate(counts):
            T = s.lens[i]
            want, A, B = reference(q[starts[i]:starts[i + 1]], s.hk[i], s.hv[i], c, 0, 0, False, 0.02 * hd ** -0.5)
            assert float(B.max()) < 1
            tol = A * (2 * (hd + 24) * U * (B + 1) + 2 * (T + 64) * U + 2.0 ** -16) + want.abs() * 2.0 ** -8
            err = (out[starts[i]:starts[i + 1]] - want).abs()
            assert (err <= tol).all(), (i, T, float((err / tol).max()))


@pytest.mark.usefixtures("tables")
def test_slots_in_any_order_twice_and_out_of_range(dev):
    s = Setup(dev, HEADS[0], torch.bfloat16, 16, [100, 40, 77, 260], seed=3)
    run_batch(s, [1, 6, 1, 30, 2], slots=[2, 0, 2, 3, 0])
    q, starts = s.queries([3, 2, 4])
    out = s.cache.attend(0, q.to(dev), i32(starts, dev), i32([1, -1, 4], dev))
    want, A, B = reference(q[:3], s.hk[1], s.hv[1], 3, 0, 0, False)
    check(out[:3], want, A, B, s.hd, 40, s.dtype, "slot 1")
    assert (out[3:] == 0).all()


def test_scale_and_layer(dev):
    s = Setup(dev, HEADS[2], torch.float32, 16, [50, 90], layers=3, seed=4)
    run_batch(s, [5, 2], scale=0.5, layer=2)
    run_batch(s, [5, 2], scale=-0.25, layer=2)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 33, 90]], ids=["tokens", "chunks"])
def test_released_and_bad_pages_are_not_seen(dev, counts, dtype):
    s = Setup(dev, HEADS[0], dtype, 16, [100, 130, 90], seed=5)
    s.rows[0][2] = -1
    s.rows[0][3] = s.k.shape[1]
    s.rows[1] = [-5, 2 ** 31 - 1, -2 ** 31] + s.rows[1][3:]
    s.rows[2] = [-1] * len(s.rows[2])  # nothing left: zeros
    s.table.copy_(i32(s.rows, dev))
    hidden = {0: [(32, 64)], 1: [(0, 48)], 2: [(0, 90)]}
    run_batch(s, counts, hidden=hidden)
    run_batch(s, counts, window=50, sinks=20, hidden=hidden)


def test_lengths_and_starts_out_of_range_are_clamped(dev):
    s = Setup(dev, HEADS[2], torch.float32, 8, [20, 30, 16], seed=6)
    cap = s.table.shape[1] * 8
    # a length past the table counts as the table's rows; a negative one as none
    s.len_t.copy_(i32([10 ** 9, -7, 16], dev))
    q, starts = s.queries([2, 3, 1])
    out = s.cache.attend(0, q.to(dev), i32(starts, dev))
    pad = torch.zeros(cap - 20, s.kvh, s.hd)
    want, A, B = reference(q[:2], torch.cat([s.hk[0], pad]), torch.cat([s.hv[0], pad]), 2, 0, 0, False,
                           hidden=[(-(-20 // 8) * 8, cap)])
    check(out[:2], want, A, B, s.hd, cap, s.dtype, "long")  # rows 20..23 of the last page hold zeros
    assert (out[2:5] == 0).all()
    # starts past n, descending, negative: no row outside [0, n) is touched
    guard = torch.full((8, s.h, s.hd), 7.0, device=dev)
    s.len_t.copy_(i32([20, 30, 16], dev))
    s.cache.attend(0, q.to(dev), i32([-3, 2, 1, 50], dev), out=guard[1:7])
    assert (guard[0] == 7).all() and (guard[7] == 7).all()


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_rows_of_no_sequence_are_left_alone(dev, dtype):
    s = Setup(dev, HEADS[0], dtype, 16, [100, 30], seed=7)
    for counts in ([1, 1], [20, 30]):
        q, starts = s.queries([3] + counts + [6])
        out = torch.full(q.shape, 5.0, dtype=dtype, device=dev)
        s.cache.attend(0, q.to(dev), i32(starts[1:4], dev), out=out)
        assert (out[:3] == 5).all() and (out[starts[3]:] == 5).all()
        for i, c in enumerate(counts):
            want, A, B = reference(q[starts[i + 1]:starts[i + 2]], s.hk[i], s.hv[i], c, 0, 0, False)
            check(out[starts[i + 1]:starts[i + 2]], want, A, B, s.hd, 100, dtype, i)


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -3e38])
@pytest.mark.parametrize("counts", [[1, 4, 1], [33, 80, 64]], ids=["tokens", "chunks"])
def test_what_unseen_rows_hold_does_not_matter(dev, counts, junk, dtype):
    """unused rows of pages, free pages, rows after the query, rows behind the window"""
    lens = [45, 100, 97]
    clean, dirty = (Setup(dev, HEADS[0], dtype, 16, lens, seed=8, junk=j) for j in (0.0, junk))
    q, starts = clean.queries(counts)
    q, st = q.to(dev), i32(starts, dev)
    for window, sinks in ((0, 0), (20, 3)):
        a = clean.cache.attend(0, q, st, window=window, sinks=sinks)
        b = dirty.cache.attend(0, q, st, window=window, sinks=sinks)
        assert torch.equal(a, b) and torch.isfinite(a).all()
    # the last cached row holds junk: every query but the last one's is as before
    for c in (clean, dirty):
        for i, n in enumerate(lens):
            c.v[0, c.rows[i][(n - 1) // 16], (n - 1) % 16] = junk if c is dirty else 0.0
    a, b = (c.cache.attend(0, q, st) for c in (clean, dirty))
    for i in range(len(lens)):
        x, y = a[starts[i]:starts[i + 1]].double().cpu(), b[starts[i]:starts[i + 1]].double().cpu()
        want, A, B = reference(q[starts[i]:starts[i + 1]].cpu(), clean.hk[i], torch.cat([clean.hv[i][:-1], 0 * clean.hv[i][-1:]]),
                               counts[i], 0, 0, False)
        check(x, want, A, B, 128, 100, dtype, i)
        check(y[:-1], want[:-1], A[:-1], B[:-1], 128, 100, dtype, (i, "junk behind"))
        if junk != junk:
            assert torch.isnan(y[-1]).all()
        elif junk > 1e38:
            assert torch.isinf(y[-1]).all() or torch.isnan(y[-1]).any()
    # a row behind the window holds junk in k and v: only queries that see it are touched
    w = 20
    for i, n in enumerate(lens):
        for c in (clean, dirty):
            fix = clean.hv[i][n - 1].to(dev)
            c.v[0, c.rows[i][(n - 1) // 16], (n - 1) % 16] = fix
        j = 10
        dirty.k[0, dirty.rows[i][j // 16], j % 16] = junk
        dirty.v[0, dirty.rows[i][j // 16], j % 16] = junk
    a, b = (c.cache.attend(0, q, st, window=w, sinks=2) for c in (clean, dirty))
    for i, n in enumerate(lens):
        pos = torch.arange(n - counts[i], n)
        blind = (pos < 10) | (pos - 10 >= w)
        x, y = (t[starts[i]:starts[i + 1]].double().cpu()[blind] for t in (a, b))
        want, A, B = reference(q[starts[i]:starts[i + 1]].cpu(), clean.hk[i], clean.hv[i], counts[i], w, 2, False)
        check(x, want[blind], A[blind], B[blind], 128, 100, dtype, i)
        check(y, want[blind], A[blind], B[blind], 128, 100, dtype, (i, "junk"))


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("counts", [[1, 1], [40, 50]], ids=["tokens", "chunks"])
def test_infinite_scores_follow_the_formula(dev, counts, dtype):
    """scores of -inf weigh nothing beside finite ones; only -inf, or +inf, gives NaN, as exp(x - max) / sum does"""
    s = Setup(dev, HEADS[0], dtype, 16, [60, 70], seed=9)
    q, starts = s.queries(counts)
    q = q.abs() + 0.1
    s.k[0, s.rows[0][1], 4] = -torch.inf  # key 20 of sequence 0
    for p in s.rows[1]:
        if p >= 0:
            s.k[0, p] = -torch.inf  # every key of sequence 1
    out = s.cache.attend(0, q.to(dev), i32(starts, dev)).double().cpu()
    want, A, B = reference(q[:counts[0]], s.hk[0], s.hv[0], counts[0], 0, 0, False, hidden=[(20, 21)])
    pos = torch.arange(60 - counts[0], 60)
    check(out[:counts[0]], want, A, B, 128, 60, dtype, "one -inf")
    assert torch.isnan(out[counts[0]:]).all()
    s.k[0, s.rows[0][1], 4] = torch.inf
    out = s.cache.attend(0, q.to(dev), i32(starts, dev)).double().cpu()
    assert torch.isnan(out[:counts[0]][pos >= 20]).all()
    check(out[:counts[0]][pos < 20], want[pos < 20], A[pos < 20], B[pos < 20], 128, 60, dtype, "before +inf")


@pytest.mark.usefixtures("tables")
def test_large_scores(dev):
    """scores of hundreds: the running maximum is subtracted before exp"""
    for dtype in (torch.bfloat16, torch.float32):
        s = Setup(dev, HEADS[2], dtype, 16, [300, 130], seed=10)
        s.k.mul_(30)
        s.hk = [x * 30 for x in s.hk]
        if dtype == torch.bfloat16:  # the pages' own rounding
            s.hk = [x.to(dtype) for x in s.hk]
        run_batch(s, [1, 1])
        run_batch(s, [90, 130])


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("sign", [1, -1], ids=["positive", "negative"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("shape,lens,counts", [((4, 2, 64), [40, 33, 200], [1, 3, 5]), ((16, 2, 128), [300, 170], [250, 130]),
                                               ((4, 1, 256), [90, 300], [60, 200]), ((4, 2, 64), [9000], [2]),
                                               ((16, 2, 128), [4000, 100], [300, 1]), ((6, 2, 192), [60] * 70, [1] * 70)],
                         ids=["few", "many", "many_256", "few_joined", "many_joined", "indexed"])
def test_scores_past_what_fp32_resolves(dev, shape, lens, counts, dtype, sign):
    """scores of 2^34 and more, of both signs, whose steps in fp32 are far wider than exp's range.  One key's score is
    at least twice as large (or half as negative) as any other's, so in 64 bits its weight is 1 and all others are 0:
    the output is its v, with the sums' and the output's roundings."""
    s = Setup(dev, shape, dtype, 16, lens, seed=27)
    h, kvh, hd = shape
    g = torch.Generator().manual_seed(28)
    starts = s.queries(counts)[1]
    u = (torch.randint(0, 2, (kvh, hd), generator=g) * 2 - 1).float()
    wins = [(n - c) // 2 for n, c in zip(lens, counts)]
    for i, n in enumerate(lens):
        rest = torch.rand(n, kvh, 1, generator=g) * 0.4
        a = (0.1 + rest) if sign > 0 else (2.1 + 4 * rest)
        a[wins[i]] = 1.0
        a = a * (2.0 ** 16 * (1 + torch.rand(1, kvh, 1, generator=g)))
        k = (a * u).to(dtype).to(dev)
        for j0 in range(0, n, 16):
            m = min(16, n - j0)
            s.k[0, s.rows[i][j0 // 16], :m] = k[j0:j0 + m]
    # one factor for all rows of a call, so that the fp32 rounding of the largest score, up or down, is the same in
    # all rows of a unit
    for draw in range(8):
        q = (2.0 ** 16 * (1 + torch.rand(1, generator=g)) * u[torch.arange(h) % kvh]).to(dtype).expand(starts[-1], h, hd)
        out = s.cache.attend(0, q.to(dev), i32(starts, dev), scale=sign * hd ** -0.5).double().cpu()
        for i, n in enumerate(lens):
            want = s.hv[i][wins[i]].double()[torch.arange(h) % kvh][None]
            err = (out[starts[i]:starts[i + 1]] - want).abs()
            tol = want.abs() * (2 * (n + 64) * U + torch.finfo(dtype).eps / 2)
            assert (err <= tol).all(), (draw, i, int((~(err <= tol)).sum()))


@pytest.mark.usefixtures("tables")
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_strides(dev, dtype):
    """heads before rows in the pages, heads before tokens in q and out, k and v interleaved"""
    lens, counts = [100, 33], [30, 1]
    s = Setup(dev, HEADS[0], dtype, 16, lens, seed=11, order="heads")
    run_batch(s, counts)
    q, starts = s.queries(counts)
    qt = q.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    big = torch.full((16, 40, 3, 128), 9.0, dtype=dtype, device=dev)
    out = big[:, 4:35, 1].transpose(0, 1)
    s.cache.attend(0, qt, i32(starts, dev), out=out)
    same = s.cache.attend(0, q.to(dev), i32(starts, dev))
    assert torch.equal(out, same)
    assert (big[:, :4] == 9).all() and (big[:, 35:] == 9).all() and (big[:, :, 0] == 9).all() and (big[:, :, 2] == 9).all()
    pool = torch.stack([s.k, s.v], 2)  # [1, pages, 2, rows, heads, dim]
    both = load_pkg().PagedCache(pool[:, :, 0], pool[:, :, 1], s.full, s.len_t, s.refs)
    assert torch.equal(both.attend(0, q.to(dev), i32(starts, dev)), same)
    # a broadcast query
    one = torch.randn(1, 16, 128, generator=s.g).to(dtype).to(dev)
    assert torch.equal(s.cache.attend(0, one.expand(31, 16, 128), i32(starts, dev)),
                       s.cache.attend(0, one.expand(31, 16, 128).contiguous(), i32(starts, dev)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_offsets_past_32_bits(dev, dtype):
    """a pool of more than 2^32 bytes and 2^31 elements, the sequence's pages at both ends"""
    kvh, hd, page = 2, 128, 64
    n_pages = (2 ** 31 + 2 ** 28) // (page * kvh * hd)
    k, v = (torch.empty(1, n_pages, page, kvh, hd, dtype=dtype, device=dev) for _ in range(2))
    ids = [n_pages - 1, 0, n_pages - 2, n_pages // 2]
    g = torch.Generator().manual_seed(12)
    T = 230
    hk, hv = (torch.randn(T, kvh, hd, generator=g).to(dtype) for _ in range(2))
    pkg = load_pkg()
    cache = pkg.PagedCache(k, v, i32([ids], dev), i32([T], dev), torch.zeros(n_pages, dtype=torch.int32, device=dev))
    cache.append(0, hk.to(dev), hv.to(dev), i32([0, T], dev))
    wide = torch.full((1, 1 << 14), -1, dtype=torch.int32, device=dev)
    wide[0, :4] = i32(ids, dev)
    for c, table in ((1, cache.table), (100, cache.table), (100, wide)):
        cache = pkg.PagedCache(k, v, table, cache.lens, cache.refs)
        q = torch.randn(c, 16, hd, generator=g).to(dtype)
        out = cache.attend(0, q.to(dev), i32([0, c], dev))
        want, A, B = reference(q, hk, hv, c, 0, 0, False)
        check(out, want, A, B, hd, T, dtype, c)


@pytest.mark.usefixtures("tables")
def test_results_repeat_to_the_bit(dev):
    for dtype in (torch.bfloat16, torch.float32):
        s = Setup(dev, HEADS[0], dtype, 16, [3000, 100, 777], seed=13)
        for counts in ([1, 1, 1], [60, 100, 300]):
            q, starts = s.queries(counts)
            q, st = q.to(dev), i32(starts, dev)
            a = s.cache.attend(0, q, st)
            for _ in range(3):
                assert torch.equal(a, s.cache.attend(0, q, st))


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("src,dst", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                     (torch.float32, torch.bfloat16)], ids=["bf16", "f32", "f32_to_bf16"])
@pytest.mark.parametrize("page", [1, 16, 21])
def test_append(dev, src, dst, page):
    lens = [1, 50, 0, 33, 200, 16, 17]
    counts = [1, 50, 0, 1, 37, 16, 3]
    for shape, order in ((0, "rows"), (1, "heads"), (4, "rows")):
        s = Setup(dev, HEADS[shape], dst, page, lens, seed=page, layers=2, junk=3.0, order=order)
        s.rows[4][170 // page] = -1  # a released page: its rows are not written
        s.table.copy_(i32(s.rows, dev))
        n = sum(counts)
        starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
        new = [torch.randn(n + 2, s.kvh, s.hd, generator=s.g).to(src) for _ in range(2)]
        want = [s.k.clone(), s.v.clone()]
        for i, c in enumerate(counts):
            for r in range(c):
                j = lens[i] - c + r
                if s.rows[i][j // page] >= 0:
                    for w, x in zip(want, new):
                        w[0, s.rows[i][j // page], j % page] = x[starts[i] + r].to(dst).to(dev)
        s.cache.append(0, new[0].to(dev), new[1].to(dev), i32(starts, dev))  # two rows of no sequence
        assert torch.equal(s.k, want[0]) and torch.equal(s.v, want[1])


def test_append_skips_rows_before_the_first_and_slots_out_of_range(dev):
    s = Setup(dev, HEADS[2], torch.float32, 8, [3, 9], seed=14)
    before = s.k.clone()
    x = torch.ones(9, 2, 64, device=dev)
    s.cache.append(0, x, x, i32([0, 5, 7, 9], dev), i32([0, 2, -1], dev))
    before[0, s.rows[0][0], :3] = 1.0
    assert torch.equal(s.k, before)


def test_append_strided_rows(dev):
    s = Setup(dev, HEADS[2], torch.bfloat16, 8, [20, 12], seed=15)
    x = torch.randn(2, 9, 3, 64, dtype=torch.bfloat16, device=dev)
    k, v = x[:, :, 0].transpose(0, 1), x[:, :, 2].transpose(0, 1)
    s.cache.append(0, k, v, i32([0, 4, 9], dev))
    for i, (a, b, n) in enumerate(((0, 4, 20), (4, 9, 12))):
        for t in range(a, b):
            j = n - (b - t)
            assert torch.equal(s.k[0, s.rows[i][j // 8], j % 8], k[t]) and torch.equal(s.v[0, s.rows[i][j // 8], j % 8], v[t])


# ---------------------------------------------------------------- pages

class Model:
    """the pages' bookkeeping in Python, with every row's contents as a number"""

    def __init__(self, n_pages, page, slots, width):
        self.page, self.width = page, width
        self.table = [[-1] * width for _ in range(slots)]
        self.lens, self.refs = [0] * slots, [0] * n_pages
        self.data = [[0.0] * page for _ in range(n_pages)]

    def pages(self, n):
        return -(-n // self.page)

    def reserve(self, slots, n_new):
        if len(set(slots)) < len(slots):
            return -1
        need = []
        for s, a in zip(slots, n_new):
            if not 0 <= s < len(self.lens) or a < 0 or self.lens[s] + a > self.width * self.page:
                return -1
            if self.lens[s] % self.page and a and self.table[s][self.lens[s] // self.page] < 0:
                return -1
        refs = list(self.refs)
        takes = []
        for s, a in zip(slots, n_new):
            n = self.lens[s]
            if n % self.page and a:
                p = self.table[s][n // self.page]
                if refs[p] > 1:
                    refs[p] -= 1
                    takes.append((s, n // self.page, p))
            takes += [(s, e, -1) for e in range(self.pages(n), self.pages(n + a))]
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if len(takes) > len(free):
            return len(takes) - len(free)
        for (s, e, old), p in zip(takes, free):
            if old >= 0:
                self.refs[old] -= 1
                self.data[p] = list(self.data[old])
            self.table[s][e] = p
            self.refs[p] = 1
        for s, a in zip(slots, n_new):
            self.lens[s] += a
        return 0

    def fork(self, src, dst, rows=None):
        S = len(self.lens)
        if len(set(dst)) < len(dst) or any(not 0 <= x < S for x in src + dst):
            return -1
        new = []
        for i, s in enumerate(src):
            n = self.lens[s] if rows is None else min(max(rows[i], 0), self.lens[s])
            new.append((n, self.table[s][:self.pages(n)] + [-1] * (self.width - self.pages(n))))
        for _, r in new:
            for p in r:
                if p >= 0:
                    self.refs[p] += 1
        for d, (n, r) in zip(dst, new):
            for p in self.table[d]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[d], self.lens[d] = r, n
        return 0

    def evict(self, slots, window, sinks):
        for s in slots:
            for e, p in enumerate(self.table[s]):
                if p >= 0 and e * self.page >= sinks and (e + 1) * self.page <= self.lens[s] - window + 1:
                    self.table[s][e] = -1
                    self.refs[p] -= 1

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] == 0]
        high = [p for p in range(used, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(high, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a], self.data[b] = self.refs[a], 0, list(self.data[a])
        self.table = [[to.get(p, p) for p in r] for r in self.table]
        return used

    def append(self, slot, c, values):
        for r in range(c):
            j = self.lens[slot] - c + r
            p = self.table[slot][j // self.page]
            if p >= 0:
                self.data[p][j % self.page] = values[r]


def same_state(cache, m, what):
    assert cache.table.tolist() == m.table, (what, "table")
    assert cache.lens.tolist() == m.lens, (what, "lens")
    assert cache.refs.tolist() == m.refs, (what, "refs")


@pytest.mark.parametrize("n_pages,page,slots,width,seed", [(40, 4, 6, 9, 0), (300, 16, 20, 12, 1), (5000, 3, 70, 40, 2),
                                                           (64, 1, 9, 11, 3), (700, 24, 33, 15, 4)])
def test_random_steps(dev, n_pages, page, slots, width, seed):
    """reserve, append, fork, trim, evict and compact at random against the model; refused calls change nothing"""
    rng = np.random.RandomState(seed)
    pkg = load_pkg()
    cache = pkg.PagedCache.allocate(2, n_pages, page, 1, 64, slots, width, torch.float32, dev)
    cache.k.zero_()
    cache.v.zero_()
    m = Model(n_pages, page, slots, width)
    mark = 1.0
    refused = 0
    for step in range(60):
        what = rng.choice(["reserve", "reserve", "reserve", "fork", "fork", "trim", "evict", "compact"])
        if what == "reserve":
            sl = rng.choice(slots, rng.randint(1, slots + 1), replace=False).tolist()
            add = [int(x) for x in rng.randint(0, 3 * page + 1, len(sl))]
            if rng.rand() < 0.1:
                sl[0] = int(rng.choice([-1, slots, sl[-1]])) if len(sl) > 1 else -1
            got, want = int(cache.reserve(i32(add, dev), i32(sl, dev))), m.reserve(sl, add)
            assert got == want, (step, got, want)
            if want == 0 and sum(add):
                starts = np.concatenate([[0], np.cumsum(add)]).tolist()
                vals = np.arange(sum(add), dtype=np.float32) + mark
                mark += sum(add)
                x = torch.from_numpy(vals).to(dev)[:, None, None].expand(-1, 1, 64).contiguous()
                for layer in range(2):
                    cache.append(layer, x + layer, -x - layer, i32(starts, dev), i32(sl, dev))
                for i, s in enumerate(sl):
                    m.append(s, add[i], vals[starts[i]:starts[i + 1]].tolist())
            refused += want != 0
        elif what in ("fork", "trim"):
            n = rng.randint(1, slots + 1)
            dst = rng.choice(slots, n, replace=False).tolist()
            src = dst if what == "trim" else rng.randint(0, slots, n).tolist()
            rows = [int(x) for x in rng.randint(-2, width * page, n)] if what == "trim" or rng.rand() < 0.5 else None
            if rng.rand() < 0.1 and n > 1:
                dst = [dst[1]] + dst[1:]
                src = dst if what == "trim" else src
            rt = None if rows is None else i32(rows, dev)
            got = int(cache.trim(i32(dst, dev), rt) if what == "trim" else cache.fork(i32(src, dev), i32(dst, dev), rt))
            assert got == m.fork(src, dst, rows), step
        elif what == "evict":
            w, sk = int(rng.randint(1, width * page)), int(rng.randint(0, 3 * page))
            if rng.rand() < 0.5:
                cache.evict(w, sk)
                m.evict(range(slots), w, sk)
            else:
                sl = rng.choice(slots, rng.randint(1, slots)).tolist()  # some named twice
                cache.evict(w, sk, i32(sl + [-1, slots], dev))
                m.evict(sl, w, sk)
        else:
            assert int(cache.compact()) == m.compact()
        same_state(cache, m, (step, what))
    assert refused > 0 or n_pages > 4000
    k, v = cache.k[:, :, :, 0], cache.v[:, :, :, 0]
    for s in range(slots):
        for j in range(m.lens[s]):
            p = m.table[s][j // page]
            if p >= 0:
                want = m.data[p][j % page]
                for layer in range(2):
                    assert (k[layer, p, j % page] == want + layer).all() and (v[layer, p, j % page] == -want - layer).all(), (s, j)


def test_reserve_refusals_change_nothing(dev):
    pkg = load_pkg()
    c = pkg.PagedCache.allocate(1, 10, 4, 1, 64, 5, 6, torch.float32, dev)
    assert int(c.reserve(i32([10, 3, 5], dev))) == 0  # 3 + 1 + 2 pages
    state = [t.clone() for t in (c.table, c.lens, c.refs)]
    for n_new, slots, want in (([20], [3], 1), ([24, 24, 24], [1, 3, 4], 13), ([1, 1], [3, 3], -1), ([1], [5], -1),
                               ([1], [-1], -1), ([-1], [0], -1), ([25], [3], -1), ([2 ** 31 - 1], [0], -1), ([15], [0], -1)):
        if want == 13:
            n_new = [21, 24, 24]
        got = int(c.reserve(i32(n_new, dev), i32(slots, dev)))
        assert got == want, (n_new, slots, got)
        assert all(torch.equal(a, b) for a, b in zip(state, (c.table, c.lens, c.refs)))
    assert int(c.reserve(i32([], dev), i32([], dev))) == 0 and int(c.fork(i32([], dev), i32([], dev))) == 0
    assert int(c.reserve(i32([0, 0, 0, 0, 16], dev))) == 0 and int(c.lens[4]) == 16
    assert int(c.reserve(i32([1, 1, 0, 0, 0], dev))) == 0  # rows left in last pages: no page is taken
    # a released partly filled last page is an error of the caller's
    c.table[0, 2] = -1  # rows 8..10 of 11
    assert int(c.reserve(i32([1], dev), i32([0], dev))) == -1


def test_needs_past_the_pool_are_refused_whatever_their_size(dev):
    """tables longer than the pool, every page free: the pages lacking are exact, and nothing changes"""
    pkg = load_pkg()
    c = pkg.PagedCache.allocate(1, 10, 1, 1, 64, 4, 1000, torch.float32, dev)
    state = [t.clone() for t in (c.table, c.lens, c.refs)]
    for n_new, slots, want in (([500], [0], 490), ([0, 500], [1, 0], 490), ([500, 0], [1, 0], 490), ([11], [3], 1),
                               ([1000] * 4, [3, 1, 0, 2], 3990), ([5, 5, 1], [0, 1, 2], 1), ([10, 1], [0, 1], 1)):
        assert int(c.reserve(i32(n_new, dev), i32(slots, dev))) == want, (n_new, slots)
        assert all(torch.equal(a, b) for a, b in zip(state, (c.table, c.lens, c.refs)))
    assert int(c.reserve(i32([0, 4, 0, 6], dev))) == 0
    assert c.lens.tolist() == [0, 4, 0, 6] and c.table[1, :5].tolist() == [0, 1, 2, 3, -1] and int(c.refs.sum()) == 10
    assert int(c.reserve(i32([500, 20], dev), i32([0, 1], dev))) == 520
    # a shared partly filled page whose copy is one page more; then lacks of more than 31 bits
    c = pkg.PagedCache.allocate(1, 3, 4, 1, 64, 3, 1000, torch.float32, dev)
    assert int(c.reserve(i32([6], dev), i32([0], dev))) == 0 and int(c.fork(i32([0], dev), i32([1], dev))) == 0
    assert int(c.reserve(i32([4000 - 6], dev), i32([1], dev))) == 998  # 998 pages and the copy, one page free
    big = pkg.PagedCache.allocate(1, 10, 1, 1, 64, 3, 1 << 30, torch.bfloat16, dev)
    assert int(big.reserve(i32([1 << 30], dev), i32([2], dev))) == (1 << 30) - 10
    assert int(big.reserve(i32([1 << 30, 1 << 30, 1 << 30], dev))) == 2 ** 31 - 1
    assert big.lens.tolist() == [0, 0, 0] and int(big.refs.sum()) == 0 and int(big.table[:, :20].max()) == -1


def test_the_last_writer_keeps_a_shared_page(dev):
    pkg = load_pkg()
    c = pkg.PagedCache.allocate(1, 12, 8, 1, 64, 5, 4, torch.float32, dev)
    assert int(c.reserve(i32([5], dev), i32([0], dev))) == 0
    assert int(c.fork(i32([0, 0], dev), i32([1, 2], dev))) == 0
    assert c.refs.tolist()[:2] == [3, 0]
    assert int(c.reserve(i32([1, 1, 0], dev), i32([2, 0, 1], dev))) == 0  # 1 still holds it: both copy
    assert c.table[:3, 0].tolist() == [2, 0, 1] and c.refs.tolist()[:3] == [1, 1, 1]
    assert int(c.fork(i32([0, 0], dev), i32([1, 2], dev))) == 0
    assert int(c.reserve(i32([1, 1, 1], dev), i32([1, 2, 0], dev))) == 0  # all write: slot 0, the last, keeps page 2
    assert c.table[:3, 0].tolist() == [2, 0, 1] and c.refs.tolist()[:3] == [1, 1, 1]


def test_beams_trade_places(dev):
    pkg = load_pkg()
    c = pkg.PagedCache.allocate(1, 20, 4, 1, 64, 4, 5, torch.float32, dev)
    assert int(c.reserve(i32([9, 4, 13, 1], dev))) == 0
    t, n = c.table.clone(), c.lens.clone()
    parents = [3, 2, 0, 0]
    assert int(c.fork(i32(parents, dev), i32([0, 1, 2, 3], dev))) == 0
    assert torch.equal(c.table, t[parents]) and torch.equal(c.lens, n[parents])
    want = torch.zeros(20, dtype=torch.int32)
    for p in c.table.flatten().tolist():
        if p >= 0:
            want[p] += 1
    assert torch.equal(c.refs.cpu(), want)


@pytest.mark.parametrize("page,window,sinks,ahead", [(4, 9, 0, 5), (8, 1, 3, 1), (1, 30, 7, 40), (16, 64, 4, 33)], ids=str)
def test_evict_spares_what_reserved_and_cut_off_rows_need(dev, page, window, sinks, ahead):
    """pages released between a reserve and its attend, and before rows are cut off and written anew: every query
    sees its whole window, and every page behind the first of them is free"""
    pkg = load_pkg()
    h, kvh, hd, lens = 4, 2, 64, [50, 120, 7]
    c = pkg.PagedCache.allocate(1, 400, page, kvh, hd, 3, 400, torch.float32, dev)
    g = torch.Generator().manual_seed(30)
    hist = [[torch.zeros(0, kvh, hd)] * 2 for _ in lens]

    def attend(counts, status):
        starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
        q, k, v = (torch.randn(sum(counts), n, hd, generator=g) for n in (h, kvh, kvh))
        c.append(0, k.to(dev), v.to(dev), i32(starts, dev), status=status)
        out = c.attend(0, q.to(dev), i32(starts, dev), window=window, sinks=sinks, status=status)
        assert int(status) == 0
        for i, m in enumerate(counts):
            a, b = starts[i], starts[i + 1]
            hist[i] = [torch.cat([hist[i][0], k[a:b]]), torch.cat([hist[i][1], v[a:b]])]
            want, A, B = reference(q[a:b], *hist[i], m, window, sinks, False)
            check(out[a:b], want, A, B, hd, hist[i][0].shape[0], torch.float32, (i, m))

    def released(back):
        """pages of the slots that no query from lens - back on sees"""
        return sum((c.table[i].cpu()[e] < 0) == ((e + 1) * page <= n - back - window + 1 and e * page >= sinks)
                   for i, n in enumerate(c.lens.tolist()) for e in range(-(-n // page))) == sum(-(-n // page) for n in c.lens.tolist())

    attend(lens, c.reserve(i32(lens, dev)))
    counts = [ahead, 1, max(1, ahead // 2)]
    status = c.reserve(i32(counts, dev))
    c.evict(window, sinks, ahead=ahead)  # the batch's rows are yet to be attended
    assert released(ahead)
    attend(counts, status)
    c.evict(window, sinks, ahead=min(ahead, 7))  # up to 7 rows may be taken back
    assert released(min(ahead, 7))
    back = [min(ahead, 7), 1, 0]
    assert int(c.trim(i32([0, 1, 2], dev), i32([x.shape[0] - b for (x, _), b in zip(hist, back)], dev))) == 0
    hist[:] = [[x[:x.shape[0] - b] for x in hh] for hh, b in zip(hist, back)]
    attend([3, 1, 2], c.reserve(i32([3, 1, 2], dev)))
    c.evict(window, sinks)
    assert released(0)
    attend([1, 1, 1], c.reserve(i32([1, 1, 1], dev)))
    held = c.table.cpu()[c.table.cpu() >= 0].long()
    assert torch.equal(c.refs.cpu().long(), torch.bincount(held, minlength=400))
    with pytest.raises(pkg.QmoeError, match="ahead"):
        c.evict(window, sinks, ahead=-1)
    with pytest.raises(pkg.QmoeError, match="window"):
        c.evict(0, sinks, ahead=3)
    before = c.table.clone()
    c.evict(2 ** 31 - 1, 0, ahead=2 ** 31 - 1)
    assert torch.equal(c.table, before)


@pytest.mark.parametrize("slots", [65536, 65537, 200001])
def test_evict_on_many_slots(dev, slots):
    """more slots than a launch has workgroups: a page of each, behind the window or not"""
    pkg = load_pkg()
    c = pkg.PagedCache.allocate(1, slots, 2, 1, 64, slots, 2, torch.bfloat16, dev)
    for named in (None, torch.randperm(slots, generator=torch.Generator().manual_seed(32)).to(torch.int32).to(dev)):
        c.table[:, 0] = torch.arange(slots, device=dev).int()
        c.refs.fill_(1)
        c.lens.copy_(torch.arange(slots, device=dev) % 5)  # rows 0 and 1 are behind a window of 1 from length 2 on
        c.evict(1, 0, named)
        gone = c.lens >= 2
        assert torch.equal(c.table[:, 0] < 0, gone) and torch.equal(c.refs == 0, gone)
        assert torch.equal(c.table[:, 0][~gone], torch.arange(slots, device=dev).int()[~gone])


@pytest.mark.parametrize("order", ["rows", "heads"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_compact_moves_contents(dev, dtype, order):
    s = Setup(dev, HEADS[4], dtype, 7, [60, 100, 5, 0, 33], seed=16, layers=3, spare=40, order=order)
    s.k.copy_(torch.randn(s.k.shape, generator=s.g))
    s.v.copy_(torch.randn(s.v.shape, generator=s.g))
    old, k, v = s.table.clone().cpu(), s.k.clone(), s.v.clone()
    used = int(s.cache.compact())
    assert used == int((s.refs > 0).sum()) and (s.refs[:used] > 0).all() and (s.refs[used:] == 0).all()
    new = s.table.cpu()
    for a, b in zip(old.flatten().tolist(), new.flatten().tolist()):
        assert (a < 0) == (b < 0)
        if a >= 0:
            assert torch.equal(s.k[:, b], k[:, a]) and torch.equal(s.v[:, b], v[:, a])
    assert int(s.cache.compact()) == used and torch.equal(s.table.cpu(), new)


def test_a_larger_pool(dev):
    """more pages than one pass of the search covers, used pages at the far end"""
    pkg = load_pkg()
    n_pages = 70001
    c = pkg.PagedCache.allocate(1, n_pages, 1, 1, 64, 3, 9000, torch.bfloat16, dev)
    c.refs.fill_(1)
    c.refs[::17] = 0
    free = list(range(0, n_pages, 17))
    assert int(c.reserve(i32([3000, 1117], dev), i32([2, 0], dev))) == 0
    assert c.table[2, :3000].tolist() == free[:3000] and c.table[0, :1117].tolist() == free[3000:4117]
    assert int(c.reserve(i32([2], dev), i32([1], dev))) == 4117 + 2 - len(free)
    c.refs.fill_(0)
    ids = list(range(n_pages - 3000, n_pages))
    c.table.fill_(-1)
    c.table[1, :3000] = i32(ids, dev)
    c.refs[n_pages - 3000:] = 1
    c.k.zero_()
    c.k[0, n_pages - 3000:, 0, 0, 0] = torch.arange(3000, device=dev).to(torch.bfloat16)
    assert int(c.compact()) == 3000
    assert c.table[1, :3000].tolist() == list(range(3000)) and int(c.refs[:3000].sum()) == 3000 and int(c.refs.sum()) == 3000
    assert torch.equal(c.k[0, :3000, 0, 0, 0], torch.arange(3000, device=dev).to(torch.bfloat16))


# ------------------------------------------------- streams, graphs, a run

def test_other_stream_and_two_at_once(dev):
    s = Setup(dev, HEADS[0], torch.bfloat16, 16, [2000, 60, 900], seed=17)
    q, starts = s.queries([1, 1, 1])
    q2, starts2 = s.queries([200, 60, 100])
    q, q2, st, st2 = q.to(dev), q2.to(dev), i32(starts, dev), i32(starts2, dev)
    a, b = s.cache.attend(0, q, st), s.cache.attend(0, q2, st2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(5):
        outs.append(s.cache.attend(0, q, st, stream=s1))
        with torch.cuda.stream(s2):
            outs.append(s.cache.attend(0, q2, st2))
    outs.append(s.cache.attend(0, q, st, stream=s1.cuda_stream))
    torch.cuda.synchronize()
    for i, o in enumerate(outs[:-1]):
        assert torch.equal(o, b if i % 2 else a)
    assert torch.equal(outs[-1], a)


def test_a_captured_step_follows_the_cache(dev):
    """one graph of reserve, append and attend, replayed as the sequences grow, against eager calls on a second
    cache; two graphs of one cache take turns"""
    pkg = load_pkg()
    h, kvh, hd, B = 16, 2, 128, 5
    caches = [pkg.PagedCache.allocate(2, 200, 8, kvh, hd, B, 30, torch.bfloat16, dev) for _ in range(2)]
    g = torch.Generator(device=dev).manual_seed(18)
    first = [3, 40, 1, 17, 8]
    starts0 = i32(np.concatenate([[0], np.cumsum(first)]).tolist(), dev)
    k0, v0 = (torch.randn(sum(first), kvh, hd, generator=g, device=dev).bfloat16() for _ in range(2))
    for c in caches:
        assert int(c.reserve(i32(first, dev))) == 0
        for layer in range(2):
            c.append(layer, k0, v0, starts0)
    starts, ones = i32(list(range(B + 1)), dev), i32([1] * B, dev)
    q, k, v = (torch.randn(B, n, hd, generator=g, device=dev).bfloat16() for n in (h, kvh, kvh))

    def step(c):
        status = c.reserve(ones)
        outs = []
        for layer in range(2):
            c.append(layer, k, v, starts)
            outs.append(c.attend(layer, q, starts, window=20, sinks=2))
        return status, outs

    # warm up on a cache of its own, then capture
    spare = pkg.PagedCache.allocate(2, 200, 8, kvh, hd, B, 30, torch.bfloat16, dev)
    spare.reserve(i32(first, dev))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(spare)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            results.append(step(caches[0]))
        graphs.append(gr)
    for i in range(12):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=dev))
        graphs[i % 2].replay()
        status, outs = step(caches[1])
        torch.cuda.synchronize()
        assert int(results[i % 2][0]) == 0 and int(status) == 0
        for a, b in zip(results[i % 2][1], outs):
            assert torch.equal(a, b), i
        for a, b in zip((caches[0].table, caches[0].lens, caches[0].refs), (caches[1].table, caches[1].lens, caches[1].refs)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,more", [([20, 20], [9, 1]), ([300, 100], [200, 90]), ([3000, 40], [1, 30]), ([7] * 80, [9] * 80)],
                         ids=["tokens", "chunks", "joined", "indexed"])
def test_a_refused_step_writes_nothing(dev, rows, more, dtype):
    """reserve, append and attend of a pool that is full, eager and captured, with the reserve's status: the cache and
    the output stay as they are, shared pages among them; after pages were released the same calls and the same graph
    do what they do without a status"""
    pkg = load_pkg()
    h, kvh, hd, page, n = 8, 2, 64, 8, len(rows)
    g = torch.Generator(device=dev).manual_seed(29)
    held = sum(-(-r // page) for r in rows)
    lacks = sum(-(-(r + m) // page) - r // page for r, m in zip(rows, more))  # new pages, copies of shared last ones
    c = pkg.PagedCache.allocate(2, held + lacks, page, kvh, hd, 2 * n, 1000, dtype, dev)
    c.k.zero_()
    c.v.zero_()
    starts0 = i32(np.concatenate([[0], np.cumsum(rows)]).tolist(), dev)
    k0, v0 = (torch.randn(sum(rows), kvh, hd, generator=g, device=dev).to(dtype) for _ in range(2))
    status = c.reserve(i32(rows, dev))
    for layer in range(2):
        c.append(layer, k0, v0, starts0, status=status)
    src, dst = i32(list(range(n)), dev), i32(list(range(n, 2 * n)), dev)
    assert int(status) == 0 and int(c.fork(src, dst)) == 0
    free = c.refs == 0
    c.refs[free] = 1  # pages of other sequences
    starts, add = i32(np.concatenate([[0], np.cumsum(more)]).tolist(), dev), i32(more, dev)
    q, k, v = (torch.randn(sum(more), m, hd, generator=g, device=dev).to(dtype) for m in (h, kvh, kvh))
    outs = [torch.full((sum(more), h, hd), 5.0, dtype=dtype, device=dev) for _ in range(2)]
    before = [t.clone() for t in (c.k, c.v, c.table, c.lens, c.refs)]

    def step():
        status = c.reserve(add, dst)
        for layer in range(2):
            c.append(layer, k, v, starts, dst, status=status)
            c.attend(layer, q, starts, dst, out=outs[layer], status=status)
        return status

    def untouched():
        return all(torch.equal(a, b) for a, b in zip(before, (c.k, c.v, c.table, c.lens, c.refs))) and \
            all((o == 5).all() for o in outs)

    assert int(step()) == lacks and untouched()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        status = step()
    for _ in range(2):
        graph.replay()
        assert int(status) == lacks and untouched()
    twice = c.reserve(add, torch.zeros_like(dst))
    c.append(0, k, v, starts, dst, status=twice)
    assert int(twice) == -1 and untouched()
    c.refs[free] = 0  # the others are done
    graph.replay()
    assert int(status) == 0 and int((c.refs == 0).sum()) == 0
    for i, (r, m) in enumerate(zip(rows, more)):
        a, b = int(starts[i]), int(starts[i + 1])
        kk, vv = (torch.cat([x[int(starts0[i]):int(starts0[i + 1])], y[a:b]]).cpu() for x, y in ((k0, k), (v0, v)))
        for layer in range(2):
            want, A, B = reference(q[a:b].cpu(), kk, vv, m, 0, 0, False)
            check(outs[layer][a:b], want, A, B, hd, r + m, dtype, (i, layer))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_a_serving_run(dev, dtype):
    """prompts in chunks, branches forked, single tokens, a window, pages released and compacted: every output
    against 64 bits over that sequence's own history"""
    pkg = load_pkg()
    h, kvh, hd, window, sinks, page = 8, 2, 64, 48, 5, 8
    c = pkg.PagedCache.allocate(1, 120, page, kvh, hd, 6, 40, dtype, dev)
    c.k.fill_(float("nan"))
    c.v.fill_(float("nan"))
    g = torch.Generator().manual_seed(19)
    hist = [[torch.zeros(0, kvh, hd)] * 2 for _ in range(6)]

    def step(slots, counts):
        starts = np.concatenate([[0], np.cumsum(counts)]).tolist()
        q, k, v = (torch.randn(sum(counts), n, hd, generator=g).to(dtype) for n in (h, kvh, kvh))
        sl, st = i32(slots, dev), i32(starts, dev)
        assert int(c.reserve(i32(counts, dev), sl)) == 0
        c.append(0, k.to(dev), v.to(dev), st, sl)
        out = c.attend(0, q.to(dev), st, sl, window=window, sinks=sinks)
        table = c.table.tolist()
        for i, s in enumerate(slots):
            a, b = starts[i], starts[i + 1]
            hist[s] = [torch.cat([hist[s][0].to(dtype), k[a:b]]), torch.cat([hist[s][1].to(dtype), v[a:b]])]
            gone = [(e * page, e * page + page) for e, p in enumerate(table[s]) if p < 0]  # after a cut, also near ones
            want, A, B = reference(q[a:b], hist[s][0], hist[s][1], b - a, window, sinks, False, hidden=gone)
            check(out[a:b], want, A, B, hd, hist[s][0].shape[0], dtype, (s, a, b))
        c.evict(window, sinks, sl)

    step([0, 1], [37, 90])
    step([0, 1], [50, 3])
    assert int(c.fork(i32([0, 0, 1], dev), i32([2, 3, 4], dev))) == 0
    for s, p in ((2, 0), (3, 0), (4, 1)):
        hist[s] = list(hist[p])
    for _ in range(9):
        step([4, 0, 2, 3, 1], [1, 1, 1, 2, 1])
    used = int((c.refs > 0).sum())
    assert int(c.compact()) == used
    step([1, 2, 0], [1, 30, 1])
    assert int(c.trim(i32([0, 4], dev), i32([0, hist[4][0].shape[0] - 2], dev))) == 0
    hist[0] = [torch.zeros(0, kvh, hd)] * 2
    hist[4] = [x[:-2] for x in hist[4]]
    step([0, 4, 3], [20, 1, 1])
    assert (c.refs >= 0).all() and int(c.refs.sum()) == int((c.table >= 0).sum())
