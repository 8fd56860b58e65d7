"""Drafted tokens at sizes where units, places in the workspace and precision
change over, and rotation by large angles, on the GPU against the restatements
in 64 bits of test_gpu_paged_tree (whose bars these are)."""
import ctypes
import random

import pytest
import torch

from conftest import load_pkg
from test_gpu_paged import Setup, U, check, i32
from test_gpu_paged_tree import DTYPES, dev, grow, masked, near, plan, sight, turned  # noqa: F401

pytestmark = pytest.mark.gpu


def guarded(s, layer, q, tree, starts, window, sinks, slack=1 << 22):
    """qmoe_paged_attn_tree on a workspace of the size that it asks for, between bytes that have to stay"""
    pkg, h, hd = load_pkg(), s.h, s.hd
    n, m = q.shape[0], starts.shape[0] - 1
    need = pkg.lib().qmoe_paged_ws_bytes(s.cache._cp, pkg.PAGED_ATTN_TREE, n, m, h)
    ws = torch.full((256 + need + slack,), 0x5A, dtype=torch.uint8, device=s.dev)
    out = torch.full((n + 2, h, hd), 7.0, dtype=s.dtype, device=s.dev)
    b = pkg.QmoePagedBatch(starts=starts.data_ptr(), slots=None, n=n, n_seqs=m, status=None)
    a = pkg.QmoePagedQuery(q=q.data_ptr(), out=out[1].data_ptr(), q_token_stride=h * hd, q_head_stride=hd, out_token_stride=h * hd,
                           out_head_stride=hd, n_heads=h, window=window, sinks=sinks, grouped=0, scale=0.0)
    t = pkg.QmoePagedTree(depths=tree.depths.data_ptr(), seen=tree.seen.data_ptr(), words=tree.words)
    e = pkg.QmoeErr()
    torch.cuda.synchronize()
    rc = pkg.lib().qmoe_paged_attn_tree(s.cache._cp, layer, ctypes.byref(b), ctypes.byref(a), ctypes.byref(t), ws[256:].data_ptr(), need,
                                        torch.cuda.current_stream().cuda_stream, ctypes.byref(e))
    assert rc == 0, e.msg
    torch.cuda.synchronize()
    assert (ws[:256] == 0x5A).all() and (ws[256 + need:] == 0x5A).all()
    assert (out[0] == 7).all() and (out[n + 1] == 7).all()
    return out[1:n + 1]


@DTYPES
@pytest.mark.parametrize("m", [64, 65, 100])
@pytest.mark.parametrize("shape,rows,nodes,window,sinks", [((16, 2, 128), 496, 4, 0, 0), ((4, 2, 64), 640, 16, 0, 0),
                                                           ((4, 2, 64), 3968, 12, 700, 3), ((6, 2, 192), 656, 8, 0, 0),
                                                           ((16, 2, 128), 2000, 3, 600, 0)], ids=str)
def test_units_of_32_rows_stay_in_their_workspace(dev, shape, rows, nodes, window, sinks, m, dtype):  # noqa: F811
    """17 to 32 rows a sequence on tables or windows of few keys, with and without an index of the sequences"""
    r = random.Random(m * 1000 + rows + nodes)
    lens = [rows] + [r.randrange(nodes, rows + 1) for _ in range(m - 1)]
    s = Setup(dev, shape, dtype, 16, lens, seed=m + rows)
    counts = [nodes - (1 if i % 7 == 3 else 0) for i in range(m)]
    ups = [grow(r, c) for c in counts]
    q, starts = s.queries(counts)
    q, st = q.to(dev), i32(starts, dev)
    tree = s.cache.tree(i32([p for u in ups for p in u], dev), st, most=nodes)
    out = guarded(s, 0, q, tree, st, window, sinks)
    for i, up in enumerate(ups):
        a, b = starts[i], starts[i + 1]
        want, A, B = masked(q[a:b].cpu(), s.hk[i], s.hv[i], sight(lens[i] - counts[i], *plan(up), window, sinks), False)
        check(out[a:b], want, A, B, s.hd, lens[i], dtype, i)
    assert torch.equal(s.cache.attend_tree(0, q, tree, window=window, sinks=sinks), out)


@pytest.mark.parametrize("lens,counts", [([90, 300, 150, 64], [60, 40, 20, 64]), ([260, 70, 100], [200, 3, 9])], ids=["large", "one_large"])
@pytest.mark.parametrize("hd", [64, 128, 192, 256])
def test_weights_of_all_trees_have_16_bits(dev, hd, lens, counts, monkeypatch):  # noqa: F811
    """bf16 outputs of more than 128 rows a sequence, and of small trees beside a large one, within the weights' 16 bits
    (2^-16 of A twice: a half step of the second part, and of the sum that leaves it out) and their own rounding.  Weights of
    one bf16 part are off by 2^-9 of the heaviest: up to 7 times this bar on contexts as short as these"""
    monkeypatch.setattr(Setup, "table_rows", 1024)
    r = random.Random(hd + len(lens))
    s = Setup(dev, (8, 1, hd), torch.bfloat16, 16, lens, seed=hd)
    ups = [grow(r, c) for c in counts]
    q, starts = s.queries(counts)
    tree = s.cache.tree(i32([p for u in ups for p in u], dev), i32(starts, dev))
    out = s.cache.attend_tree(0, q.to(dev), tree).double().cpu()
    for i, up in enumerate(ups):
        T = lens[i]
        want, A, B = masked(q[starts[i]:starts[i + 1]], s.hk[i], s.hv[i], sight(T - counts[i], *plan(up), 0, 0), False)
        tol = A * (2 * (hd + 24) * U * (B + 1) + 2 * (T + 64) * U + 2 * 2.0 ** -16)
        tol = tol + (want.abs() + tol) * 2.0 ** -8
        err = (out[starts[i]:starts[i + 1]] - want).abs()
        assert (err <= tol).all(), (i, float((err / tol).max()))


def test_rotary_of_large_angles(dev):  # noqa: F811
    """freqs up to 2^48 - 2^24 at positions up to 2^29: up to 2^77 radians"""
    kvh, hd, page = 2, 128, 4096
    lens = [2 ** 29, 2 ** 29 - 1, 2 ** 28 + 12345, 1000003, 4097, 2]
    table = torch.full((len(lens), 2 ** 29 // page), -1, dtype=torch.int32, device=dev)
    for i, n in enumerate(lens):
        table[i, (n - 1) // page] = i
    k, v = (torch.zeros(1, len(lens), page, kvh, hd, device=dev) for _ in range(2))
    cache = load_pkg().PagedCache(k, v, table, i32(lens, dev), torch.ones(len(lens), dtype=torch.int32, device=dev))
    g = torch.Generator().manual_seed(61)
    n = len(lens)
    for low, high in ((0, 8), (8, 32), (32, 47)):
        freqs = torch.exp2(low + (high - low) * torch.rand(64, generator=g, dtype=torch.float64)).float()
        freqs[0] = 2.0 ** high * (1 if high < 47 else 2 - 2.0 ** -23)
        q, kn, vn = (torch.randn(n, m, hd, generator=g) for m in (3, kvh, kvh))
        got = cache.append_rotary(0, kn.to(dev), vn.to(dev), i32(list(range(n + 1)), dev), freqs.to(dev), q=q.to(dev))
        want, mag = turned(q, torch.tensor(lens) - 1, freqs, False, None, 0)
        near(got, want, mag, torch.float32, (low, high))
