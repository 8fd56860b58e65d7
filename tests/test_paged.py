"""The paged cache without a GPU: its index arithmetic against plain
restatements (tests/c/paged_index.c, bad table entries and lengths among
them), and the refusals of every qmoe_paged_* call, which come back as -1
with a message before the device is touched (the pointers here are no
memory at all)."""
import ctypes
import os
import shutil
import subprocess

import pytest

from conftest import ROOT, load_pkg

CSRC = os.path.join(ROOT, "qwen3.8-flash-next_amd", "csrc")


def test_index_arithmetic(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc is not available")
    exe = str(tmp_path / "paged_index")
    r = subprocess.run([gcc, "-std=c11", "-O2", "-Wall", "-Wextra", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC,
                        os.path.join(ROOT, "tests", "c", "paged_index.c"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


A = 0x1000  # an aligned address that nothing follows


def cache(pkg, **kw):
    f = dict(k=A, v=A, layer_stride=1 << 20, page_stride=4096, row_stride=256, head_stride=128, dtype=pkg.BF16, n_layers=2,
             n_pages=10, page_rows=16, n_kv_heads=2, head_dim=128, table=A, table_stride=8, lens=A, refs=A, n_slots=4,
             max_pages=8)
    f.update(kw)
    return pkg.QmoePagedCache(**f)


def batch(pkg, **kw):
    f = dict(starts=A, slots=A, n=5, n_seqs=3)
    f.update(kw)
    return pkg.QmoePagedBatch(**f)


def query(pkg, **kw):
    f = dict(q=A, out=A, q_token_stride=1024, q_head_stride=128, out_token_stride=1024, out_head_stride=128, n_heads=8,
             window=0, sinks=0, grouped=0, scale=0.0)
    f.update(kw)
    return pkg.QmoePagedQuery(**f)


def calls(pkg, c):
    """every call on cache c with arguments that are otherwise right"""
    L, b, q = pkg.lib(), batch(pkg), query(pkg)
    e = pkg.QmoeErr()
    cp, bp, qp, ep = (ctypes.byref(x) if x is not None else None for x in (c, b, q, e))
    big = ctypes.c_size_t(1 << 40)
    yield e, L.qmoe_paged_append(cp, 0, bp, A, A, pkg.BF16, 256, 128, 256, 128, None, ep)
    yield e, L.qmoe_paged_attn(cp, 0, bp, qp, A, big, None, ep)
    yield e, L.qmoe_paged_reserve(cp, A, A, 3, A, A, big, None, ep)
    yield e, L.qmoe_paged_fork(cp, A, A, None, 3, A, A, big, None, ep)
    yield e, L.qmoe_paged_evict(cp, A, 3, 64, 0, None, ep)
    yield e, L.qmoe_paged_compact(cp, A, A, big, None, ep)


BAD_CACHE = [
    (dict(dtype=7), "dtype"), (dict(head_dim=96), "head_dim"), (dict(head_dim=320), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(n_kv_heads=0), "n_kv_heads"), (dict(page_rows=0), "page_rows"), (dict(page_rows=5000), "page_rows"),
    (dict(n_layers=0), "n_layers"), (dict(n_pages=0), "n_pages"), (dict(n_pages=(1 << 20) + 1), "n_pages"),
    (dict(n_slots=0), "n_slots"), (dict(max_pages=0), "max_pages"),
    (dict(max_pages=1 << 27, table_stride=1 << 27), "rows"), (dict(table_stride=7), "table_stride"),
    (dict(k=None), "k is NULL"), (dict(v=None), "v is NULL"), (dict(table=None), "table is NULL"),
    (dict(lens=None), "lens is NULL"), (dict(refs=None), "refs is NULL"), (dict(k=A + 8), "aligned"), (dict(v=A + 2), "aligned"),
    (dict(page_stride=-4096), "page_stride"), (dict(row_stride=260), "row_stride"), (dict(head_stride=132), "head_stride"),
    (dict(row_stride=128), "overlap"), (dict(page_stride=2048), "overlap"), (dict(layer_stride=4096), "overlap"),
    (dict(head_stride=64), "overlap"), (dict(layer_stride=1 << 62), "overlap"), (dict(page_stride=0), "overlap"),
]


@pytest.mark.parametrize("kw,msg", BAD_CACHE, ids=[f"{list(k)[0]}_{i}" for i, (k, _) in enumerate(BAD_CACHE)])
def test_bad_caches_are_refused(kw, msg):
    pkg = load_pkg()
    c = cache(pkg, **kw)
    for e, rc in calls(pkg, c):
        assert rc == -1 and msg in e.msg.decode(), (rc, e.msg)
    for call in range(4):
        assert pkg.lib().qmoe_paged_ws_bytes(ctypes.byref(c), call, 5, 3, 8) == 0


def test_null_arguments_are_refused():
    pkg = load_pkg()
    L, e = pkg.lib(), pkg.QmoeErr()
    for err, rc in calls(pkg, None):
        assert rc == -1 and b"cache is NULL" in err.msg
    c, b, q = cache(pkg), batch(pkg), query(pkg)
    cp, bp, qp, ep = (ctypes.byref(x) for x in (c, b, q, e))
    for rc, msg in ((L.qmoe_paged_append(cp, 0, None, A, A, pkg.BF16, 256, 128, 256, 128, None, ep), b"batch is NULL"),
                    (L.qmoe_paged_append(cp, 0, bp, None, A, pkg.BF16, 256, 128, 256, 128, None, ep), b"k is NULL"),
                    (L.qmoe_paged_append(cp, 0, bp, A, None, pkg.BF16, 256, 128, 256, 128, None, ep), b"v is NULL"),
                    (L.qmoe_paged_attn(cp, 0, bp, None, A, 1 << 40, None, ep), b"query is NULL"),
                    (L.qmoe_paged_attn(cp, 0, bp, qp, None, 1 << 40, None, ep), b"workspace"),
                    (L.qmoe_paged_reserve(cp, A, None, 3, A, A, 1 << 40, None, ep), b"n_new is NULL"),
                    (L.qmoe_paged_reserve(cp, A, A, 3, None, A, 1 << 40, None, ep), b"status is NULL"),
                    (L.qmoe_paged_fork(cp, None, A, None, 3, A, A, 1 << 40, None, ep), b"src is NULL"),
                    (L.qmoe_paged_fork(cp, A, None, None, 3, A, A, 1 << 40, None, ep), b"dst is NULL"),
                    (L.qmoe_paged_fork(cp, A, A, None, 3, None, A, 1 << 40, None, ep), b"status is NULL"),
                    (L.qmoe_paged_compact(cp, None, A, 1 << 40, None, ep), b"used is NULL")):
        assert rc == -1
    # the messages, one call at a time
    assert L.qmoe_paged_append(cp, 0, None, A, A, pkg.BF16, 256, 128, 256, 128, None, ep) == -1 and b"batch is NULL" in e.msg
    assert L.qmoe_paged_reserve(cp, A, A, 3, None, A, 1 << 40, None, ep) == -1 and b"status is NULL" in e.msg
    assert L.qmoe_paged_fork(cp, A, None, None, 3, A, A, 1 << 40, None, ep) == -1 and b"dst is NULL" in e.msg
    # a NULL err is allowed
    assert L.qmoe_paged_evict(None, A, 3, 64, 0, None, None) == -1


def test_every_null_argument_is_named():
    """each call on its own, its message read before the next"""
    pkg = load_pkg()
    L, e, big = pkg.lib(), pkg.QmoeErr(), 1 << 40
    structs = cache(pkg), batch(pkg), query(pkg), query(pkg, q=None), query(pkg, out=None), batch(pkg, starts=None), e
    cp, bp, qp, no_q, no_out, no_starts, ep = (ctypes.byref(x) for x in structs)
    append = lambda b, k, v: L.qmoe_paged_append(cp, 0, b, k, v, pkg.BF16, 256, 128, 256, 128, None, ep)
    attn = lambda b, q, ws=A: L.qmoe_paged_attn(cp, 0, b, q, ws, big, None, ep)
    reserve = lambda add, status=A, ws=A: L.qmoe_paged_reserve(cp, A, add, 3, status, ws, big, None, ep)
    fork = lambda src, dst, status=A, ws=A: L.qmoe_paged_fork(cp, src, dst, None, 3, status, ws, big, None, ep)
    compact = lambda used, ws=A: L.qmoe_paged_compact(cp, used, ws, big, None, ep)
    for call, args, msg in ((append, (None, A, A), "batch is NULL"), (append, (bp, None, A), "k is NULL"),
                            (append, (bp, A, None), "v is NULL"), (append, (no_starts, A, A), "starts is NULL"),
                            (attn, (None, qp), "batch is NULL"), (attn, (bp, None), "query is NULL"),
                            (attn, (bp, no_q), "q is NULL"), (attn, (bp, no_out), "out is NULL"),
                            (attn, (no_starts, qp), "starts is NULL"), (attn, (bp, qp, None), "workspace is NULL"),
                            (reserve, (None,), "n_new is NULL"), (reserve, (A, None), "status is NULL"),
                            (reserve, (A, A, None), "workspace is NULL"), (fork, (None, A), "src is NULL"),
                            (fork, (A, None), "dst is NULL"), (fork, (A, A, None), "status is NULL"),
                            (fork, (A, A, A, None), "workspace is NULL"), (compact, (None,), "used is NULL"),
                            (compact, (A, None), "workspace is NULL")):
        e.msg = b"nothing"
        assert call(*args) == -1 and msg in e.msg.decode(), (msg, e.msg)


BAD_ATTN = [
    (dict(), dict(n=-1), dict(), 0, "n = -1"), (dict(), dict(n_seqs=-1), dict(), 0, "n_seqs"),
    (dict(), dict(n_seqs=70000), dict(), 0, "n_seqs"), (dict(), dict(slots=None, n_seqs=5), dict(), 0, "slots"),
    (dict(), dict(starts=None), dict(), 0, "starts is NULL"), (dict(), dict(), dict(), 2, "layer 2"),
    (dict(), dict(), dict(), -1, "layer -1"), (dict(), dict(), dict(n_heads=0), 0, "n_heads"),
    (dict(), dict(), dict(n_heads=7), 0, "n_heads"), (dict(), dict(n=1 << 29), dict(), 0, "heads are more"),
    (dict(), dict(), dict(window=-1), 0, "window"), (dict(), dict(), dict(sinks=-1), 0, "sinks"),
    (dict(), dict(), dict(grouped=2), 0, "grouped"), (dict(), dict(), dict(scale=float("nan")), 0, "scale"),
    (dict(), dict(), dict(scale=float("inf")), 0, "scale"), (dict(), dict(), dict(scale=-3e38), 0, "scale"),
    (dict(), dict(), dict(q=None), 0, "q is NULL"),
    (dict(), dict(), dict(out=None), 0, "out is NULL"), (dict(), dict(), dict(q=A + 4), 0, "aligned"),
    (dict(), dict(), dict(out=A + 8), 0, "aligned"), (dict(), dict(), dict(q_token_stride=1025), 0, "q_token_stride"),
    (dict(), dict(), dict(q_head_stride=-128), 0, "q_head_stride"), (dict(), dict(), dict(out_token_stride=512), 0, "overlap"),
    (dict(), dict(), dict(out_head_stride=64), 0, "overlap"), (dict(), dict(), dict(out_token_stride=0), 0, "overlap"),
]


@pytest.mark.parametrize("ckw,bkw,qkw,layer,msg", BAD_ATTN, ids=[str(i) for i in range(len(BAD_ATTN))])
def test_bad_attention_calls_are_refused(ckw, bkw, qkw, layer, msg):
    pkg = load_pkg()
    e = pkg.QmoeErr()
    c, b, q = cache(pkg, **ckw), batch(pkg, **bkw), query(pkg, **qkw)
    rc = pkg.lib().qmoe_paged_attn(ctypes.byref(c), layer, ctypes.byref(b), ctypes.byref(q), A, 1 << 40, None, ctypes.byref(e))
    assert rc == -1 and msg in e.msg.decode(), (rc, e.msg)


def test_other_bad_calls_are_refused():
    pkg = load_pkg()
    L, e = pkg.lib(), pkg.QmoeErr()
    c, b = cache(pkg), batch(pkg)
    f = cache(pkg, dtype=pkg.F32)
    cp, fp, bp, ep = (ctypes.byref(x) for x in (c, f, b, e))

    def refused(rc, msg):
        assert rc == -1 and msg in e.msg.decode(), (rc, e.msg)

    refused(L.qmoe_paged_append(fp, 0, bp, A, A, pkg.BF16, 256, 128, 256, 128, None, ep), "dtype")
    refused(L.qmoe_paged_append(cp, 0, bp, A, A, 5, 256, 128, 256, 128, None, ep), "dtype")
    refused(L.qmoe_paged_append(cp, 5, bp, A, A, pkg.BF16, 256, 128, 256, 128, None, ep), "layer 5")
    refused(L.qmoe_paged_append(cp, 0, bp, A, A, pkg.BF16, 250, 128, 256, 128, None, ep), "k_token_stride")
    refused(L.qmoe_paged_append(cp, 0, bp, A, A, pkg.BF16, 256, 128, 256, -128, None, ep), "v_head_stride")
    refused(L.qmoe_paged_append(cp, 0, bp, A + 4, A, pkg.BF16, 256, 128, 256, 128, None, ep), "aligned")
    many = batch(pkg, n=1 << 28)
    refused(L.qmoe_paged_append(cp, 0, ctypes.byref(many), A, A, pkg.BF16, 256, 128, 256, 128, None, ep), "too many")
    refused(L.qmoe_paged_reserve(cp, A, A, 1025, A, A, 1 << 40, None, ep), "n_seqs")
    refused(L.qmoe_paged_reserve(cp, None, A, 5, A, A, 1 << 40, None, ep), "slots")
    refused(L.qmoe_paged_fork(cp, A, A, None, 1025, A, A, 1 << 40, None, ep), "n_seqs")
    refused(L.qmoe_paged_evict(cp, A, 3, 0, 0, None, ep), "window")
    refused(L.qmoe_paged_evict(cp, A, 3, 4, -1, None, ep), "sinks")
    refused(L.qmoe_paged_evict(cp, None, 5, 4, 0, None, ep), "slots")
    # workspaces: too small by one byte, NULL, misaligned
    for call, run in ((1, lambda w, n: L.qmoe_paged_reserve(cp, A, A, 3, A, w, n, None, ep)),
                      (2, lambda w, n: L.qmoe_paged_fork(cp, A, A, None, 3, A, w, n, None, ep)),
                      (3, lambda w, n: L.qmoe_paged_compact(cp, A, w, n, None, ep)),
                      (0, lambda w, n: L.qmoe_paged_attn(cp, 0, bp, ctypes.byref(query(pkg)), w, n, None, ep))):
        need = L.qmoe_paged_ws_bytes(cp, call, 5, 3, 8)
        assert need > 0
        refused(run(A, need - 1), "workspace")
        refused(run(None, need), "workspace")
        refused(run(A + 8, need), "workspace")


# a workgroup of 256 threads per sequence and kv head; 128 rows of 512 threads
@pytest.mark.parametrize("ckw,n,n_seqs,heads,fits", [
    (dict(n_kv_heads=256, head_dim=64, max_pages=1), 65536, 65536, 256, False),
    (dict(n_kv_heads=256, head_dim=64, max_pages=1), 65535, 65535, 256, True),
    (dict(n_kv_heads=256, head_dim=64, max_pages=4096), 65535, 65535, 256, False),  # and parts of the keys
    (dict(n_kv_heads=256, head_dim=64, max_pages=4096), 65527, 65527, 256, True),
    (dict(n_kv_heads=1024, head_dim=256, max_pages=1, dtype=0), 1 << 20, 1 << 15, 1024, False),
    (dict(n_kv_heads=1024, head_dim=64, max_pages=1), 1 << 20, 65536, 1024, False),
    (dict(n_kv_heads=8, head_dim=64, max_pages=1), 1 << 20, 1, 1024, True),
])
def test_more_work_than_a_launch_holds_is_refused(ckw, n, n_seqs, heads, fits):
    pkg = load_pkg()
    L, e = pkg.lib(), pkg.QmoeErr()
    hd = ckw["head_dim"]
    c = cache(pkg, **dict(dict(head_stride=hd, row_stride=hd * ckw["n_kv_heads"], page_stride=16 * hd * ckw["n_kv_heads"],
                               layer_stride=1 << 40, n_slots=65536, table_stride=ckw["max_pages"]), **ckw))
    assert (L.qmoe_paged_ws_bytes(ctypes.byref(c), 0, n, n_seqs, heads) > 0) == fits
    if not fits:
        q = query(pkg, n_heads=heads, q_token_stride=heads * hd, q_head_stride=hd, out_token_stride=heads * hd, out_head_stride=hd)
        b = batch(pkg, n=n, n_seqs=n_seqs)
        rc = L.qmoe_paged_attn(ctypes.byref(c), 0, ctypes.byref(b), ctypes.byref(q), A, 1 << 40, None, ctypes.byref(e))
        assert rc == -1 and b"more work" in e.msg, e.msg


def test_calls_with_nothing_to_do_touch_nothing():
    pkg = load_pkg()
    L, e = pkg.lib(), pkg.QmoeErr()
    c, q = cache(pkg), query(pkg)
    cp, ep = ctypes.byref(c), ctypes.byref(e)
    for b in (batch(pkg, n=0), batch(pkg, n_seqs=0)):
        assert L.qmoe_paged_append(cp, 0, ctypes.byref(b), None, None, pkg.BF16, 256, 128, 256, 128, None, ep) == 0
        assert L.qmoe_paged_attn(cp, 0, ctypes.byref(b), ctypes.byref(q), None, 0, None, ep) == 0
    assert L.qmoe_paged_evict(cp, A, 0, 4, 0, None, ep) == 0


def test_scales_that_round_to_the_default_are_refused():
    pkg = load_pkg()
    for bad in (0, 0.0, -0.0, 1e-46, -1e-46, 1e-300):
        with pytest.raises(pkg.QmoeError, match="scale"):
            pkg.PagedCache._scale(bad)
    for good in (1e-45, -1e-38, 1.0, float("nan"), float("inf")):  # the last two are refused by the library
        pkg.PagedCache._scale(good)


def test_sizes_that_c_would_cut_off_are_refused():
    import torch
    pkg = load_pkg()
    i32 = torch.int32
    k, lens, refs = torch.zeros(1, 4, 8, 2, 64), torch.zeros(3, dtype=i32), torch.zeros(4, dtype=i32)
    table = torch.zeros(3, 5, dtype=i32)
    many = k[:, :1].expand(1, 2 ** 32 + 4, 8, 2, 64)
    wide = table[:, :1].expand(3, 2 ** 32 + 5)
    for bad in ((many, many, table, lens, refs), (k, k, wide, lens, refs)):
        with pytest.raises(pkg.QmoeError, match="below 2\\^31"):
            pkg.PagedCache(*bad)


def test_the_class_refuses_other_tensors():
    import torch
    pkg = load_pkg()
    i32 = torch.int32
    k = torch.zeros(1, 4, 8, 2, 64)
    table, lens, refs = torch.zeros(3, 5, dtype=i32), torch.zeros(3, dtype=i32), torch.zeros(4, dtype=i32)
    for bad, msg in (((k, k[:, :3], table, lens, refs), "one shape"), ((k, k.bfloat16(), table, lens, refs), "one shape"),
                     ((k[0], k[0], table, lens, refs), "layers"),
                     ((k.transpose(3, 4), k.transpose(3, 4), table, lens, refs), "contiguous"),
                     ((k, k, table.long(), lens, refs), "int32"), ((k, k, table[:2], lens, refs), "table"),
                     ((k, k, table, lens, refs[:3]), "refs"), ((k.double(), k.double(), table, lens, refs), "dtype"),
                     ((k, k, table, lens, refs), "GPU")):
        with pytest.raises(pkg.QmoeError, match=msg):
            pkg.PagedCache(*bad)


def test_a_misaligned_status_is_refused():
    pkg = load_pkg()
    L, e = pkg.lib(), pkg.QmoeErr()
    c, b, q = cache(pkg), batch(pkg, status=A + 2), query(pkg)
    cp, bp, ep = (ctypes.byref(x) for x in (c, b, e))
    assert L.qmoe_paged_append(cp, 0, bp, A, A, pkg.BF16, 256, 128, 256, 128, None, ep) == -1 and b"status" in e.msg
    assert L.qmoe_paged_attn(cp, 0, bp, ctypes.byref(q), A, 1 << 40, None, ep) == -1 and b"status" in e.msg
