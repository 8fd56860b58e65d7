"""Drafted tokens on the paged cache without a GPU: the refusals of
qmoe_paged_tree_build, _attn_tree, _append_rotary, _follow and _keep, which
come back as -1 with a message before the device is touched (the pointers here
are no memory at all)."""
import ctypes
import os
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT, load_pkg
from test_paged import A, BAD_ATTN, BAD_CACHE, CSRC, batch, cache, query

BIG = 1 << 40


def tree(pkg, **kw):
    f = dict(depths=A, seen=A, words=2)
    f.update(kw)
    return pkg.QmoePagedTree(**f)


def rotary(pkg, **kw):
    f = dict(q=A, k=A, v=A, out=A + 4096, q_token_stride=1024, q_head_stride=128, k_token_stride=256, k_head_stride=128,
             v_token_stride=256, v_head_stride=128, out_token_stride=1024, out_head_stride=128, src_dtype=pkg.BF16, n_heads=8,
             freqs=A, rot=32, interleaved=0, q_norm=A, k_norm=A, eps=1e-6)
    f.update(kw)
    return pkg.QmoePagedRotary(**f)


class Calls:
    """each call with right arguments, but for those given"""

    def __init__(self, pkg, c=None, b=None, q=None, r=None, t=None):
        self.pkg, self.L, self.e = pkg, pkg.lib(), pkg.QmoeErr()
        self.parts = (c if c is not None else cache(pkg), b if b is not None else batch(pkg), q if q is not None else query(pkg),
                      r if r is not None else rotary(pkg), t if t is not None else tree(pkg))
        self.c, self.b, self.q, self.r, self.t = (ctypes.byref(x) for x in self.parts)

    def build(self, parents=A, starts=A, n=5, n_seqs=3, t=True):
        return self.L.qmoe_paged_tree_build(parents, starts, n, n_seqs, self.t if t else None, None, ctypes.byref(self.e))

    def attn(self, layer=0, b=True, q=True, t=True, ws=A, size=BIG):
        return self.L.qmoe_paged_attn_tree(self.c, layer, self.b if b else None, self.q if q else None, self.t if t else None,
                                           ws, size, None, ctypes.byref(self.e))

    def rotary(self, layer=0, b=True, r=True, t=True):
        return self.L.qmoe_paged_append_rotary(self.c, layer, self.b if b else None, self.r if r else None,
                                               self.t if t else None, None, ctypes.byref(self.e))

    def follow(self, t=True, parents=A, tokens=A, chosen=A, starts=A, n=5, n_seqs=3, rows=A, counts=A, last=A):
        return self.L.qmoe_paged_follow(self.t if t else None, parents, tokens, chosen, starts, n, n_seqs, rows, counts, last,
                                        None, ctypes.byref(self.e))

    def keep(self, b=True, rows=A, counts=A, status=A, ws=A, size=BIG):
        return self.L.qmoe_paged_keep(self.c, self.b if b else None, rows, counts, status, ws, size, None, ctypes.byref(self.e))

    def refused(self, rc, msg):
        assert rc == -1 and msg in self.e.msg.decode(), (rc, self.e.msg, msg)


@pytest.mark.parametrize("kw,msg", BAD_CACHE, ids=[f"{list(k)[0]}_{i}" for i, (k, _) in enumerate(BAD_CACHE)])
def test_bad_caches_are_refused(kw, msg):
    pkg = load_pkg()
    x = Calls(pkg, c=cache(pkg, **kw))
    for call in (x.attn, x.rotary, x.keep):
        x.refused(call(), msg)
    assert pkg.lib().qmoe_paged_ws_bytes(x.c, pkg.PAGED_KEEP, 5, 3, 0) == 0


@pytest.mark.parametrize("ckw,bkw,qkw,layer,msg", BAD_ATTN, ids=[str(i) for i in range(len(BAD_ATTN))])
def test_bad_attention_calls_are_refused(ckw, bkw, qkw, layer, msg):
    pkg = load_pkg()
    x = Calls(pkg, c=cache(pkg, **ckw), b=batch(pkg, **bkw), q=query(pkg, **qkw))
    x.refused(x.attn(layer), msg)


@pytest.mark.parametrize("kw,msg", [(dict(words=0), "words 0"), (dict(words=33), "words 33"), (dict(words=-1), "words -1"),
                                    (dict(depths=None), "depths is NULL"), (dict(seen=None), "seen is NULL"),
                                    (dict(depths=A + 2), "aligned"), (dict(seen=A + 1), "aligned")])
def test_bad_trees_are_refused(kw, msg):
    pkg = load_pkg()
    x = Calls(pkg, t=tree(pkg, **kw))
    for call in (x.build, x.attn, x.rotary, x.follow):
        x.refused(call(), msg)


def test_every_null_argument_is_named():
    pkg = load_pkg()
    x = Calls(pkg)
    for call in (x.build, x.attn, x.follow):
        x.refused(call(t=False), "tree is NULL")
    x.refused(x.build(parents=None), "parents is NULL")
    x.refused(x.build(starts=None), "starts is NULL")
    for call in (x.attn, x.rotary, x.keep):
        x.refused(call(b=False), "batch is NULL")
    x.refused(x.attn(q=False), "query is NULL")
    x.refused(x.attn(ws=None), "workspace is NULL")
    x.refused(x.rotary(r=False), "rotary is NULL")
    for name, arg in (("parents", "parents"), ("tokens", "tokens"), ("chosen", "chosen"), ("rows", "rows"), ("counts", "counts"),
                      ("next", "last"), ("starts", "starts")):
        x.refused(x.follow(**{arg: None}), f"{name} is NULL")
    for name in ("rows", "counts", "status"):
        x.refused(x.keep(**{name: None}), f"{name} is NULL")
    x.refused(x.keep(ws=None), "workspace is NULL")
    x.parts[1].starts = None
    for call in (x.attn, x.rotary, x.keep):
        x.refused(call(), "starts is NULL")
    # a NULL err is allowed
    assert x.L.qmoe_paged_tree_build(A, A, 5, 3, None, None, None) == -1
    assert x.L.qmoe_paged_keep(None, x.b, A, A, A, A, BIG, None, None) == -1


@pytest.mark.parametrize("kw,msg", [
    (dict(k=None), "k is NULL"), (dict(v=None), "v is NULL"), (dict(q=None), "q is NULL"), (dict(out=None), "out is NULL"),
    (dict(freqs=None), "freqs is NULL"), (dict(rot=0), "rot 0"), (dict(rot=130), "rot 130"), (dict(rot=33), "rot 33"),
    (dict(rot=-2), "rot -2"), (dict(interleaved=2), "interleaved"), (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(src_dtype=7), "dtype"), (dict(n_heads=-1), "heads"), (dict(n_heads=1 << 29), "heads"),
    (dict(k=A + 8), "aligned"), (dict(v=A + 4), "aligned"), (dict(q=A + 2), "aligned"), (dict(out=A + 4100), "aligned"),
    (dict(freqs=A + 2), "aligned"), (dict(q_norm=A + 1), "aligned"), (dict(k_norm=A + 3), "aligned"),
    (dict(q_token_stride=1025), "q_token_stride"), (dict(q_head_stride=-128), "q_head_stride"),
    (dict(k_token_stride=260), "k_token_stride"), (dict(k_head_stride=1), "k_head_stride"), (dict(v_token_stride=-8), "v_token_stride"),
    (dict(v_head_stride=132), "v_head_stride"), (dict(out_token_stride=1028), "out_token_stride"),
    (dict(out_head_stride=4), "out_head_stride"), (dict(out_token_stride=512), "overlap"), (dict(out_head_stride=0), "overlap"),
    (dict(out=A, out_token_stride=2048), "out is q"), (dict(out=A, q_head_stride=256), "out is q"),
    (dict(out=A, src_dtype=0), "out is q"),
])
def test_bad_rotary_calls_are_refused(kw, msg):
    pkg = load_pkg()
    x = Calls(pkg, r=rotary(pkg, **kw))
    x.refused(x.rotary(), msg)
    x.refused(x.rotary(t=False), msg)


def test_other_bad_calls_are_refused():
    pkg = load_pkg()
    x = Calls(pkg)
    x.refused(x.rotary(layer=2), "layer 2")
    x.refused(x.rotary(layer=-1), "layer -1")
    for call in (x.build, x.follow):
        x.refused(call(n=-1), "n = -1")
        x.refused(call(n=(1 << 30) + 1), "out of range")
        x.refused(call(n_seqs=-1), "n_seqs")
        x.refused(call(n_seqs=65537), "n_seqs")
    x.refused(x.keep(status=A + 2), "aligned")
    for kw, msg in ((dict(n_seqs=1025), "n_seqs"), (dict(n_seqs=-1), "n_seqs"), (dict(slots=None, n_seqs=5), "slots"),
                    (dict(n=-1), "n = -1"), (dict(status=A + 2), "status")):
        y = Calls(pkg, b=batch(pkg, **kw))
        y.refused(y.keep(), msg)
        y.refused(y.rotary(), msg) if "n_seqs" not in kw or kw["n_seqs"] != 1025 else None
    need = x.L.qmoe_paged_ws_bytes(x.c, pkg.PAGED_KEEP, 5, 3, 0)
    assert need > 0
    x.refused(x.keep(size=need - 1), "workspace")
    x.refused(x.keep(ws=A + 8, size=need), "workspace")
    assert x.L.qmoe_paged_ws_bytes(x.c, pkg.PAGED_KEEP, 5, 1025, 0) == 0
    assert x.L.qmoe_paged_ws_bytes(x.c, pkg.PAGED_KEEP, -1, 3, 0) == 0
    assert x.L.qmoe_paged_ws_bytes(x.c, 6, 5, 3, 8) == 0
    need = x.L.qmoe_paged_ws_bytes(x.c, pkg.PAGED_ATTN_TREE, 5, 3, 8)
    assert need > 0
    x.refused(x.attn(size=need - 1), "workspace")
    x.refused(x.attn(ws=A + 8, size=need), "workspace")


def test_calls_with_nothing_to_do_touch_nothing():
    pkg = load_pkg()
    for kw in (dict(n=0), dict(n_seqs=0)):
        x = Calls(pkg, b=batch(pkg, **kw), r=rotary(pkg, k=None, v=None, q=None, out=None, freqs=None))
        assert x.rotary() == 0 and x.attn(ws=None, size=0) == 0
        assert x.build(**kw) == 0
    assert Calls(pkg).follow(n_seqs=0) == 0


def test_packed_structs_are_the_header_s():
    """a call's structs as the binding packs them, field by field against the ctypes ones"""
    pkg = load_pkg()
    q = sys.modules["qmoe_amd.qmoe"]
    for packed, cls, values in (
            (q._BATCH, pkg.QmoePagedBatch, (1, 2, 3, 4, 5)),
            (q._QUERY, pkg.QmoePagedQuery, (1, 2, 3, 4, 5, 6, 7, 8, 9, 1, 0.5)),
            (q._ROTARY, pkg.QmoePagedRotary, tuple(range(1, 13)) + (13, 14, 15, 16, 1, 18, 19, 0.25)),
            (q._TREE, pkg.QmoePagedTree, (1, 2, 3))):
        raw = packed.pack(*values).ljust(ctypes.sizeof(cls), b"\0")
        got = cls.from_buffer_copy(raw)
        assert tuple(getattr(got, f) for f, _ in cls._fields_) == values


def test_trees_of_other_tensors_are_refused():
    import torch
    pkg = load_pkg()
    d, s = torch.zeros(5, dtype=torch.int32), torch.zeros(5, 2, dtype=torch.int32)
    pkg.DraftTree(None, None, d, s)
    for bad in ((d.float(), s), (d, s.float()), (d.long(), s), (d[:4], s), (d, s[0]), (d, s.t().contiguous().t()), (d[::2], s[::2])):
        with pytest.raises(pkg.QmoeError, match="depths"):
            pkg.DraftTree(None, None, *bad)


def test_workspaces_hold_what_their_launches_take(tmp_path):
    """every call's places in its workspace, of trees and in causal order, over types, head shapes, tables, windows, sequences
    and rows (tests/c/paged_plan.cpp)"""
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ is not available")
    exe = str(tmp_path / "paged_plan")
    r = subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Wextra", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC,
                        os.path.join(ROOT, "tests", "c", "paged_plan.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


@pytest.mark.parametrize("shape,pages,nodes,index", [((16, 2, 128), 33, 4, 25559040), ((4, 2, 64), 250, 12, 19464192)])
def test_the_index_of_32_row_units_is_inside(shape, pages, nodes, index):
    """65 sequences of 17 to 32 rows on few keys (of the table, or of a window of 700): units of 32 rows, whose index begins
    at byte `index` (1536 slots of 32 rows of 8 + 4 * 128 bytes; 2304 of 8 + 4 * 64) and has 16 bytes a sequence"""
    pkg = load_pkg()
    h, kvh, hd = shape
    c = cache(pkg, page_stride=16 * kvh * hd, row_stride=kvh * hd, head_stride=hd, n_kv_heads=kvh, head_dim=hd, table_stride=pages,
              max_pages=pages, n_slots=65)
    for call in (pkg.PAGED_ATTN_TREE, pkg.PAGED_ATTN):
        assert pkg.lib().qmoe_paged_ws_bytes(ctypes.byref(c), call, 65 * nodes, 65, h) >= index + 16 * 65


def hosted(pkg):
    """a PagedCache whose tensors would lie on the host: its checks, which come before any call"""
    import torch
    c = object.__new__(pkg.PagedCache)
    c._torch, c._index, c.device, c._i32, c._f32 = torch, -1, torch.device("cpu"), torch.int32, torch.float32
    c.n_layers, c.kvh, c.hd, c.dtype = 1, 2, 64, torch.bfloat16
    c._own, c._src = (torch.bfloat16,), (torch.bfloat16, torch.float32)
    return c


def test_follow_checks_the_tree_s_own_tensors():
    """a DraftTree of the caller's: parents and starts are read as int32 vectors of n and m + 1 entries"""
    import torch
    pkg = load_pkg()
    c = hosted(pkg)
    d, seen, parents, starts = (torch.zeros(n, dtype=torch.int32) for n in (5, 5, 5, 3))
    tree = lambda p=parents, s=starts: pkg.DraftTree(p, s, d, seen.view(5, 1))
    tokens = torch.zeros(5, dtype=torch.int32)
    wide = torch.zeros(10, dtype=torch.int32)
    for bad, msg in ((tree(p=None), "parents"), (tree(p=parents.long()), "parents"), (tree(p=parents[:4]), "parents"),
                     (tree(p=wide[::2]), "parents"), (tree(p=parents.float()), "parents"),
                     (tree(s=None), "starts"), (tree(s=starts[:0]), "starts"), (tree(s=starts.long()), "starts"),
                     (tree(s=wide[:6:2]), "starts"), (tree(s=starts.view(3, 1)), "starts"), (None, "tree")):
        with pytest.raises(pkg.QmoeError, match=msg):
            c.follow(bad, tokens, tokens)


@pytest.mark.parametrize("kw", [dict(window=None), dict(window=0.0), dict(window=""), dict(sinks=None), dict(sinks=[]),
                                dict(window=3.0), dict(window=5, sinks=None)], ids=str)
def test_windows_that_are_no_integers_are_refused(kw):
    """also those that are false, which are no 0"""
    import torch
    pkg = load_pkg()
    c, starts = hosted(pkg), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    tree = pkg.DraftTree(None, starts, torch.zeros(1, dtype=torch.int32), torch.ones(1, 1, dtype=torch.int32))
    for call in (lambda: c.attend(0, q, starts, **kw), lambda: c.attend_tree(0, q, tree, **kw)):
        with pytest.raises(TypeError):
            call()


def test_structs_of_the_binding_are_typed():
    """lib()'s paged calls take a struct as it is or by reference, and no other struct in its place"""
    pkg = load_pkg()
    L, e = pkg.lib(), pkg.QmoeErr()
    c, b, q = cache(pkg), batch(pkg, n=0), query(pkg)
    for r in (lambda x: x, ctypes.byref):
        assert L.qmoe_paged_append(r(c), 0, r(b), A, A, pkg.BF16, 256, 128, 256, 128, None, r(e)) == 0, e.msg
        assert L.qmoe_paged_attn(r(c), 0, r(b), r(q), A, BIG, None, r(e)) == 0, e.msg
        with pytest.raises(ctypes.ArgumentError):
            L.qmoe_paged_append(r(c), 0, r(q), A, A, pkg.BF16, 256, 128, 256, 128, None, r(e))
        with pytest.raises(ctypes.ArgumentError):
            L.qmoe_paged_attn(r(c), 0, r(q), r(b), A, BIG, None, r(e))
