"""What the paged caches' entries refuse, before anything is launched (no GPU: the context is never touched by a refused
call), and their sizes."""
import ctypes
import subprocess
import os

import pytest

from windlass_amd import _lib
from windlass_amd._lib import WL_E_ARG, WL_E_SHAPE, WL_E_UNSUPPORTED, ShapeError, load
from windlass_amd.backend import LayerDesc, PageRows, Pages, SparseOpts

CTX = ctypes.create_string_buffer(1 << 14)  # stands for a context: refusals come before its first use
BUF = (ctypes.c_char * 256)()
X = (ctypes.addressof(BUF) + 63) // 64 * 64
NULL = ctypes.c_void_p()


def desc(**kw):
    a = dict(d_K=X, d_V=X, d_bounds=X, d_table=X, pages=9, page=16, kv_heads=2, head_dim=64, sequences=4, table_pages=5)
    a.update(kw)
    return Pages(**a)


def call(name, seq=(0, 1), pos=(3, 0), rows=None, ctx=CTX, q=X, H=4, k=X, v=X, out=X, prefix=0, rope=64, opts=(1, 1, 1),
         sid=0, first=0, ids=(1, 2), pos0=0, T=1, p=None, r=None, o=None, L=None, x=X, **kw):
    L0 = load()
    p = ctypes.byref(desc(**kw)) if p is None else p
    r = ctypes.byref(PageRows(seq, pos, rows)) if r is None else r
    o = ctypes.byref(SparseOpts(*(opts or ()))) if o is None else o
    if name == "assign":
        return L0.wl_paged_assign_dev(ctx, p, sid, first, len(ids), (ctypes.c_int32 * len(ids))(*ids))
    if name == "store":
        return L0.wl_paged_store_dev(ctx, p, r, q, H, k, v, rope, 0, 10000.0, 1.0, None, out)
    if name == "read":
        return L0.wl_paged_read_dev(ctx, p, sid, pos0, T, k, v)
    if name == "attend":
        return L0.wl_paged_attention_dev(ctx, p, r, q, H, prefix, 1.0, out)
    if name == "sparse":
        return L0.wl_paged_sparse_dev(ctx, p, r, q, H, o, 1.0, out, None)
    L = LayerDesc(heads=H, kv_heads=2, head_dim=64) if L is None else L
    return L0.wl_layer_paged_dev(ctx, ctypes.byref(L), x, p, r, prefix, None if opts is None else o)


ALL = ["assign", "store", "read", "attend", "sparse", "layer"]
ROWS = ["store", "attend", "sparse", "layer"]


def test_sizes():
    f, g = load().wl_page_bytes, load().wl_page_bounds_bytes
    assert f(16, 8, 128) == 16 * 8 * 128 * 2 and f(256, 1, 64) == 256 * 64 * 2
    assert f(256, 1 << 17, 128) == 2 ** 33  # past 32 bits
    assert g(8, 128) == 8 * 128 * 4 and g(1 << 18, 64) == 1 << 26
    bad = [(8, 1, 64), (0, 1, 64), (-16, 1, 64), (48, 1, 64), (512, 1, 64), (16, 0, 64), (16, -1, 64), (16, 1, 96), (16, 1, 256),
           (16, 1 << 18, 128), (16, 1 << 30, 64)]
    assert [f(*b) for b in bad] == [0] * len(bad) and g(0, 64) == g(1, 80) == 0


def test_struct_layouts_match_the_header(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"wl_pages": Pages, "wl_page_rows": PageRows, "wl_sparse_opts": SparseOpts}
    src = tmp_path / "layout.c"
    lines = ['printf("%%zu\\n", offsetof(%s, %s));' % (n, f[0]) for n, s in structs.items() for f in s._fields_]
    lines += ['printf("%%zu\\n", sizeof(%s));' % n for n in structs]
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "windlass_hip.h"\nint main(void) {' + "\n".join(lines)
                   + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [getattr(s, f[0]).offset for s in structs.values() for f in s._fields_] + [ctypes.sizeof(s) for s in structs.values()]
    assert got == want


def test_entries_of_unequal_lengths():
    for a in (([0], [1, 2]), ([0, 1], [1]), ([0], [1], [1, 1])):
        with pytest.raises(ShapeError):
            PageRows(*a)


@pytest.mark.parametrize("name", ALL)
def test_null_arguments(name):
    names = {"assign": "ctx p", "store": "ctx p r q k v out", "read": "ctx p k v", "attend": "ctx p r q out",
             "sparse": "ctx p r o q out", "layer": "ctx p r x"}[name]
    for n in names.split():
        assert call(name, **{n: NULL}) == WL_E_ARG, n
    for n in ("d_K", "d_V", "d_table"):
        assert call(name, **{n: None}) == WL_E_ARG, n
    for n in ("d_K", "d_V", "d_bounds"):
        assert call(name, **{n: X + 8}) == WL_E_ARG, n
    assert call(name, d_table=X + 2) == WL_E_ARG


@pytest.mark.parametrize("name", ALL)
def test_pool_shapes(name):
    for hd in (32, 80, 96, 192, 256):
        assert call(name, head_dim=hd) == WL_E_UNSUPPORTED
    for kw in (dict(head_dim=0), dict(kv_heads=0), dict(kv_heads=-2), dict(kv_heads=1 << 30), dict(page=0), dict(page=8),
               dict(page=48), dict(page=512), dict(page=-16), dict(pages=0), dict(sequences=0), dict(table_pages=0),
               dict(pages=-1)):
        assert call(name, **kw) == WL_E_SHAPE, kw


@pytest.mark.parametrize("name", ROWS)
def test_entries(name):
    none = PageRows([0], [0])
    none.seq = None
    assert call(name, r=ctypes.byref(none)) == WL_E_ARG
    few = PageRows([0], [0])
    few.n = -1
    assert call(name, r=ctypes.byref(few)) == WL_E_SHAPE
    assert call(name, rows=(1, -1)) == WL_E_SHAPE
    for kw in (dict(seq=(0, 4)), dict(seq=(-1, 1)), dict(pos=(80, 0)), dict(pos=(-1, 0)), dict(pos=(79, 0), rows=(2, 1)),
               dict(pos=(2 ** 31 - 1, 0), rows=(2 ** 31 - 1, 1))):
        assert call(name, **kw) == WL_E_ARG, kw
    # a table of 2^31 positions and more: a position is 31 bits
    assert call(name, table_pages=2 ** 30, pos=(2 ** 31 - 1, 0), rows=(1, 1)) == WL_E_ARG
    assert call(name, table_pages=2 ** 30, pos=(0, 0), rows=(2 ** 24, 1)) == WL_E_SHAPE
    if name in ("store", "layer"):
        assert call(name, seq=(1, 1)) == WL_E_ARG
    for h in (3, -4, 1 << 30) + (() if name == "store" else (0,)):
        assert call(name, H=h) == WL_E_SHAPE, h


def test_prefixes():
    for name in ("attend", "layer"):
        kw = dict(opts=None) if name == "layer" else {}
        for prefix in (-16, 8, 17, 32):
            assert call(name, prefix=prefix, pos=(31, 40), **kw) == WL_E_ARG, prefix
    assert call("layer", prefix=16, pos=(31, 40)) == WL_E_ARG  # and a choice of pages


def test_choices():
    for name in ("sparse", "layer"):
        assert call(name, d_bounds=None) == WL_E_ARG
        for o in ((-1, 1, 1), (0, 0, 4), (0, 1, -1), (2 ** 30, 1, 2 ** 30), (2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1)):
            assert call(name, opts=o) == WL_E_ARG, o


def test_rotations():
    for n in (-2, 3, 66, 128):
        assert call("store", rope=n) == WL_E_SHAPE


def test_table_entries():
    for kw in (dict(sid=-1), dict(sid=4), dict(first=-1), dict(first=4), dict(first=2 ** 31 - 1), dict(ids=(9,)), dict(ids=(-2,))):
        assert call("assign", **kw) == WL_E_ARG, kw
    for kw in (dict(sid=4), dict(pos0=-1), dict(pos0=80), dict(T=81)):
        assert call("read", **kw) == WL_E_ARG, kw
    assert call("read", T=-1) == WL_E_SHAPE


def test_layers_of_other_shapes():
    assert call("layer", opts=None, L=LayerDesc(heads=4, kv_heads=1, head_dim=64)) == WL_E_SHAPE
    assert call("layer", opts=None, L=LayerDesc(heads=4, kv_heads=2, head_dim=128)) == WL_E_SHAPE
    assert call("layer", opts=None, rows=(0, 0)) == WL_E_SHAPE


def test_every_entry_is_bound():
    assert {n for n in _lib.SIGNATURES if "page" in n} == {
        "wl_page_bytes", "wl_page_bounds_bytes", "wl_paged_assign_dev", "wl_paged_store_dev", "wl_paged_read_dev",
        "wl_paged_attention_dev", "wl_paged_sparse_dev", "wl_layer_paged_dev"}


@pytest.mark.parametrize("make", [
    lambda v: PageRows([v], [0]), lambda v: PageRows([0], [v]), lambda v: PageRows([0], [0], [v]),
    lambda v: SparseOpts(v, 1, 1), lambda v: SparseOpts(1, v, 1), lambda v: SparseOpts(1, 1, v),
    lambda v: desc(pages=v), lambda v: desc(page=v), lambda v: desc(kv_heads=v), lambda v: desc(head_dim=v),
    lambda v: desc(sequences=v), lambda v: desc(table_pages=v)])
def test_numbers_past_32_bits(make):
    """2^32 + 1 would reach the library as 1."""
    for v in ((1 << 32) + 1, 1 << 31, -(1 << 31) - 1):
        with pytest.raises(ShapeError):
            make(v)
    make((1 << 31) - 1)
