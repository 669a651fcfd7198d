"""What the C entries of drafting and forking on the 8-bit cache refuse on the host, before any launch.  No GPU needed."""
import ctypes

import pytest

from smoltts_b200 import _capi_lm as cl
from test_cache8_host import call, good

P = 1 << 20


def tree(**over):
    a = dict(n_tokens=5, n_seqs=2, max_new=3, seq_start=P, seq_pos0=P, parents=P, positions=P, sees=P, words=1, err=P)
    a.update(over)
    return cl.load().smol_lm_cache8_tree(ctypes.byref(cl.SmolLmCache8Tree(**a)), None)


@pytest.mark.parametrize("field,value,code", [("n_tokens", 0, -1), ("n_seqs", 0, -1), ("max_new", 0, -1), ("max_new", 4097, -5), ("max_new", 33, -1), ("words", 0, -1), ("seq_start", None, -1),
                                              ("seq_pos0", None, -1), ("parents", None, -1), ("positions", None, -1), ("sees", None, -1), ("err", None, -1)])
def test_tree(field, value, code):
    assert tree(**{field: value}) == code
    assert b"smol_lm_cache8_tree" in cl.load().smol_lm_last_error()


def caches(n=2):
    c = (cl.SmolLmCache8 * n)()
    for i in range(n):
        at = P * (1 + 8 * i)
        c[i] = cl.SmolLmCache8(k=at, v=at + P, k_scale=at + 2 * P, v_scale=at + 3 * P, n_pages=4, page_size=32, kv_heads=2, dim=64, vdim=48, err=P)
    return c


def keep(c, **over):
    a = dict(n_seqs=1, max_pages=2, max_keep=3, seq_pos0=P, block_table=P, rows=P, counts=P)
    a.update(over)
    return cl.load().smol_lm_cache8_keep(c, len(c), ctypes.byref(cl.SmolLmCache8Keep(**a)), None)


@pytest.mark.parametrize("field,value,code", [("n_seqs", 0, -1), ("n_seqs", 65536, -5), ("max_pages", 0, -1), ("max_keep", 0, -1), ("seq_pos0", None, -1), ("block_table", None, -1), ("rows", None, -1),
                                              ("counts", None, -1)])
def test_keep(field, value, code):
    assert keep(caches(), **{field: value}) == code
    assert b"smol_lm_cache8_keep" in cl.load().smol_lm_last_error()


def copy(c, src, dst, n=None):
    n = len(src) if n is None else n
    ints = ctypes.c_int32 * max(len(src), 1)
    return cl.load().smol_lm_cache8_copy_pages(c, len(c), ints(*src), ints(*dst), n, None)


@pytest.mark.parametrize("src,dst", [([0], [4]), ([0], [-1]), ([4], [0]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([1], [1]), ([0, 2], [3, 2])])
def test_pages_that_cannot_be_copied(src, dst):
    assert copy(caches(), src, dst) == -1
    assert b"smol_lm_cache8_copy_pages" in cl.load().smol_lm_last_error()


def test_many_pages_are_looked_at_too():
    c = caches(1)
    c[0].n_pages = 1000
    src, dst = list(range(100)), list(range(500, 600))
    for at, page in ((99, 500), (3, 1000), (50, 99)):
        bad = list(dst)
        bad[at] = page
        assert copy(c, src, bad) == -1
    src[70] = 510
    assert copy(c, src, dst) == -1


def test_no_pages_are_no_call():
    assert copy(caches(), [], []) == 0 and copy(caches(), [], [], n=-1) == -1


@pytest.mark.parametrize("which", ["keep", "copy"])
@pytest.mark.parametrize("field,value,code", [("page_size", 16, -1), ("kv_heads", 1, -1), ("dim", 48, -1), ("vdim", 64, -1), ("n_pages", 5, -1), ("k", None, -1), ("v", 8, -1), ("err", None, -1), ("dim", 300, -4),
                                              ("k", P, -1), ("v", 2 * P, -1), ("k_scale", 3 * P, -1), ("k_page", 8192, -1), ("v_scale_page", 64, -1)])
def test_layers_of_one_shape_and_none_twice(which, field, value, code):
    c = caches()
    setattr(c[1], field, value)
    assert (keep(c) if which == "keep" else copy(c, [0], [1])) == code


def test_no_caches():
    lib = cl.load()
    a = cl.SmolLmCache8Keep(n_seqs=1, max_pages=2, max_keep=3, seq_pos0=P, block_table=P, rows=P, counts=P)
    assert lib.smol_lm_cache8_keep(None, 1, ctypes.byref(a), None) == -1 and lib.smol_lm_cache8_keep(caches(), 0, ctypes.byref(a), None) == -1
    assert lib.smol_lm_cache8_keep(caches(), 1, None, None) == -1
    assert lib.smol_lm_cache8_copy_pages(None, 1, P, P, 1, None) == -1 and lib.smol_lm_cache8_copy_pages(caches(), 1, None, P, 1, None) == -1


@pytest.mark.parametrize("fields", [dict(positions=P), dict(positions=P, n_axes=-1), dict(n_axes=1), dict(axis=P), dict(n_axes=2, axis=P)])
def test_positions_and_axes_come_together(fields):
    cache, batch, app, att = good()
    for k, v in fields.items():
        setattr(app, k, v)
    assert call(cl.load(), "append", cache, batch, app, att) == -1


@pytest.mark.parametrize("fields", [dict(tree_positions=P), dict(tree_sees=P, tree_words=1), dict(tree_positions=P, tree_sees=P), dict(tree_positions=P, tree_sees=P, tree_words=-1)])
def test_a_tree_has_positions_and_bits(fields):
    cache, batch, app, att = good()
    for k, v in fields.items():
        setattr(att, k, v)
    assert call(cl.load(), "attend", cache, batch, app, att) == -1
