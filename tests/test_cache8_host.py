"""The 8-bit cache's C entries check their arguments on the host, before any launch."""
import ctypes

import pytest

from smoltts_b200 import _capi_lm as cl


def good():
    p = 1 << 20
    cache = cl.SmolLmCache8(k=p, v=p, k_scale=p, v_scale=p, n_pages=4, page_size=32, kv_heads=2, dim=64, vdim=48, err=p)
    batch = cl.SmolLmCache8Batch(n_tokens=3, n_seqs=1, max_pages=2, max_new=3, max_len=40, seq_start=p, seq_pos0=p, block_table=p)
    app = cl.SmolLmCache8Append(dtype=0, k=p, v=p, k_row=128, k_head=64, v_row=96, v_head=48, rot_mult=1.0)
    att = cl.SmolLmCache8Attend(dtype=0, heads=4, q=p, out=p, q_row=256, q_head=64, out_row=192, out_head=48, scale=0.1, out_scale=1.0)
    return cache, batch, app, att


def call(lib, which, cache, batch, app, att):
    if which == "append":
        return lib.smol_lm_cache8_append(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(app), None)
    return lib.smol_lm_cache8_attend(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(att), None, 0, None)


@pytest.mark.parametrize("which", ["append", "attend"])
@pytest.mark.parametrize("part,field,value,code", [
    ("cache", "k", None, -1), ("cache", "v_scale", None, -1), ("cache", "err", None, -1), ("cache", "k", 8, -1), ("cache", "page_size", 24, -1), ("cache", "page_size", 0, -1),
    ("cache", "n_pages", 0, -1), ("cache", "kv_heads", 0, -1), ("cache", "dim", 0, -1), ("cache", "dim", 257, -4), ("cache", "vdim", 300, -4), ("cache", "k_page", 24, -1),
    ("batch", "n_tokens", 0, -1), ("batch", "n_seqs", 0, -1), ("batch", "n_seqs", 65536, -5), ("batch", "max_new", 0, -1), ("batch", "max_pages", 0, -1), ("batch", "seq_start", None, -1),
    ("batch", "block_table", None, -1)])
def test_cache_and_batch(which, part, field, value, code):
    lib = cl.load()
    args = dict(zip(("cache", "batch", "app", "att"), good()))
    setattr(args[part], field, value)
    assert call(lib, which, **args) == code
    assert b"smol_lm_cache8_" + which.encode() in lib.smol_lm_last_error()


@pytest.mark.parametrize("which,field,value,code", [
    ("append", "dtype", 2, -1), ("append", "k", None, -1), ("append", "rot_dims", 3, -1), ("append", "rot_dims", 66, -1), ("append", "rot_dims", 32, -1), ("append", "q", 4096, -1),
    ("append", "q_out", 4096, -1), ("attend", "dtype", -1, -1), ("attend", "heads", 3, -1), ("attend", "heads", 0, -1), ("attend", "window", -1, -1), ("attend", "first", -2, -1),
    ("attend", "softcap", -1.0, -1), ("attend", "softcap", float("nan"), -1), ("attend", "dist_r1", 4096, -1), ("attend", "q", None, -1), ("attend", "out", None, -1)])
def test_operators(which, field, value, code):
    lib = cl.load()
    cache, batch, app, att = good()
    setattr(app if which == "append" else att, field, value)
    assert call(lib, which, cache, batch, app, att) == code


def test_null_structs():
    lib = cl.load()
    cache, batch, app, att = good()
    assert lib.smol_lm_cache8_append(None, ctypes.byref(batch), ctypes.byref(app), None) == -1
    assert lib.smol_lm_cache8_attend(ctypes.byref(cache), None, ctypes.byref(att), None, 0, None) == -1
    assert lib.smol_lm_cache8_workspace_bytes(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(att), None) == -1


def lm_config(**over):
    c = dict(dtype=0, vocab=64, width=32, n_layers=1, n_runs=1, page_size=32, max_step_tokens=64, max_step_seqs=2, max_want=8, max_context=256, use_graph=1, embed_scale=1.0,
             norm_eps=1e-5, kv_bits=8)
    c.update(over)
    layers = (cl.SmolLmLayer * 1)()
    layers[0].mixer, layers[0].heads, layers[0].kv_heads, layers[0].dim, layers[0].vdim = 0, 4, 2, 24, 64
    return cl.SmolLmConfig(**c), layers


def test_engine_pages_of_codes():
    """A page: 2 heads x 32 positions x (24 rounded up to 32, 64) codes, and as many scales as 16-position blocks for keys and values."""
    lib, h, runs = cl.load(), ctypes.c_void_p(), (ctypes.c_int32 * 1)(0)

    def create(layers, cfg):
        return lib.smol_lm_create(ctypes.byref(cfg), layers, runs, ctypes.byref(h))

    cfg, layers = lm_config()
    assert create(layers, cfg) == 0
    assert lib.smol_lm_page_bytes(h) == 2 * 32 * (32 + 64) + 2 * 2 * 2 * 4
    lib.smol_lm_destroy(h)
    layers[0].window, layers[0].first_visible = 10, 4
    assert create(layers, cfg) == 0
    lib.smol_lm_destroy(h)
    assert create(layers, lm_config(kv_bits=16)[0]) == -4 and create(layers, lm_config(kv_bits=4)[0]) == -1 and create(layers, lm_config(page_size=40)[0]) == -1
    layers[0].first_visible = -1
    assert create(layers, cfg) == -4
    layers[0].first_visible, layers[0].n_maps = 0, 2
    assert create(layers, cfg) == -4
    layers[0].n_maps, layers[0].dim = 0, 257
    assert create(layers, cfg) == -4
    layers[0].dim, layers[0].mixer, layers[0].rot_dim, layers[0].q_rank, layers[0].kv_rank = 24, 2, 0, 8, 8
    assert create(layers, cfg) == -4
