"""What is measured of drafting and forking on the 8-bit key/value cache: trees of drafted tokens, rows whose rotary positions are not
their places in the cache, and rows and pages that move.

A cache holds, per page, key/value head and position, a row of e4m3 codes for the key and one for the value; 16 positions that
follow one another share one power-of-two scale per head (keys and values each their own).

* ``tree`` -- of each drafted row's parent among the rows of its sequence: its position (behind the context, by its depth) and a bit
  for every row of the sequence that is the row itself or in front of it on its path.
* ``append`` -- rotates the step's keys and queries by positions that are given, one per axis (time, height, width; or a drafted
  row's depth), every pair of coordinates by the axis it belongs to, and writes keys and values behind the context.
* ``attend`` -- softmax attention of drafted rows: over the context in the cache, behind a window if asked, and over the drafted
  rows that their bits name; soft cap, distance penalties and a sink logit.
* ``keep`` -- moves the rows of the accepted path, of every layer's cache, together behind the context.
* ``copy`` -- copies pages of every layer's cache, as forking a sequence does.

Heads and head sizes are those of the language models' benchmark configurations (12 heads over 4 of 64 or 128) or generic.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 16                       # positions that share a scale
LEAST, MOST = -110, 2.0 ** 100   # least exponent of a scale; magnitudes above are clamped


def listed():
    return [
        # one chat, its draft tree: latency
        dict(name="tree_25", kind="tree", seqs=1, new=25, context=2047, shape="random"),
        # a serving batch's trees, unequal sizes
        dict(name="tree_batch_64", kind="tree", seqs=64, new=64, context=8192, shape="random"),
        # a serving batch's drafted rows, each at the position its depth gives it, slices of one fused projection
        dict(name="append_drafts_32", kind="append", seqs=32, new=16, context=4096, heads=32, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16", rot=128, half=True, fused=True, axes=1, mix=False),
        # prompts of text and video: time, height and width
        dict(name="append_video_2", kind="append", seqs=2, new=6001, context=70, heads=32, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16", rot=128, half=True, fused=True, axes=3, mix=True),
        # one chat, one layer: latency
        dict(name="attend_tree_chat", kind="attend", seqs=1, new=16, context=2047, heads=12, kv_heads=4, dim=64, vdim=64, page=64, dtype="bfloat16", window=0, first=0, options="plain", shape="random"),
        # a serving batch, four drafted rows each behind a window whose first tokens stay visible, soft cap, linear penalty and sink
        dict(name="attend_tree_few", kind="attend", seqs=48, new=4, context=20000, heads=32, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16", window=4000, first=4, options="capped", shape="fan"),
        # a serving batch with large trees behind unequal contexts
        dict(name="attend_tree_batch", kind="attend", seqs=32, new=64, context=8192, heads=32, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16", window=0, first=0, options="plain", shape="random"),
        # the float32 engine: logarithmic penalty and sink, odd head sizes
        dict(name="attend_tree_f32", kind="attend", seqs=3, new=21, context=901, heads=12, kv_heads=4, dim=80, vdim=72, page=32, dtype="float32", window=0, first=0, options="penalty", shape="random"),
        # one chat: the accepted path of its tree, in every layer
        dict(name="keep_chat", kind="keep", layers=12, seqs=1, new=48, keep=4, context=2043, heads=12, kv_heads=4, dim=64, vdim=64, page=64),
        # a serving batch
        dict(name="keep_batch_64", kind="keep", layers=28, seqs=64, new=64, keep=7, context=250, heads=32, kv_heads=8, dim=128, vdim=128, page=64),
        # one chat is forked: its last page, in every layer
        dict(name="copy_fork", kind="copy", layers=12, pairs=1, kv_heads=4, dim=64, vdim=64, page=64),
        # beams change places, or a pool is tidied up
        dict(name="copy_pages_128", kind="copy", layers=28, pairs=128, kv_heads=8, dim=128, vdim=128, page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["tree", "append", "attend", "attend", "keep", "copy"])
    shape = rng.choice(["random", "random", "fan", "chain"])
    if kind == "tree":
        seqs = _log_int(rng, 1, 64)
        return dict(kind=kind, seqs=seqs, new=_log_int(rng, 1, min(256, 4096 // seqs)), context=_log_int(rng, 1, 100000), shape=shape)
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 160, 256])
    vdim = dim if rng.random() < 0.7 else rng.choice([40, 64, 72, 128])
    case = dict(kind=kind, kv_heads=kv_heads, dim=dim, vdim=vdim, page=rng.choice([16, 32, 64, 128]))
    if kind == "copy":
        case["layers"] = _log_int(rng, 1, 28)
        bytes_of_page = case["layers"] * kv_heads * case["page"] * (dim + vdim)
        case["pairs"] = _log_int(rng, 1, max(1, min(600, 400_000_000 // bytes_of_page)))
        return case
    case["heads"] = heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    if kind == "keep":
        case.update(layers=_log_int(rng, 1, 28), seqs=_log_int(rng, 1, 64), new=_log_int(rng, 1, 100), context=_log_int(rng, 1, 300))
        case["keep"] = rng.randint(1, min(case["new"], 16))
        return case
    case["dtype"] = "float32" if rng.random() < 0.2 else "bfloat16"
    if kind == "append":
        case["seqs"] = _log_int(rng, 1, 32)
        case["new"] = _log_int(rng, 1, 8192 // case["seqs"])
        case["context"] = _log_int(rng, 1, 4096 // case["seqs"])
        case.update(rot=rng.choice([16, dim // 2 // 2 * 2, dim]), half=rng.random() < 0.5, fused=rng.random() < 0.5, axes=rng.choice([1, 2, 3, 3, 4]), mix=rng.random() < 0.5)
        return case
    case["seqs"] = seqs = _log_int(rng, 1, 64)
    case["new"] = new = _log_int(rng, 1, min(256, 2048 // seqs))
    room = (16_000_000_000 if case["dtype"] == "float32" else 64_000_000_000) // (seqs * new * heads * (dim + vdim))       # positions: at most half the work of the largest listed case
    case["context"] = _log_int(rng, 1, max(1, min(131072 // seqs, room)))
    window = rng.choice([0, 0, _log_int(rng, 1, 4000)])
    case.update(window=window, first=rng.choice([0, 1, 4, 33]) if window else 0, options=rng.choice(["plain", "plain", "capped", "penalty"]), shape=shape)
    return case


# ---------------------------------------------------------------------------------------------- what a case holds

def _lens(case):
    """(cached before, new) of every sequence, the first one the longest."""
    c, n, S = case["context"], case["new"], case["seqs"]
    return [(c - (c // 2) * s // S if S > 1 else c, n if n < 4 else max(1, n - (n // 3) * s // S)) for s in range(S)]


def _pages(case):
    return [-(-(c + n) // case["page"]) for c, n in _lens(case)]


def _words(case):
    return -(-case["new"] // 32)


def _seq_rng(seed, s):
    return np.random.default_rng([int(seed), 77, s])


def _parents(case, n, rng):
    """A row's parent among the rows of its sequence, -1 for one that follows the context."""
    i = np.arange(n)
    if case["shape"] == "chain":
        return i - 1
    if case["shape"] == "fan":
        return np.where(i == 0, -1, (i - 1) // 3)
    return np.floor(np.sqrt(rng.random(n)) * (i + 1)).astype(np.int64) - 1


def _tree_of(parents):
    """(depth, [rows, rows] of who is on whose path) of one sequence."""
    n = len(parents)
    depth, on = np.zeros(n, np.int64), np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            depth[i] = depth[p] + 1
            on[i] = on[p]
        on[i, i] = True
    return depth, on


def _packed(on, words):
    n = on.shape[0]
    bits = np.zeros((n, words * 32), np.uint8)
    bits[:, :on.shape[1]] = on
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32).reshape(n, words)


def _kept(case, seed):
    """(rows of the accepted path, in order) of every sequence.  Its first rows are the tree's first, the others lie behind the
    blocks that they move to, as in a tree whose first levels are wide (and so a second pass over the same state finds the same rows)."""
    got = []
    for s, (c, n) in enumerate(_lens(case)):
        rng = _seq_rng(seed, s)
        m = min(n, 1 + int(rng.integers(0, case["keep"])) if s else case["keep"])
        behind = -(-(c + m) // BLOCK) * BLOCK - c
        far = min(m, max(0, n - behind), int(rng.integers(0, m + 1)) if s else m - 1)
        rows = list(range(m - far)) + sorted(int(x) for x in rng.choice(np.arange(behind, n), far, replace=False)) if far else list(range(m))
        got.append(rows)
    return got


def _context_seen(case, c, n):
    """(pairs of a row and a context key, context keys some row sees), rows at the depths of a chain of about log(n)."""
    w, f = case["window"], case["first"]
    if not w or w > c:
        return n * c, c
    return n * (w + min(f, c - w)), min(c, w + f)


def work(case):
    if case["kind"] == "copy":
        return {"bytes": 2 * case["layers"] * case["pairs"] * case["kv_heads"] * case["page"] * (case["dim"] + case["vdim"] + 8 / BLOCK), "flops": 0}
    lens = _lens(case)
    T = sum(n for _, n in lens)
    if case["kind"] == "tree":
        return {"bytes": 4 * T * (2 + _words(case)) + 8 * case["seqs"], "flops": T * _words(case)}
    G, d, dv = case["kv_heads"], case["dim"], case["vdim"]
    if case["kind"] == "keep":
        rows = sum(len(r) for r in _kept(case, 0))
        return {"bytes": case["layers"] * rows * G * (2 * (d + dv) + 16), "flops": case["layers"] * rows * G * (d + dv)}
    H, e = case["heads"], 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "append":
        return {"bytes": T * (G * (d + dv) + 2 * H * d) * e + T * G * (d + dv) + 8 * G * (T // BLOCK + case["seqs"]) + 4 * T * case["axes"],
                "flops": T * (3 * (H + G) * case["rot"] + 2 * G * (d + dv))}
    read, flops = T * (H * (d + dv) * e + 4 + 4 * _words(case)), 0
    for c, n in lens:
        pairs, keys = _context_seen(case, c, n)
        pairs += n * (n + 1) // 2 if case["shape"] == "chain" else n * min(n, int(2 * math.log(n + 1)) + 1)
        read += G * (keys + n) * (d + dv) + 8 * G * (keys + n) // BLOCK
        flops += 2 * H * pairs * (d + dv)
    return {"bytes": read, "flops": flops}


def _up16(n):
    return -(-n // 16) * 16


def _fill(codes, scales, held, g):
    """Codes and scales of the positions already cached; `held` [pages, page] tells which."""
    pages, G, page, ld = codes.shape
    step = max(1, (1 << 25) // (G * page * ld))
    for a in range(0, pages, step):
        x = torch.randn(codes[a:a + step].shape, generator=g, device="cuda") * torch.linspace(0.5, 2.0, G, device="cuda").view(1, G, 1, 1)
        x = (x * held[a:a + step].view(-1, 1, page, 1)).view(-1, G, page // BLOCK, BLOCK * ld)
        top = torch.frexp(x.abs().amax(-1) / 448.0)
        e = torch.where(top.mantissa == 0.5, top.exponent - 1, top.exponent).clamp(LEAST).float()
        codes[a:a + step] = (x * torch.exp2(-e).unsqueeze(-1)).to(torch.float8_e4m3fn).view(-1, G, page, ld)
        scales[a:a + step] = torch.exp2(e)


def _pools(case, layers, n_pages, held, g):
    """Codes and scales of `layers` caches, one behind the other."""
    got = {}
    for name, width in (("k", case["dim"]), ("v", case["vdim"])):
        codes = torch.zeros(layers * n_pages, case["kv_heads"], case["page"], _up16(width), dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.zeros(layers * n_pages, case["kv_heads"], case["page"] // BLOCK, device="cuda")
        _fill(codes, scales, held.repeat(layers, 1), g)
        codes.view(torch.uint8)[..., width:] = 0
        got[name + "_codes"], got[name + "_scale"] = codes, scales
    return got


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _grid_positions(case, n, base, axes):
    """[axes, n]: a text in front, whose axes agree, then pictures of 14 x 22 patches that follow one another in time."""
    text = n // 8
    at = np.arange(n)
    patch = np.maximum(at - text, 0)
    grid = [patch // 308, patch // 22 % 14, patch % 22, patch % 7]
    return np.stack([base + np.where(at < text, at, text + grid[a]) for a in range(axes)])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    kind = case["kind"]
    state = dict(case)
    if kind == "copy":
        pairs, layers = case["pairs"], case["layers"]
        n_pages = 2 * pairs + 3
        state.update(_pools(case, layers, n_pages, torch.ones(n_pages, case["page"], device="cuda"), g), n_pages=n_pages)
        order = np.random.default_rng([int(seed), 5]).permutation(n_pages)
        state["src"], state["dst"] = [int(x) for x in order[:pairs]], [int(x) for x in order[pairs:2 * pairs]]
        state["src"][pairs // 2] = state["src"][0]          # a page that is forked twice
        if own:
            state["caches"] = _caches_of(state, layers)
        return state
    lens = _lens(case)
    S, new = len(lens), [n for _, n in lens]
    T = sum(new)
    state.update(T=T, max_new=max(new), max_len=max(c + n for c, n in lens), start=_ints([0] + [sum(new[:i + 1]) for i in range(S)]), pos0=_ints([c for c, _ in lens]))
    if kind in ("tree", "attend"):
        parents = [_parents(case, n, _seq_rng(seed, s)) for s, n in enumerate(new)]
        trees = [_tree_of(p) for p in parents]
        if kind == "tree":
            state["parents"] = _ints(np.concatenate(parents))
            state["pos0"] += _ints([int(_seq_rng(seed, s).integers(0, 1000)) for s in range(S)])
        else:
            state["positions"] = _ints(np.concatenate([c + t[0] for (c, _), t in zip(lens, trees)]))
            state["sees"] = _ints(np.concatenate([_packed(t[1], _words(case)) for t in trees]))
    if kind == "tree":
        if own:
            from smoltts_b200.kv_cache import KVCache8
            state["cache"] = KVCache8.allocate(1, 16, 1, 16)      # (its error word is what a tree's faults are reported in)
        return state
    counts, page = _pages(case), case["page"]
    H, G, d, dv = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    n_pages = sum(counts) + 2
    order = torch.randperm(n_pages, generator=g, device="cuda")
    table = torch.full((S, max(counts)), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(n_pages, page, device="cuda")
    at = 0
    for s, ((c, n), k) in enumerate(zip(lens, counts)):
        mine = order[at:at + k]
        table[s, :k] = mine.int()
        held[mine] = (torch.arange(k * page, device="cuda") < (c if kind == "append" else c + n)).float().view(k, page)
        at += k
    layers = case.get("layers", 1)
    state.update(_pools(case, layers, n_pages, held, g), n_pages=n_pages, table=table)
    if kind == "keep":
        kept = _kept(case, seed)
        most = max(len(r) for r in kept)
        state["rows"], state["counts"] = _ints([r + [-1] * (most - len(r)) for r in kept]), _ints([len(r) for r in kept])
        if own:
            state["caches"] = _caches_of(state, layers)
        return state
    dt = getattr(torch, case["dtype"])
    if kind == "append":
        pairs, axes = case["rot"] // 2, case["axes"]
        state["freq"] = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float32) * 2 / case["rot"])
        # the axes in turn, pair by pair, or one behind the other in sections
        state["axis"] = _ints([i % axes if case["mix"] else min(axes - 1, i * axes // pairs) for i in range(pairs)])
        if axes == 1:
            state["positions"] = _ints(np.concatenate([c + _tree_of(_parents(dict(case, shape="random"), n, _seq_rng(seed, s)))[0] if n <= 256 else c + np.arange(n) // 2
                                                       for s, (c, n) in enumerate(lens)])).view(1, T)
        else:
            state["positions"] = _ints(np.concatenate([_grid_positions(case, n, c, axes) for c, n in lens], 1))
        widths = [H * d, G * d, G * dv]
        rows = [torch.randn(T, w, generator=g, device="cuda") for w in widths]
        rows[1] = rows[1] * torch.linspace(0.5, 2.0, G, device="cuda").repeat_interleave(d)
        parts = torch.cat(rows, 1).to(dt).split(widths, 1) if case["fused"] else [r.to(dt) for r in rows]
        state["new_q"], state["new_k"], state["new_v"] = parts[0].view(T, H, d), parts[1].view(T, G, d), parts[2].view(T, G, dv)
    else:
        state["q"] = torch.randn(T, H, d, generator=g, device="cuda").to(dt)
        state["scale"] = d ** -0.5
        state["softcap"] = 30.0 if case["options"] == "capped" else 0.0
        state["slope"] = torch.exp2(-8.0 * (torch.arange(H, device="cuda") + 1) / H) if case["options"] == "capped" else None
        state["sink"] = torch.randn(H, generator=g, device="cuda") if case["options"] != "plain" else None
        state["penalty"] = (torch.rand(H, generator=g, device="cuda"), torch.rand(H, generator=g, device="cuda")) if case["options"] == "penalty" else None
    if own:
        state["cache"] = _caches_of(state, 1)[0]
    return state


def _caches_of(s, layers):
    from smoltts_b200.kv_cache import KVCache8
    n = s["n_pages"]
    return [KVCache8(*(s[x][i * n:(i + 1) * n] for x in ("k_codes", "v_codes", "k_scale", "v_scale")), dim=s["dim"], vdim=s["vdim"]) for i in range(layers)]


# ---------------------------------------------------------------------------------------------- plain forms

def _sequence_of_rows(s):
    return torch.searchsorted(s["start"][1:].long(), torch.arange(s["T"], device="cuda"), right=True)


def _tree(s):
    """Paths by doubling: who is within 2^k steps in front of a row, and the row that is 2^k steps in front of it."""
    seq = _sequence_of_rows(s)
    first = s["start"].long()[seq]
    T, words = s["T"], -(-s["max_new"] // 32)
    at = torch.arange(T, device="cuda")
    sees = torch.zeros(T + 1, words * 32, dtype=torch.bool, device="cuda")      # (the last row: nobody)
    sees[at, at - first] = True
    up = torch.cat([torch.where(s["parents"] >= 0, first + s["parents"], torch.full_like(first, T)), torch.full_like(first[:1], T)])
    for _ in range(max(1, (s["max_new"] - 1).bit_length())):
        sees = sees | sees[up]
        up = up[up]
    sees = sees[:T]
    bits = (sees.view(T, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    return {"positions": (s["pos0"].long()[seq] + sees.sum(-1) - 1).int(), "sees": torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()}


def _rotated(x, s):
    """x [T, heads, d] in 32 bits, its leading coordinates turned, every pair by the position on its axis (angles in 64 bits)."""
    x, half = x.float(), s["half"]
    angle = s["positions"].double()[s["axis"].long()].T * s["freq"].double()
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    n = s["freq"].numel()
    a, b = (x[..., :n], x[..., n:2 * n]) if half else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _write(x, count, pos0, table, page_size, codes, scales):
    """Rows x [S, most, G, row] (the first count[s] of them) behind position pos0[s] of every sequence."""
    S, most = x.shape[:2]
    pos0, count = pos0.view(S, 1), count.view(S, 1)
    blocks = (most + 2 * BLOCK - 2) // BLOCK
    b = pos0 // BLOCK + torch.arange(blocks, device="cuda")
    b = torch.where(b * BLOCK < pos0 + count, b, pos0 // BLOCK)      # a block too many: the first one again
    per = page_size // BLOCK
    page, blk = table.long().gather(1, b // per), b % per
    p = b.unsqueeze(-1) * BLOCK + torch.arange(BLOCK, device="cuda")
    new = ((p >= pos0.unsqueeze(-1)) & (p < (pos0 + count).unsqueeze(-1))).unsqueeze(2).unsqueeze(-1)
    n_pages, G, _, ld = codes.shape
    x = torch.nn.functional.pad(x, (0, ld - x.shape[-1])).clamp(-MOST, MOST)
    rows = x[torch.arange(S, device="cuda").view(S, 1, 1), (p - pos0.unsqueeze(-1)).clamp(0, most - 1)].transpose(2, 3)
    rows = torch.where(new, rows, torch.zeros_like(rows))
    top = torch.frexp(rows.abs().amax((-1, -2)) / 448.0)
    need = torch.where(top.mantissa == 0.5, top.exponent - 1, top.exponent).clamp(LEAST).float()
    whole, every = codes.view(torch.uint8).view(n_pages, G, per, BLOCK, ld), scales
    had = every[page, :, blk]
    before = torch.where((p[..., 0] < pos0).unsqueeze(-1), torch.frexp(had).exponent.float() - 1.0, torch.full_like(had, float(LEAST)))
    e = torch.maximum(need, before)
    old = whole[page, :, blk]
    again = (old.view(torch.float8_e4m3fn).float() * torch.exp2(before - e)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    kept = torch.where((p < pos0.unsqueeze(-1)).unsqueeze(2).unsqueeze(-1), again, old)
    put = (rows * torch.exp2(-e)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    whole[page, :, blk] = torch.where(new, put, kept)
    every[page, :, blk] = torch.exp2(e)


def _append(s):
    start, S = s["start"].long(), s["pos0"].numel()
    at = (start[:-1].view(S, 1) + torch.arange(s["max_new"], device="cuda")).clamp(max=s["T"] - 1)
    for x, name in ((_rotated(s["new_k"], s), "k"), (s["new_v"].float(), "v")):
        _write(x[at], start[1:] - start[:-1], s["pos0"].long(), s["table"], s["page"], s[name + "_codes"], s[name + "_scale"])
    return _rotated(s["new_q"], s).to(s["new_q"].dtype)


def _layered(s):
    """Every layer's sequences one behind the other, with the pages of the pool that holds all layers."""
    L, n = s["layers"], s["n_pages"]
    table = torch.cat([torch.where(s["table"] >= 0, s["table"] + i * n, s["table"]) for i in range(L)])
    return table, s["pos0"].long().repeat(L), s["counts"].long().repeat(L), s["rows"].long().repeat(L, 1)


def _keep(s):
    table, pos0, counts, rows = _layered(s)
    p = pos0.unsqueeze(1) + rows.clamp(min=0)
    page, at = table.long().gather(1, p // s["page"]), p % s["page"]
    moved = []
    for name in ("k", "v"):
        codes, scales = s[name + "_codes"], s[name + "_scale"]
        moved.append(codes.view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn).float() * scales[page, :, at // BLOCK].unsqueeze(-1))
    for name, x in zip(("k", "v"), moved):
        _write(x, counts, pos0, table, s["page"], s[name + "_codes"], s[name + "_scale"])


def _copy(s):
    src, dst = (torch.tensor(s[x], device="cuda") for x in ("src", "dst"))
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        x = s[name].view(torch.uint8) if "codes" in name else s[name]
        x = x.view(s["layers"], s["n_pages"], -1)
        x[:, dst] = x[:, src]


def _cached(s, codes, scales, width):
    """Values of every sequence's pages [S, G, positions, width] in 32 bits."""
    pages = s["table"].long().clamp(0)
    x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()
    S, P, G, page, ld = x.shape
    x = x.view(S, P, G, page // BLOCK, BLOCK, ld) * scales[pages][..., None, None]
    return x.view(S, P, G, page, ld).transpose(1, 2).reshape(S, G, P * page, ld)[..., :width]


def _attend(s):
    S, G, H, n, q = s["pos0"].numel(), s["kv_heads"], s["heads"], s["max_new"], s["q"]
    start, pos0 = s["start"].long(), s["pos0"].long().view(S, 1)
    at = (start[:-1].view(S, 1) + torch.arange(n, device="cuda")).clamp(max=s["T"] - 1)
    rows = q.float()[at].view(S, n, G, H // G, s["dim"]).permute(0, 2, 3, 1, 4).reshape(S, G, -1, s["dim"])
    score = (rows @ _cached(s, s["k_codes"], s["k_scale"], s["dim"]).transpose(-1, -2)).mul_(s["scale"]).view(S, H, n, -1)
    place = torch.arange(score.shape[-1], device="cuda")
    row = place - pos0                                                  # of a drafted key
    drafted = (row >= 0) & (row < start[1:].view(S, 1) - start[:-1].view(S, 1))
    key = torch.where(drafted, s["positions"].long()[(start[:-1].view(S, 1) + row).clamp(0, s["T"] - 1)], place)
    bits = s["sees"].long()[at].unsqueeze(-1) >> torch.arange(32, device="cuda")
    bits = (bits & 1).bool().flatten(-2)                                # [S, n, 32 words]
    named = bits.gather(2, row.clamp(0, bits.shape[-1] - 1).unsqueeze(1).expand(-1, n, -1))
    sees = torch.where(drafted.unsqueeze(1), named, (row < 0).unsqueeze(1))
    dist = s["positions"].long()[at].unsqueeze(-1) - key.unsqueeze(1)
    if s["window"]:
        sees = sees & ((dist < s["window"]) | (key < s["first"]).unsqueeze(1))
    if s["softcap"]:
        score = score.div_(s["softcap"]).tanh_().mul_(s["softcap"])
    far = dist.clamp(0).float().unsqueeze(1)
    if s["penalty"] is not None:
        score = score - s["penalty"][0].view(H, 1, 1) * torch.log1p(s["penalty"][1].view(H, 1, 1) * far)
    if s["slope"] is not None:
        score = score - s["slope"].view(H, 1, 1) * far
    score = score.masked_fill_(~sees.unsqueeze(1), -math.inf)
    top = score.amax(-1, keepdim=True)
    sink = s["sink"].view(H, 1, 1) if s["sink"] is not None else None
    top = torch.maximum(top, sink) if sink is not None else top
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    total = total + (sink - top).exp() if sink is not None else total
    out = weight.view(S, G, -1, weight.shape[-1]) @ _cached(s, s["v_codes"], s["v_scale"], s["vdim"])
    out = (out.view(S, H, n, -1) / total).transpose(1, 2)
    seq = _sequence_of_rows(s)
    return out[seq, torch.arange(s["T"], device="cuda") - start[seq]].to(q.dtype)


def _state_of_caches(s):
    return {"k": s["k_codes"], "v": s["v_codes"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def run(s):
    kind = s["kind"]
    if own:
        if kind == "tree":
            tree = s["cache"].draft_tree(s["parents"], s["start"], s["pos0"], max_new=s["max_new"])
            return {"positions": tree.positions, "sees": tree.sees}
        if kind == "append":
            q = s["cache"].append(s["new_k"], s["new_v"], s["start"], s["pos0"], s["table"], max_new=s["max_new"], q=s["new_q"], freq=s["freq"], rot_half=s["half"],
                                  positions=s["positions"], axis=s["axis"])
            return {"q": q, **_state_of_caches(s)}
        if kind == "attend":
            from smoltts_b200.kv_cache import DraftTree
            return {"out": s["cache"].attend(s["q"], s["start"], s["pos0"], s["table"], max_new=s["max_new"], max_len=s["max_len"], scale=s["scale"], window=s["window"], first=s["first"],
                                             softcap=s["softcap"], slope=s["slope"], sink=s["sink"], penalty=s["penalty"], tree=DraftTree(s["positions"], s["sees"]))}
        from smoltts_b200.kv_cache import copy_pages, keep_rows
        if kind == "keep":
            keep_rows(s["caches"], s["pos0"], s["table"], s["rows"], s["counts"])
        else:
            copy_pages(s["caches"], s["src"], s["dst"])
        return _state_of_caches(s)
    if kind == "tree":
        return _tree(s)
    if kind == "append":
        return {"q": _append(s), **_state_of_caches(s)}
    if kind == "attend":
        return {"out": _attend(s)}
    _keep(s) if kind == "keep" else _copy(s)
    return _state_of_caches(s)


# ---------------------------------------------------------------------------------------------- in 64 bits

def _put(codes, scales, table_row, page_size, c, x):
    """Rows x [n, G, row] in 64 bits behind position c of one sequence (codes as bytes, scales in 64 bits)."""
    powers = torch.tensor([2.0 ** e for e in range(LEAST, 101)], dtype=torch.float64, device="cuda")      # (a library's logarithm of a power of two may be off by a bit)
    n, G = x.shape[:2]
    first, last = c // BLOCK, (c + n - 1) // BLOCK
    base = torch.zeros(((last - first + 1) * BLOCK, G, x.shape[-1]), dtype=torch.float64, device="cuda")
    base[c - first * BLOCK:c - first * BLOCK + n] = x
    base = base.view(-1, BLOCK, G, x.shape[-1])
    scale = powers[torch.searchsorted(448.0 * powers, base.abs().amax((1, 3)))]      # the smallest that holds the block
    where = torch.arange(first, last + 1, device="cuda")
    pg, bl = table_row[where * BLOCK // page_size].long(), where % (page_size // BLOCK)
    if c % BLOCK:
        had = scales[pg[0], :, bl[0]]
        scale[0] = torch.maximum(scale[0], had)
        before = slice(bl[0] * BLOCK, bl[0] * BLOCK + c % BLOCK)
        old = codes[pg[0], :, before].contiguous().view(torch.float8_e4m3fn).double() * (had / scale[0]).view(G, 1, 1)
        codes[pg[0], :, before] = old.to(torch.float8_e4m3fn).view(torch.uint8)
    scales[pg, :, bl] = scale
    put = (base / scale.view(-1, 1, G, 1)).flatten(0, 1)[c - first * BLOCK:c - first * BLOCK + n]
    at = torch.arange(c, c + n, device="cuda")
    codes[table_row[at // page_size].long(), :, at % page_size, :x.shape[-1]] = put.to(torch.float8_e4m3fn).view(torch.uint8)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "tree":
        parents, pos0, got = s["parents"].cpu().numpy(), s["pos0"].tolist(), {"positions": [], "sees": []}
        at = 0
        for c, (_, n) in zip(pos0, _lens(case)):
            bits, depth = np.zeros((n, _words(case) * 32), bool), []
            for i in range(n):
                path, j = [i], i
                while parents[at + j] >= 0:
                    j = parents[at + j]
                    path.append(j)
                bits[i, path] = True
                depth.append(c + len(path) - 1)
            got["positions"].append(np.array(depth))
            got["sees"].append(_packed(bits, _words(case)))
            at += n
        return {k: _ints(np.concatenate(v)) for k, v in got.items()}
    codes = {name: s[name + "_codes"].view(torch.uint8) for name in ("k", "v")}
    scales = {name: s[name + "_scale"].double() for name in ("k", "v")}
    widths = {"k": case["dim"], "v": case["vdim"]}
    page = case["page"]
    got = {}

    def cached():
        return {"k": codes["k"].view(torch.float8_e4m3fn).double(), "v": codes["v"].view(torch.float8_e4m3fn).double(), "k_scale": scales["k"], "v_scale": scales["v"]}

    if kind == "copy":
        for i in range(case["layers"]):
            for a, b in zip(s["src"], s["dst"]):
                for x in (*codes.values(), *scales.values()):
                    x[i * s["n_pages"] + b] = x[i * s["n_pages"] + a]
        return cached()
    lens = _lens(case)
    if kind == "keep":
        kept = _kept(case, seed)
        for layer in range(case["layers"]):
            for i, (c, _) in enumerate(lens):
                at = c + torch.tensor(kept[i], device="cuda")
                mine = torch.where(s["table"][i] >= 0, s["table"][i] + layer * s["n_pages"], s["table"][i])
                for name in ("k", "v"):
                    pg = mine[at // page].long()
                    x = codes[name][pg, :, at % page].contiguous().view(torch.float8_e4m3fn).double() * scales[name][pg, :, at % page // BLOCK].unsqueeze(-1)
                    _put(codes[name], scales[name], mine, page, c, x)
        return cached()
    H, G, dv = case["heads"], case["kv_heads"], case["vdim"]
    starts = [sum(n for _, n in lens[:i]) for i in range(len(lens))]
    if kind == "append":
        def turned(x):
            y = x.double().clone()
            for i in range(case["rot"] // 2):
                a, b = (i, i + case["rot"] // 2) if case["half"] else (2 * i, 2 * i + 1)
                t = (s["positions"][int(s["axis"][i])].double() * s["freq"][i].double()).unsqueeze(1)
                y[:, :, a], y[:, :, b] = x[:, :, a].double() * t.cos() - x[:, :, b].double() * t.sin(), x[:, :, b].double() * t.cos() + x[:, :, a].double() * t.sin()
            return y

        got["q"] = turned(s["new_q"])
        for name, x in (("k", turned(s["new_k"])), ("v", s["new_v"].double())):
            for i, (c, n) in enumerate(lens):
                _put(codes[name], scales[name], s["table"][i], page, c, x[starts[i]:starts[i] + n])
        return {**got, **cached()}
    q, positions, sees = s["q"].double(), s["positions"].long(), s["sees"].cpu().numpy()
    out = torch.zeros(s["T"], H, dv, dtype=torch.float64, device="cuda")
    for i, (c, n) in enumerate(lens):
        pages, L, mine = s["table"][i, :-(-(c + n) // page)].long(), c + n, slice(starts[i], starts[i] + n)
        key = torch.cat([torch.arange(c, device="cuda"), positions[mine]])
        named = np.unpackbits(sees[mine].view(np.uint8), axis=1, bitorder="little")[:, :n]
        hidden = torch.cat([torch.zeros(n, c, dtype=torch.bool), torch.from_numpy(named == 0)], 1).cuda()
        dist = (positions[mine].view(n, 1) - key).double()
        if case["window"]:
            hidden |= (dist >= case["window"]) & (key >= case["first"])
        for h in range(H):
            kv = [(codes[x][pages, h // (H // G)].contiguous().view(torch.float8_e4m3fn).double().reshape(-1, codes[x].shape[-1])[:L, :widths[x]]
                   * scales[x][pages, h // (H // G)].reshape(-1).repeat_interleave(BLOCK)[:L, None]) for x in ("k", "v")]
            z = q[mine, h] @ kv[0].T * s["scale"]
            if s["softcap"]:
                z = s["softcap"] * torch.tanh(z / s["softcap"])
            if s["penalty"] is not None:
                z = z - s["penalty"][0][h].double() * torch.log1p(s["penalty"][1][h].double() * dist.clamp(min=0))
            if s["slope"] is not None:
                z = z - s["slope"][h].double() * dist.clamp(min=0)
            z = z.masked_fill(hidden, -math.inf)
            if s["sink"] is not None:
                z = torch.cat([z, s["sink"][h].double().expand(n, 1)], 1)
            out[mine, h] = torch.softmax(z, -1)[:, :L] @ kv[1]
    return {"out": out}
