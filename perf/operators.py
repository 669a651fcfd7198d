"""What is measured of the 8-bit key/value cache: appending to it with the position rotation on the way, and attention over it.

A cache holds, per page, key/value head and position, a row of e4m3 codes for the key and one for the value; 16 positions
that follow one another share one power-of-two scale per head (keys and values each their own).

* ``append`` -- rotates the step's keys (and queries) by position and writes keys and values into the pages.  A block begun
  by an earlier step keeps the larger of its old scale and the one the new tokens need; old codes follow a scale that grows.
* ``attend`` -- softmax attention of the step's queries over the pages: causal, behind a window if asked, with the first
  positions of the sequence left visible, soft cap, linear and logarithmic distance penalties and a sink logit.
* ``step`` -- both, as a layer calls them.

Heads and head sizes are those of the language models' benchmark configurations (12 heads over 4 of 64 or 128) or generic.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 16                       # positions that share a scale
LEAST, MOST = -110, 2.0 ** 100   # least exponent of a scale; magnitudes above are clamped


def listed():
    return [
        # one chat, one layer of the small benchmark model: latency
        dict(name="append_token_1", kind="append", seqs=1, new=1, context=2047, heads=12, kv_heads=4, dim=64, vdim=64, page=64, dtype="bfloat16", rot=64, half=True, fused=True),
        # a serving batch at unequal lengths, one token each
        dict(name="append_tokens_64", kind="append", seqs=64, new=1, context=4096, heads=32, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16", rot=128, half=True, fused=True),
        # prompts of three requests in one step, unequal lengths, slices of one fused projection
        dict(name="append_prompts_3", kind="append", seqs=3, new=4001, context=70, heads=32, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16", rot=128, half=True, fused=True),
        # the float32 engine: neighbours rotated, a part of the head only
        dict(name="append_prompts_f32", kind="append", seqs=2, new=301, context=33, heads=12, kv_heads=4, dim=96, vdim=64, page=32, dtype="float32", rot=64, half=False, fused=False),
        # one chat, one layer: append and attention of a token
        dict(name="step_token_1", kind="step", seqs=1, new=1, context=2047, heads=12, kv_heads=4, dim=64, vdim=64, page=64, dtype="bfloat16", rot=64, half=True, fused=True, window=0, first=0, options="plain"),
        # a serving batch at unequal lengths: the keys and values of everybody's context
        dict(name="attend_tokens_64", kind="attend", seqs=64, new=1, context=8192, heads=32, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16", window=0, first=0, options="plain"),
        # one chat behind a very long context
        dict(name="attend_token_long", kind="attend", seqs=1, new=1, context=131071, heads=12, kv_heads=4, dim=128, vdim=128, page=64, dtype="bfloat16", window=0, first=0, options="plain"),
        # long chats behind a window whose first tokens stay visible
        dict(name="attend_tokens_window", kind="attend", seqs=32, new=1, context=30000, heads=32, kv_heads=4, dim=128, vdim=128, page=64, dtype="bfloat16", window=1024, first=4, options="plain"),
        # a long prompt
        dict(name="attend_prompt_4096", kind="attend", seqs=1, new=4096, context=0, heads=32, kv_heads=8, dim=128, vdim=128, page=64, dtype="bfloat16", window=0, first=0, options="plain"),
        # a long prompt behind a window whose first tokens stay visible
        dict(name="attend_prompt_window", kind="attend", seqs=1, new=7900, context=0, heads=16, kv_heads=4, dim=128, vdim=128, page=64, dtype="bfloat16", window=1000, first=16, options="plain"),
        # portions of several prompts behind their cached beginnings, soft cap, linear penalty and sink, odd head sizes
        dict(name="attend_prompts_5", kind="attend", seqs=5, new=340, context=1001, heads=12, kv_heads=4, dim=80, vdim=72, page=32, dtype="bfloat16", window=0, first=0, options="capped"),
        # the float32 engine: logarithmic penalty and sink
        dict(name="attend_prompt_f32", kind="attend", seqs=1, new=300, context=0, heads=12, kv_heads=4, dim=64, vdim=64, page=64, dtype="float32", window=0, first=0, options="penalty"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "step"])
    few = rng.random() < 0.5
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 160, 256])
    vdim = dim if rng.random() < 0.7 else rng.choice([40, 64, 72, 128])
    case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, page=rng.choice([16, 32, 64, 128]), dtype="float32" if rng.random() < 0.2 else "bfloat16")
    if few:
        case["seqs"] = _log_int(rng, 1, 64)
        case["new"] = rng.choice([1, 1, 1, 2, 5])
        case["context"] = _log_int(rng, 1, 131072 // case["seqs"])
    else:
        case["seqs"] = rng.choice([1, 1, 2, 3, 7])
        case["new"] = _log_int(rng, 9, 4096 // case["seqs"])
        case["context"] = rng.choice([0, _log_int(rng, 1, 4096 // case["seqs"])])
    if kind != "attend":
        case.update(rot=rng.choice([0, 16, dim // 2 // 2 * 2, dim]), half=rng.random() < 0.5, fused=rng.random() < 0.5)
    if kind != "append":
        window = rng.choice([0, 0, _log_int(rng, 1, 2000)])
        case.update(window=window, first=rng.choice([0, 1, 4, 33]) if window else 0, options=rng.choice(["plain", "plain", "plain", "capped", "penalty"]))
    return case


# ---------------------------------------------------------------------------------------------- what a case holds

def _lens(case):
    """(cached before, new) of every sequence, the first one the longest."""
    c, n, S = case["context"], case["new"], case["seqs"]
    return [(c - (c // 2) * s // S if S > 1 else c, n if n < 4 else max(1, n - (n // 3) * s // S)) for s in range(S)]


def _pages(case):
    return [-(-(c + n) // case["page"]) for c, n in _lens(case)]


def _seen(case, pos, n):
    """(pairs of a row and a key it sees, keys that some row sees) for rows pos .. pos + n - 1."""
    w, f = case.get("window", 0), case.get("first", 0)
    if not w:
        return n * pos + n * (n + 1) // 2, pos + n
    pairs = sum(min(i + 1, w) + min(f, max(0, i + 1 - w)) for i in range(pos, pos + n))
    start = max(0, pos + 1 - w)
    return pairs, pos + n - start + min(f, start)


def work(case):
    H, G, d, dv, e = case["heads"], case["kv_heads"], case["dim"], case["vdim"], 4 if case["dtype"] == "float32" else 2
    T, read, flops = sum(n for _, n in _lens(case)), 0, 0
    if case["kind"] != "attend":
        read += T * (G * (d + dv) + 2 * H * d) * e + T * G * (d + dv) + 8 * G * (T // BLOCK + case["seqs"])
        flops += T * (3 * (H + G) * case["rot"] + 2 * G * (d + dv))
    if case["kind"] != "append":
        read += T * H * (dv if case["kind"] == "step" else d + dv) * e
        for c, n in _lens(case):
            pairs, keys = _seen(case, c, n)
            read += G * keys * (d + dv) + 8 * G * keys // BLOCK
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


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    lens, counts, page = _lens(case), _pages(case), case["page"]
    H, G, d, dv = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    dt = getattr(torch, case["dtype"])
    n_pages, T = sum(counts) + 2, sum(n for _, n in lens)
    order = torch.randperm(n_pages, generator=g, device="cuda")
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(n_pages, page, device="cuda")
    at = 0
    for s, ((c, n), k) in enumerate(zip(lens, counts)):
        mine = order[at:at + k]
        table[s, :k] = mine.int()
        held[mine] = (torch.arange(k * page, device="cuda") < (c if case["kind"] != "attend" else c + n)).float().view(k, page)
        at += k
    new = [n for _, n in lens]
    state = dict(case, page=page, T=T, table=table, max_new=max(new), max_len=max(c + n for c, n in lens),
                 start=torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device="cuda"),
                 pos0=torch.tensor([c for c, _ in lens], dtype=torch.int32, device="cuda"))
    for name, width in (("k", d), ("v", dv)):
        codes = torch.zeros(n_pages, G, page, _up16(width), dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.zeros(n_pages, G, page // BLOCK, device="cuda")
        _fill(codes, scales, held, g)
        codes.view(torch.uint8)[..., width:] = 0
        state[name + "_codes"], state[name + "_scale"] = codes, scales
    if case["kind"] != "attend":
        state["freq"] = 10000.0 ** (-torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float32) * 2 / max(case["rot"], 1)) if case["rot"] else None
        widths = [H * d, G * d, G * dv]
        rows = [torch.randn(T, w, generator=g, device="cuda") for w in widths]
        rows[1] = rows[1] * torch.linspace(0.5, 2.0, G, device="cuda").repeat_interleave(d)
        parts = torch.cat(rows, 1).to(dt).split(widths, 1) if case["fused"] else [r.to(dt) for r in rows]
        state["new_q"], state["new_k"], state["new_v"] = parts[0].view(T, H, d), parts[1].view(T, G, d), parts[2].view(T, G, dv)
    else:
        state["q"] = torch.randn(T, H, d, generator=g, device="cuda").to(dt)
    if case["kind"] != "append":
        state["scale"] = d ** -0.5
        state["softcap"] = 30.0 if case["options"] == "capped" else 0.0
        state["slope"] = torch.exp2(-8.0 * (torch.arange(H, device="cuda") + 1) / H) if case["options"] == "capped" else None
        state["sink"] = torch.randn(H, generator=g, device="cuda") if case["options"] != "plain" else None
        state["penalty"] = (torch.rand(H, generator=g, device="cuda"), torch.rand(H, generator=g, device="cuda")) if case["options"] == "penalty" else None
    if own:
        from smoltts_b200.kv_cache import KVCache8
        state["cache"] = KVCache8(state["k_codes"], state["v_codes"], state["k_scale"], state["v_scale"], dim=d, vdim=dv)
    return state


# ---------------------------------------------------------------------------------------------- plain forms

def _rotated(x, pos, freq, half):
    """x [T, heads, d] in 32 bits, its leading coordinates turned by pos * freq (angles in 64 bits)."""
    x = x.float()
    if freq is None:
        return x
    angle = pos.double().unsqueeze(1) * freq.double()
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    n = freq.numel()
    a, b = (x[..., :n], x[..., n:2 * n]) if half else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * n:]], -1)


def _positions(s):
    at = torch.arange(s["T"], device="cuda")
    seq = torch.searchsorted(s["start"][1:].long(), at, right=True)
    return s["pos0"].long()[seq] + at - s["start"].long()[seq]


def _write(s, x, codes, scales):
    """New rows x [T, G, d] into the blocks they fall into: [sequences, blocks, G, 16, row]."""
    d, ld, S = x.shape[-1], codes.shape[-1], s["pos0"].numel()
    start, pos0 = s["start"].long(), s["pos0"].long()
    count = (start[1:] - start[:-1]).view(S, 1)
    blocks = (s["max_new"] + 2 * BLOCK - 2) // BLOCK
    b = pos0.view(S, 1) // BLOCK + torch.arange(blocks, device="cuda")
    b = torch.where(b * BLOCK < pos0.view(S, 1) + count, b, pos0.view(S, 1) // BLOCK)      # a block too many: the first one again
    per = s["page"] // BLOCK
    page, blk = s["table"].long().gather(1, b // per), b % per
    p = b.unsqueeze(-1) * BLOCK + torch.arange(BLOCK, device="cuda")
    new = ((p >= pos0.view(S, 1, 1)) & (p < (pos0.view(S, 1) + count).unsqueeze(-1))).unsqueeze(2).unsqueeze(-1)
    x = torch.nn.functional.pad(x, (0, ld - d)).clamp(-MOST, MOST)
    rows = x[(start[:-1].view(S, 1, 1) + p - pos0.view(S, 1, 1)).clamp(0, s["T"] - 1)].transpose(2, 3)
    rows = torch.where(new, rows, torch.zeros_like(rows))
    top = torch.frexp(rows.abs().amax((-1, -2)) / 448.0)
    need = torch.where(top.mantissa == 0.5, top.exponent - 1, top.exponent).clamp(LEAST).float()
    n_pages, G = codes.shape[:2]
    whole, every = codes.view(torch.uint8).view(n_pages, G, per, BLOCK, ld), scales
    had = every[page, :, blk]
    before = torch.where((p[..., 0] < pos0.view(S, 1)).unsqueeze(-1), torch.frexp(had).exponent.float() - 1.0, torch.full_like(had, float(LEAST)))
    e = torch.maximum(need, before)
    old = whole[page, :, blk]
    again = (old.view(torch.float8_e4m3fn).float() * torch.exp2(before - e)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    kept = torch.where((p < pos0.view(S, 1, 1)).unsqueeze(2).unsqueeze(-1), again, old)
    put = (rows * torch.exp2(-e)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    whole[page, :, blk] = torch.where(new, put, kept)
    every[page, :, blk] = torch.exp2(e)


def _append(s):
    pos = _positions(s)
    _write(s, _rotated(s["new_k"], pos, s["freq"], s["half"]), s["k_codes"], s["k_scale"])
    _write(s, s["new_v"].float(), s["v_codes"], s["v_scale"])
    return _rotated(s["new_q"], pos, s["freq"], s["half"]).to(s["new_q"].dtype)


def _cached(s, codes, scales, width):
    """Values of every sequence's pages [S, G, positions, width] in 32 bits."""
    pages = s["table"].long().clamp(0)
    x = codes.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()
    S, P, G, page, ld = x.shape
    x = x.view(S, P, G, page // BLOCK, BLOCK, ld) * scales[pages][..., None, None]
    return x.view(S, P, G, page, ld).transpose(1, 2).reshape(S, G, P * page, ld)[..., :width]


def _attend(s, q):
    S, G, H, n = s["pos0"].numel(), s["kv_heads"], s["heads"], s["max_new"]
    start, pos0 = s["start"].long(), s["pos0"].long()
    at = start[:-1].view(S, 1) + torch.arange(n, device="cuda")
    rows = q.float()[at.clamp(max=s["T"] - 1)].view(S, n, G, H // G, s["dim"]).permute(0, 2, 3, 1, 4).reshape(S, G, -1, s["dim"])
    score = (rows @ _cached(s, s["k_codes"], s["k_scale"], s["dim"]).transpose(-1, -2)).mul_(s["scale"]).view(S, H, n, -1)
    dist = (pos0.view(S, 1) + torch.arange(n, device="cuda")).unsqueeze(-1) - torch.arange(score.shape[-1], device="cuda")
    sees = dist >= 0
    if s["window"]:
        sees = sees & ((dist < s["window"]) | (torch.arange(score.shape[-1], device="cuda") < s["first"]))
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
    seq = torch.searchsorted(start[1:], torch.arange(s["T"], device="cuda"), right=True)
    return out[seq, torch.arange(s["T"], device="cuda") - start[seq]].to(q.dtype)


def _caches(s):
    return {"k": s["k_codes"], "v": s["v_codes"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def run(s):
    if own:
        cache, out = s["cache"], {}
        q = s.get("q")
        if s["kind"] != "attend":
            q = out["q"] = cache.append(s["new_k"], s["new_v"], s["start"], s["pos0"], s["table"], max_new=s["max_new"], q=s["new_q"], freq=s["freq"], rot_half=s["half"])
            out.update(_caches(s))
        if s["kind"] != "append":
            out["out"] = cache.attend(q, s["start"], s["pos0"], s["table"], max_new=s["max_new"], max_len=s["max_len"], scale=s["scale"], window=s["window"],
                                      first=s["first"], softcap=s["softcap"], slope=s["slope"], sink=s["sink"], penalty=s["penalty"])
        return out
    out = {}
    q = s.get("q")
    if s["kind"] != "attend":
        q = out["q"] = _append(s)
        out.update(_caches(s))
    if s["kind"] != "append":
        out["out"] = _attend(s, q)
    return out


# ---------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    H, G, d, dv, page = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    lens, got = _lens(case), {}
    values = {}
    for name in ("k", "v"):
        values[name] = [s[name + "_codes"].view(torch.uint8), s[name + "_scale"].double()]
    q = s["q"].double() if case["kind"] == "attend" else None
    starts = [sum(n for _, n in lens[:i]) for i in range(len(lens))]
    if case["kind"] != "attend":
        pos = torch.cat([torch.arange(c, c + n, device="cuda") for c, n in lens]).double()

        def turned(x):
            y = x.double().clone()
            for i in range(case["rot"] // 2):
                a, b = (i, i + case["rot"] // 2) if case["half"] else (2 * i, 2 * i + 1)
                t = (pos * s["freq"][i].double()).unsqueeze(1)
                y[:, :, a], y[:, :, b] = x[:, :, a].double() * t.cos() - x[:, :, b].double() * t.sin(), x[:, :, b].double() * t.cos() + x[:, :, a].double() * t.sin()
            return y

        q = turned(s["new_q"])
        got["q"] = q
        for name, x in (("k", turned(s["new_k"])), ("v", s["new_v"].double())):
            codes, scales = values[name]
            for i, (c, n) in enumerate(lens):
                first = c // BLOCK
                last = (c + n - 1) // BLOCK
                base = torch.zeros(((last - first + 1) * BLOCK, G, x.shape[-1]), dtype=torch.float64, device="cuda")
                base[c - first * BLOCK:c - first * BLOCK + n] = x[starts[i]:starts[i] + n]
                need = base.view(-1, BLOCK, G, x.shape[-1]).abs().amax((1, 3))
                e = torch.ceil(torch.log2(need / 448.0)).clamp(min=LEAST)
                where = torch.arange(first, last + 1, device="cuda")
                pg, bl = s["table"][i, where * BLOCK // page].long(), where % (page // BLOCK)
                if c % BLOCK:
                    o = torch.log2(scales[pg[0], :, bl[0]])
                    e[0] = torch.maximum(e[0], o)
                    keep = codes[pg[0], :, bl[0] * BLOCK:bl[0] * BLOCK + c % BLOCK]
                    keep = keep.contiguous().view(torch.float8_e4m3fn).double() * torch.exp2(o - e[0]).view(G, 1, 1)
                    codes[pg[0], :, bl[0] * BLOCK:bl[0] * BLOCK + c % BLOCK] = keep.to(torch.float8_e4m3fn).view(torch.uint8)
                scales[pg, :, bl] = torch.exp2(e)
                put = (base.view(-1, BLOCK, G, x.shape[-1]) * torch.exp2(-e).view(-1, 1, G, 1)).flatten(0, 1)[c - first * BLOCK:c - first * BLOCK + n]
                at = torch.arange(c, c + n, device="cuda")
                codes[s["table"][i, at // page].long(), :, at % page, :x.shape[-1]] = put.to(torch.float8_e4m3fn).view(torch.uint8)
            got[name], got[name + "_scale"] = codes.view(torch.float8_e4m3fn).double(), scales
        if case["kind"] == "append":
            return got
        q = q.to(s["new_q"].dtype).double()      # the attention takes the queries as they are handed over
    out = torch.zeros(q.shape[0], H, dv, dtype=torch.float64, device="cuda")
    for i, (c, n) in enumerate(lens):
        pages, L = s["table"][i, :-(-(c + n) // page)].long(), c + n
        dist = (torch.arange(c, c + n, device="cuda").view(n, 1) - torch.arange(L, device="cuda")).double()
        hidden = dist < 0
        if case["window"]:
            hidden |= (dist >= case["window"]) & (torch.arange(L, device="cuda") >= case["first"])
        for h in range(H):
            kv = []
            for name, width in (("k", d), ("v", dv)):
                codes, scales = values[name]
                x = codes[pages, h // (H // G)].contiguous().view(torch.float8_e4m3fn).double().reshape(-1, codes.shape[-1])[:L, :width]
                kv.append(x * scales[pages, h // (H // G)].reshape(-1).repeat_interleave(BLOCK)[:L, None])
            z = q[starts[i]:starts[i] + n, h] @ kv[0].T * s["scale"]
            if s["softcap"]:
                z = s["softcap"] * torch.tanh(z / s["softcap"])
            if s["penalty"] is not None:
                z = z - s["penalty"][0][h].double() * torch.log1p(s["penalty"][1][h].double() * dist.clamp(min=0))
            if s["slope"] is not None:
                z = z - s["slope"][h].double() * dist
            z = z.masked_fill(hidden, -math.inf)
            if s["sink"] is not None:
                z = torch.cat([z, s["sink"][h].double().expand(n, 1)], 1)
            out[starts[i]:starts[i] + n, h] = torch.softmax(z, -1)[:, :L] @ kv[1]
    got["out"] = out
    return got
