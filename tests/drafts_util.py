"""References of drafting and forking on the 8-bit key/value cache: trees, attention along their paths, rows that move."""
from __future__ import annotations

import math
import random

import torch

from cache8_util import BLOCK, exponent


def parents_of(shape, n, seed=0):
    rng = random.Random(f"{shape} {n} {seed}")
    if shape == "chain":
        return [i - 1 for i in range(n)]
    if shape == "roots":
        return [-1] * n
    if shape == "fan":
        return [-1 if i == 0 else (i - 1) // 3 for i in range(n)]
    if shape == "comb":      # a chain with a leaf at every row
        return [-1 if i == 0 else (i - 1 if i % 2 else max(i - 2, 0)) for i in range(n)]
    return [rng.randint(-1, i - 1) if i else -1 for i in range(n)]


def paths_of(parents):
    """Rows on every row's way, itself among them."""
    ways = []
    for i, p in enumerate(parents):
        ways.append([i] + (ways[p] if p >= 0 else []))
    return ways


def layout(parents, words):
    """(depth of every row, its bits as signed 32-bit words)."""
    on = torch.zeros(len(parents), words * 32, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            on[i] = on[p]
        on[i, i] = True
    bits = (on.view(len(parents), words, 32).long() << torch.arange(32)).sum(-1)
    return on.sum(1) - 1, torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()


def named(sees, n):
    """Bits as [rows, n] truth values."""
    bits = (sees.long().unsqueeze(-1) >> torch.arange(32, device=sees.device)) & 1
    bits = bits.flatten(-2).bool()
    return bits[:, :n] if bits.shape[1] >= n else torch.nn.functional.pad(bits, (0, n - bits.shape[1]))


def tree_attention(q, k, v, pos0, positions, sees, scale, window=0, first=0, softcap=0.0, sink=None, slope=None, penalty=None, kv_len=None):
    """One sequence in 64 bits: rows q [n, H, d] at positions [n], keys / values [pos0 + m, G, .], the last m of them the sequence's rows at the first m of the positions.
    Returns the result, the sum of weight * |value| over the denominator, and the largest sum of |q_i k_i| * scale of each row, as ``cache8_util.attention`` does."""
    n, H, _ = q.shape
    L, G, dv = v.shape
    key = torch.cat([torch.arange(pos0, device=q.device), positions.long()])[:L]
    seen = torch.cat([torch.ones(n, pos0, dtype=torch.bool, device=q.device), named(sees, L - pos0)], 1)
    dist = positions.long()[:n].view(n, 1) - key
    if window:
        seen = seen & ((dist < window) | (key < first))
    if kv_len is not None:
        seen = seen & (torch.arange(L, device=q.device) < kv_len)
    out, spread, size = (torch.zeros(n, H, w, dtype=torch.float64, device=q.device) for w in (dv, dv, 1))
    some = seen.any(1, keepdim=True)
    for h in range(H):
        g = h // (H // G)
        s = q[:, h].double() @ k[:, g].double().T * scale
        size[:, h] = ((q[:, h].double().abs() @ k[:, g].double().abs().T) * abs(scale)).masked_fill(~seen, 0.0).nan_to_num(0.0).amax(1, keepdim=True)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        far = dist.clamp(min=0).double()
        if penalty is not None:
            s = s - penalty[0][h].double() * torch.log1p(penalty[1][h].double() * far)
        if slope is not None:
            s = s - slope[h].double() * far
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(1, keepdim=True)
        if sink is not None:
            top = top.clamp(min=sink[h].item())
        top = top.masked_fill(~some & (sink is None), 0.0)
        w = torch.exp(s - top)
        total = w.sum(1, keepdim=True) + (torch.exp(sink[h].double() - top) if sink is not None else 0.0)
        total = total.masked_fill(total == 0, 1.0)
        values = torch.where(seen.any(0).view(L, 1), v[:, g].double(), 0.0)      # (what nobody sees may be anything)
        out[:, h], spread[:, h] = w @ values / total, w @ values.abs() / total
    return out, spread, size


def kept(values, had, rows, pos0):
    """What a head's rows [positions, width] (64 bits) become when `rows` behind pos0 are kept: values of positions 0 .. pos0 + len(rows) - 1, and the exponents of the
    blocks they are in from pos0's on.  had: exponent of pos0's block."""
    out, m, exps = values[:pos0 + len(rows)].clone(), len(rows), []
    moved = values[[pos0 + r for r in rows]]
    for b in range(pos0 // BLOCK, (pos0 + m - 1) // BLOCK + 1):
        lo, hi = max(pos0, b * BLOCK), min(pos0 + m, (b + 1) * BLOCK)
        part = moved[lo - pos0:hi - pos0]
        e = exponent(part.nan_to_num(0.0).abs().max().item())
        if lo > b * BLOCK:
            if had < e:
                old = out[b * BLOCK:lo]
                out[b * BLOCK:lo] = (old * 2.0 ** -e).float().to(torch.float8_e4m3fn).double() * 2.0 ** e
            e = max(e, had)
        out[lo:hi] = (part * 2.0 ** -e).float().to(torch.float8_e4m3fn).double() * 2.0 ** e
        exps.append(e)
    return out, exps
