"""Reference of the 8-bit key/value cache in 64 bits, and batches to try it on."""
from __future__ import annotations

import math

import torch

BLOCK = 16
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def exponent(top: float) -> int:
    """Smallest E >= -110 with top <= 448 * 2^E."""
    if top == 0.0:
        return -110
    m, e = math.frexp(top / 448.0)
    return max(e - 1 if m == 0.5 else e, -110)


def pages_of(lens, page, seed=0, spare=2):
    """(pages in the pool, block table): the sequences' pages in a shuffled pool, -1 behind them."""
    counts = [max(1, -(-n // page)) for n in lens]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(counts) + spare, generator=g).tolist()
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32)
    for s, c in enumerate(counts):
        table[s, :c] = torch.tensor(order[:c], dtype=torch.int32)
        order = order[c:]
    return sum(counts) + spare, table


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def starts(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


def rotated(x, pos, freq, half, mult=1.0):
    """x [rows, heads, d] turned in 64 bits."""
    y = x.double().clone()
    n = 0 if freq is None else freq.numel()
    for i in range(n):
        a, b = (i, i + n) if half else (2 * i, 2 * i + 1)
        t = (pos.double() * freq[i].double().item()).view(-1, 1)
        y[:, :, a] = mult * (x[:, :, a].double() * t.cos() - x[:, :, b].double() * t.sin())
        y[:, :, b] = mult * (x[:, :, b].double() * t.cos() + x[:, :, a].double() * t.sin())
    return y


def quantised(x):
    """What a cache holds of rows x [positions, heads, width] that came in one call, from position 0 on: values in 64 bits, exponents."""
    out, exps = torch.zeros_like(x, dtype=torch.float64), []
    for b in range(0, x.shape[0], BLOCK):
        for g in range(x.shape[1]):
            part = x[b:b + BLOCK, g].double()
            e = exponent(part.abs().max().item())
            out[b:b + BLOCK, g] = (part * 2.0 ** -e).float().to(torch.float8_e4m3fn).double() * 2.0 ** e
            exps.append(e)
    return out, exps


def attention(q, k, v, pos, scale, window=0, first=0, softcap=0.0, sink=None, slope=None, penalty=None, kv_len=None):
    """One sequence in 64 bits: q [n, H, d] at positions pos [n], keys / values [L, G, .]; returns the result [n, H, dv], the sum of
    weight * |value| over the denominator, and the largest sum of |q_i k_i| * scale of each row."""
    n, H, _ = q.shape
    L, G, dv = v.shape
    out, spread, size = torch.zeros(n, H, dv, dtype=torch.float64, device=q.device), torch.zeros(n, H, dv, dtype=torch.float64, device=q.device), torch.zeros(n, H, 1, dtype=torch.float64, device=q.device)
    dist = pos.view(n, 1) - torch.arange(L, device=q.device)
    seen = dist >= 0
    if window:
        seen &= (dist < window) | (torch.arange(L, device=q.device) < first)
    if kv_len is not None:
        seen &= torch.arange(L, device=q.device) < kv_len
    for h in range(H):
        g = h // (H // G)
        s = q[:, h].double() @ k[:, g].double().T * scale
        size[:, h] = ((q[:, h].double().abs() @ k[:, g].double().abs().T) * abs(scale)).masked_fill(~seen, 0.0).nan_to_num(0.0).amax(1, keepdim=True) if L else 0.0
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if penalty is not None:
            s = s - penalty[0][h].double() * torch.log1p(penalty[1][h].double() * dist.clamp(min=0))
        if slope is not None:
            s = s - slope[h].double() * dist
        s = s.masked_fill(~seen, -math.inf)
        for i in range(n):
            on = seen[i].nonzero().flatten()
            if on.numel() == 0:
                continue
            z = s[i, on]
            top = max(z.max().item(), sink[h].item() if sink is not None else -math.inf)
            w = torch.exp(z - top)
            total = w.sum() + (math.exp(sink[h].item() - top) if sink is not None else 0.0)
            out[i, h] = w @ v[on, g].double() / total
            spread[i, h] = w @ v[on, g].double().abs() / total
    return out, spread, size


def tolerance(dtype, want, spread, size, bent=0.0):
    """How far a result may be off, element by element.  Rounding of the result: half a step.  A weight's relative error times the sum of
    weight * |value|: its rounding, and 2^-22 from the exponential; its score's absolute error -- a
    product of d <= 256 terms is at most 32 tensor-core sums, each cut off below 2^-23 of what is summed, `size` at most (2^-18 size), the
    parts of the query 2^-22 size, roundings of the scaled score and of its difference to the maximum 2^-22 size, and what the soft cap and the
    penalties add, a few 2^-21 of their own size `bent`; the weighted sum itself, at most 32 cut-off sums in a warp's share (2^-18).

    A weight's rounding for float32: two f16 parts, 2^-22.  For bfloat16: two e4m3 parts.  Let the weight be x in [1, 2) of its binade.  e4m3 has three
    bits behind the point, steps of 2^-3, so the first part leaves a remainder of at most 2^-4.  The second part takes that remainder in a binade of
    at most [2^-5, 2^-4), whose steps are 2^-8, and is off by half of one: 2^-9 absolute, at most 2^-9 of x.  (A remainder of exactly 2^-4 is a
    power of two and exact.)  The f16 number taken apart is itself off by 2^-11."""
    part = 2.0 ** -9 + 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22
    return HALF_STEP[dtype] * want.abs() + (part + 2.0 ** -17 * (1.0 + size) + 2.0 ** -19 * bent) * spread + 1e-30
