"""The 8-bit key/value cache: appending with rotation, attention for few and for many rows, both together, and what they refuse."""
from __future__ import annotations

import math

import pytest
import torch

from cache8_util import BLOCK, HALF_STEP, attention, exponent, ints, pages_of, quantised, rotated, starts, tolerance

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed), device="cuda")


def cache_of(lens, page, G, d, dv, seed=0, garbage=True):
    """A cache whose unwritten places hold what an earlier user left there: large codes, NaN codes, scales of any kind."""
    from smoltts_b200.kv_cache import KVCache8

    n, table = pages_of(lens, page, seed)
    c = KVCache8.allocate(n, page, G, d, dv)
    if garbage:
        for x, w in ((c.k, d), (c.v, dv)):
            x.view(torch.uint8)[..., :w] = torch.randint(0, 256, x[..., :w].shape, generator=gen(seed + 1), device="cuda").to(torch.uint8)
        for x in (c.k_scale, c.v_scale):
            x.copy_(torch.exp2(torch.randint(-20, 21, x.shape, generator=gen(seed + 2), device="cuda").float()))
            x[::3] = -x[::3]
    return c, table.cuda()


def held(c, table, s, length):
    k, v = c.values(table[s].clamp(min=0).long())
    return k.transpose(1, 2).reshape(-1, c.kv_heads, c.dim)[:length], v.transpose(1, 2).reshape(-1, c.kv_heads, c.vdim)[:length]


def fill(c, table, lens, seed=0, scale=1.0, dtype=torch.float32):
    """The sequences' first positions, in one call."""
    T = sum(lens)
    k, v = randn(T, c.kv_heads, c.dim, seed=seed + 5).to(dtype) * scale, randn(T, c.kv_heads, c.vdim, seed=seed + 6).to(dtype) * scale
    c.append(k, v, ints(starts(lens)), ints([0] * len(lens)), table, max_new=max(lens))
    return k, v


def check_attention(c, table, q, counts, pos0, out, **options):
    at, kv_len = starts(counts), options.pop("kv_len", None)
    for s, n in enumerate(counts):
        if n == 0:
            continue
        L = pos0[s] + n
        k, v = held(c, table, s, max(L, 0))
        pos = torch.arange(pos0[s], pos0[s] + n, device="cuda")
        want, spread, size = attention(q[at[s]:at[s] + n], k, v, pos, options.get("scale", c.dim ** -0.5), kv_len=None if kv_len is None else kv_len[s],
                                       **{x: options[x] for x in ("window", "first", "softcap", "sink", "slope", "penalty") if x in options})
        bent = options.get("softcap", 0.0) + (options["slope"].max().item() * L if options.get("slope") is not None else 0.0)
        if options.get("penalty") is not None:
            bent += options["penalty"][0].abs().max().item() * math.log1p(options["penalty"][1].max().item() * L)
        far = (out[at[s]:at[s] + n].double() - want).abs() - tolerance(q.dtype, want, spread, size, bent)
        assert far.max().item() <= 0, (s, far.max().item(), (far > 0).float().mean().item())


# ---------------------------------------------------------------------------------------------- append

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G,d,dv,page", [(2, 64, 64, 16), (4, 128, 128, 64), (1, 16, 48, 32), (3, 80, 72, 48), (2, 33, 7, 16), (1, 256, 200, 16), (2, 1, 3, 32)])
def test_append_writes_what_the_definition_says(dtype, G, d, dv, page):
    """Without a rotation nothing is rounded before the codes: equal to the bit, whatever lay there."""
    lens = [1, 15, 16, 17, 50, 3]
    c, table = cache_of(lens, page, G, d, dv)
    before = c.k.view(torch.uint8).clone(), c.k_scale.clone()
    k, v = fill(c, table, lens, scale=3.0, dtype=dtype)
    at = starts(lens)
    for s, n in enumerate(lens):
        got_k, got_v = held(c, table, s, n)
        for got, x in ((got_k, k), (got_v, v)):
            want, _ = quantised(x[at[s]:at[s] + n])
            assert torch.equal(got.double(), want)
    # scales: blocks of the sequences only; rows behind the last position as they were
    per = page // BLOCK
    used = {(int(table[s, b // per]), b % per): s for s, n in enumerate(lens) for b in range(-(-n // BLOCK))}
    for p in range(c.n_pages):
        for b in range(per):
            if (p, b) not in used:
                assert torch.equal(c.k_scale[p, :, b], before[1][p, :, b]) and torch.equal(c.k.view(torch.uint8)[p, :, b * BLOCK:(b + 1) * BLOCK], before[0][p, :, b * BLOCK:(b + 1) * BLOCK])
    s, n = 3, 17
    p, b = int(table[s, 1 // per if per else 1]) if page == BLOCK else int(table[s, 0]), (0 if page == BLOCK else 1)
    assert torch.equal(c.k.view(torch.uint8)[p, :, b * BLOCK + 1:(b + 1) * BLOCK], before[0][p, :, b * BLOCK + 1:(b + 1) * BLOCK])
    assert (c.k.view(torch.uint8)[..., d:] == 0).all() and (c.v.view(torch.uint8)[..., dv:] == 0).all()
    c.check_device_errors()


def test_a_scale_that_grows_takes_the_older_codes_along():
    """Token by token with magnitudes that rise, fall and rise again; the exponent is the largest needed so far, codes that stay normal keep
    their bits, and a call that repeats the last one changes nothing."""
    c, table = cache_of([40], 32, 1, 32, 32)
    x = randn(40, 1, 32, seed=3) * torch.exp2(torch.tensor([0, 3, 1, 8, -4, 8, 12, 0] * 5, device="cuda").float()).view(-1, 1, 1)
    want = torch.zeros(40, 32, dtype=torch.float64, device="cuda")
    e = 0
    for p in range(40):
        c.append(x[p:p + 1], -x[p:p + 1], ints([0, 1]), ints([p]), table, max_new=1)
        need, b = exponent(x[p].abs().max().item()), p - p % BLOCK
        old, e = e, need if p % BLOCK == 0 else max(e, need)
        if p % BLOCK:
            want[b:p] = (want[b:p] * 2.0 ** -e).float().to(torch.float8_e4m3fn).double() * 2.0 ** e
        want[p] = (x[p, 0].double() * 2.0 ** -e).float().to(torch.float8_e4m3fn).double() * 2.0 ** e
        k, v = held(c, table, 0, p + 1)
        assert torch.equal(k[:, 0].double(), want[:p + 1]) and torch.equal(v, -k)
        assert c.k_scale[table[0, p // 32], 0, p % 32 // BLOCK].item() == 2.0 ** e
    kept = c.k.view(torch.uint8).clone()
    c.append(x[39:], -x[39:], ints([0, 1]), ints([39]), table, max_new=1)
    assert torch.equal(kept, c.k.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,pairs,half,mult", [(64, 32, True, 1.0), (128, 64, False, 1.0), (96, 16, True, 1.25), (80, 40, True, 1.0), (33, 5, True, 1.0), (33, 5, False, 1.0), (256, 128, True, 1.0), (256, 127, False, 1.0)])
def test_rotation(dtype, d, pairs, half, mult):
    """Near and far positions.  A rotated element's error: 2^-22 of both terms (sine and cosine, two roundings), then the code's half step (2^-4 of the value, 2^-10 of
    the scale below the smallest normal code), or the query's own."""
    lens, pos0, H = [5, 37], [0, 99990], 6
    c, table = cache_of([5, 99990 + 37], 64, 2, d, 16, garbage=False)
    freq = (10000.0 ** (-torch.arange(pairs, device="cuda") / pairs)).float()
    T = sum(lens)
    k, v, q = randn(T, 2, d, seed=1).to(dtype), randn(T, 2, 16, seed=2).to(dtype), randn(T, H, d, seed=3).to(dtype)
    got = c.append(k, v, ints(starts(lens)), ints(pos0), table, max_new=37, q=q, freq=freq, rot_half=half, rot_mult=mult)
    at = starts(lens)
    for s, n in enumerate(lens):
        pos = torch.arange(pos0[s], pos0[s] + n, device="cuda")
        size = 2.0 * mult * 2.0 ** -22
        want = rotated(q[at[s]:at[s] + n], pos, freq, half, mult)
        err = (got[at[s]:at[s] + n].double() - want).abs()
        assert (err <= HALF_STEP[dtype] * want.abs() * 1.01 + size * q.abs().max().item()).all(), err.max()
        want = rotated(k[at[s]:at[s] + n], pos, freq, half, mult)
        k8, _ = held(c, table, s, pos0[s] + n)
        scale = c.k_scale[table[s].clamp(min=0).long()].transpose(1, 2).reshape(-1, 2)[pos // BLOCK].double().unsqueeze(-1)
        err = (k8[pos0[s]:].double() - want).abs()
        assert (err <= 2.0 ** -4 * want.abs() * 1.01 + 2.0 ** -10 * scale + size * k.abs().max().item()).all(), err.max()


def test_append_takes_slices_and_leaves_other_rows_alone():
    """Slices of a fused projection, odd strides, a padded batch: rows in front of the first sequence, an empty one, rows behind the last."""
    H, G, d, T = 4, 2, 24, 30
    c, table = cache_of([9, 1, 30], 16, G, d, d)
    fused = randn(T, (H + 2 * G) * d + 3, seed=8)
    q, k, v = fused[:, :H * d].view(T, H, d), fused[:, H * d:(H + G) * d].view(T, G, d), fused[:, (H + G) * d:(H + 2 * G) * d].view(T, G, d)
    out = torch.full((T, H, d), 7.0, device="cuda")
    c.append(k, v, ints([2, 11, 11, 25]), ints([0, 0, 3]), table, max_new=14, q=q, q_out=out)
    assert torch.equal(out[2:25], q[2:25]) and (out[:2] == 7).all() and (out[25:] == 7).all()
    assert torch.equal(held(c, table, 0, 9)[0].double(), quantised(k[2:11])[0])
    e = c.k_scale[table[2, 0].long(), :, 0].abs()
    got = held(c, table, 2, 16)[1][3:16].double()
    scale = c.v_scale[table[2, 0].long(), :, 0].abs().double().view(1, G, 1)
    assert torch.equal(got, (v[11:24].double() / scale).float().to(torch.float8_e4m3fn).double() * scale) and (e > 0).all()
    c.check_device_errors()


def test_append_of_infinities_nan_and_extremes():
    c, table = cache_of([48], 16, 1, 16, 16, garbage=False)
    x = torch.zeros(48, 1, 16, device="cuda")
    x[0, 0, 0], x[1, 0, 1], x[2, 0, 2], x[3, 0, 3] = math.inf, -math.inf, 3e38, 1.0
    x[16, 0, 5], x[17, 0, 1] = math.nan, 2.0
    x[32:] = torch.tensor(2.0 ** -140)
    c.append(x, x, ints([0, 48]), ints([0]), table, max_new=48)
    k, _ = held(c, table, 0, 48)
    assert k[0, 0, 0] == 2.0 ** 100 and k[1, 0, 1] == -2.0 ** 100 and k[2, 0, 2] == 2.0 ** 100 and k[3, 0, 3] == 0
    assert torch.isnan(k[16, 0, 5]) and k[17, 0, 1] == 2.0 and torch.isnan(k).sum() == 1
    assert c.k_scale[table[0, 1], 0, 0] < 0 and c.k_scale[table[0, 0], 0, 0] > 0 and (k[32:] == 0).all()
    c.append(x[17:18], x[17:18], ints([0, 1]), ints([18]), table, max_new=1)      # a later token of the block: the mark stays
    assert c.k_scale[table[0, 1], 0, 0] < 0


# ---------------------------------------------------------------------------------------------- attention, few rows

FEW = [
    # heads, kv_heads, d, dv, page, counts, pos0
    (12, 4, 64, 64, 64, [1], [0]),
    (12, 4, 64, 64, 64, [1, 1, 1, 1], [2047, 15, 16, 700]),
    (8, 8, 128, 128, 16, [1, 1], [63, 4000]),
    (32, 4, 128, 128, 32, [2, 5, 1], [100, 11, 0]),
    (3, 1, 80, 72, 48, [3, 1], [50, 333]),
    (40, 2, 33, 7, 16, [1, 2], [1, 70]),
    (4, 2, 256, 200, 64, [1, 3], [129, 20]),
    (2, 1, 1, 1, 16, [1, 1], [30, 5]),
    (1, 1, 64, 64, 128, [1], [20000]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,d,dv,page,counts,pos0", FEW)
def test_attention_of_few_rows(dtype, H, G, d, dv, page, counts, pos0):
    lens = [p + n for p, n in zip(pos0, counts)]
    c, table = cache_of(lens, page, G, d, dv, seed=H)
    fill(c, table, lens, seed=H)
    q = randn(sum(counts), H, d, seed=4).to(dtype)
    out = c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=max(counts), max_len=max(lens))
    check_attention(c, table, q, counts, pos0, out)
    c.check_device_errors()


OPTIONS = {
    "window": dict(window=20), "window_of_one": dict(window=1), "window_first": dict(window=37, first=5), "window_first_blocks": dict(window=64, first=33),
    "first_beyond": dict(window=10, first=10000), "softcap": dict(softcap=5.0), "slope": dict(slope=0.05), "penalty": dict(penalty=(0.7, 0.3)), "sink": dict(sink=1.5),
    "all": dict(window=90, first=3, softcap=8.0, slope=0.01, penalty=(0.2, 1.0), sink=-0.5, scale=0.3),
}


def options_of(name, H):
    o = dict(OPTIONS[name])
    ramp = torch.linspace(0.5, 1.5, H, device="cuda")
    for x in ("slope", "sink"):
        if x in o:
            o[x] = o[x] * ramp
    if "penalty" in o:
        o["penalty"] = (o["penalty"][0] * ramp, o["penalty"][1] * ramp)
    return o


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", list(OPTIONS))
@pytest.mark.parametrize("counts,pos0", [([1, 1, 1], [200, 36, 1]), ([40, 3], [150, 90]), ([150], [0])])
def test_masks_and_scores(dtype, name, counts, pos0):
    H, G, d = 6, 2, 64
    lens = [p + n for p, n in zip(pos0, counts)]
    c, table = cache_of(lens, 32, G, d, d, seed=2)
    fill(c, table, lens, seed=2)
    q = randn(sum(counts), H, d, seed=4).to(dtype)
    o = options_of(name, H)
    out = c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=max(counts), max_len=max(lens), **o)
    check_attention(c, table, q, counts, pos0, out, **o)


@pytest.mark.parametrize("n", [1, 70])
def test_rows_that_see_nothing_are_zeros(n):
    """Hidden keys (kv_len), no positions at all, a window that the hidden keys have left empty; with a sink, and next to a row that sees something."""
    H, G, d = 4, 2, 128
    pos0, counts, kv_len = [100, 50, 300], [n, n, n], [0, 20, 310]
    lens = [p + c for p, c in zip(pos0, counts)]
    c, table = cache_of(lens, 64, G, d, d)
    fill(c, table, lens)
    q = randn(3 * n, H, d, seed=4).to(torch.bfloat16)
    for o in (dict(), dict(sink=torch.ones(H, device="cuda")), dict(window=10), dict(window=10, first=3)):
        out = c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=n, max_len=max(lens), kv_len=ints(kv_len), **o)
        assert (out[:n] == 0).all()
        if o.get("window") and not o.get("first"):
            assert (out[n:2 * n] == 0).all()
        check_attention(c, table, q, counts, pos0, out, kv_len=kv_len, **o)
    out = c.attend(q[:n], ints([0, n]), ints([-n]), table[:1], max_new=n, max_len=1)      # every row in front of the sequence's first position
    assert (out == 0).all()


@pytest.mark.parametrize("n", [1, 90])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_shows_where_it_is_seen_and_nowhere_else(n, dtype):
    H, G, d, L = 4, 2, 64, 200
    c, table = cache_of([L + n], 32, G, d, d)
    k, v = randn(L + n, G, d, seed=1), randn(L + n, G, d, seed=2)
    k[30, 0, 3], v[70, 1, 9], v[L + n - 1, 0, 5], v[100, 0, 1] = math.nan, math.nan, math.nan, math.inf
    c.append(k, v, ints([0, L + n]), ints([0]), table, max_new=L + n)
    q = randn(n, H, d, seed=3).to(dtype)
    pos = torch.arange(L, L + n, device="cuda")
    for window, first in ((0, 0), (60, 0), (60, 31), (60, 30), (150, 71)):
        out = c.attend(q, ints([0, n]), ints([L]), table, max_new=n, max_len=L + n, window=window, first=first)

        def seen(j):
            return (pos >= j) & (((pos - j) < window) | (j < first) if window else torch.ones_like(pos, dtype=torch.bool))

        want = torch.zeros(n, H, d, dtype=torch.bool, device="cuda")
        want[:, :2] |= seen(30).view(-1, 1, 1)
        want[:, 2:, 9] |= seen(70).view(-1, 1)
        want[:, :2, 5] |= seen(L + n - 1).view(-1, 1)
        assert torch.equal(torch.isnan(out), want), (window, first)
        assert torch.isfinite(out[~want]).all()
    for bad in (math.nan, math.inf):
        q2 = q.clone()
        q2[0, 1, 7] = bad
        out = c.attend(q2, ints([0, n]), ints([20]), table, max_new=n, max_len=L, kv_len=ints([29]))
        assert torch.isnan(out[0, 1]).all() and torch.isfinite(out[0, 0]).all() and torch.isfinite(out[1:]).all()


def test_value_scales_far_apart():
    """Blocks whose values differ by 2^40: each weighs what it is worth; small ones in front of large ones and behind them."""
    H, G, d = 2, 1, 64
    for order in ([1.0, 2.0 ** 20, 2.0 ** -20, 2.0 ** 5], [2.0 ** -20, 1.0, 2.0 ** 3, 2.0 ** -12]):
        L = 64 * len(order)
        c, table = cache_of([L], 64, G, d, d)
        k, v = randn(L, G, d, seed=1), randn(L, G, d, seed=2) * torch.tensor(order, device="cuda").repeat_interleave(64).view(-1, 1, 1)
        c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
        q = randn(1, H, d, seed=3)
        out = c.attend(q, ints([0, 1]), ints([L - 1]), table, max_new=1, max_len=L)
        check_attention(c, table, q, [1], [L - 1], out)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1e4, 1e20])
def test_queries_of_any_size(scale):
    H, G, d, L = 4, 2, 128, 333
    c, table = cache_of([L], 64, G, d, d)
    fill(c, table, [L])
    for dtype in (torch.bfloat16, torch.float32):
        q = (randn(1, H, d, seed=3) * scale).to(dtype)
        out = c.attend(q, ints([0, 1]), ints([L - 1]), table, max_new=1, max_len=L, scale=d ** -0.5 / scale)
        check_attention(c, table, q, [1], [L - 1], out, scale=d ** -0.5 / scale)


# ---------------------------------------------------------------------------------------------- attention, many rows

MANY = [
    (4, 4, 64, 64, 64, [300], [0]), (12, 4, 64, 64, 16, [129, 257], [0, 77]), (8, 2, 128, 128, 64, [200, 31, 128], [500, 0, 1]), (3, 1, 80, 72, 32, [333], [50]),
    (4, 2, 33, 7, 16, [65, 66], [1, 0]), (4, 2, 256, 200, 64, [90], [129]), (16, 2, 128, 64, 48, [100], [1000]), (2, 2, 64, 128, 32, [513], [0]), (10, 2, 96, 128, 64, [140, 9], [3, 300]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,d,dv,page,counts,pos0", MANY)
def test_attention_of_many_rows(dtype, H, G, d, dv, page, counts, pos0):
    lens = [p + n for p, n in zip(pos0, counts)]
    c, table = cache_of(lens, page, G, d, dv, seed=H)
    fill(c, table, lens, seed=H)
    q = randn(sum(counts), H, d, seed=4).to(dtype)
    out = c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=max(counts), max_len=max(lens))
    check_attention(c, table, q, counts, pos0, out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G", [(8, 2), (40, 1)])
def test_portions_and_single_tokens_in_one_batch(dtype, H, G):
    """Long contexts: sequences of few rows beside one of many, which may go to different kernels; the shares of either are joined."""
    d, counts, pos0 = 64, [1, 150, 0, 3, 9, 1], [5000, 100, 7, 2500, 3000, 0]
    lens = [p + n for p, n in zip(pos0, counts)]
    c, table = cache_of(lens, 64, G, d, d, seed=1)
    fill(c, table, lens, seed=1)
    q = randn(sum(counts) + 2, H, d, seed=4).to(dtype)
    for o in (dict(), dict(window=700, first=5)):
        out = torch.full((sum(counts) + 2, H, d), 7.0, device="cuda", dtype=dtype)
        c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=150, max_len=max(lens), out=out, **o)
        check_attention(c, table, q, counts, pos0, out, **o)
        assert (out[sum(counts):] == 7).all()
    one = c.attend(q[:1], ints([0, 1]), ints([5000]), table[:1], max_new=1, max_len=5001, window=700, first=5)      # a row does not depend on its company
    assert (one.double() - out[:1].double()).abs().max() <= 4 * HALF_STEP[dtype] * out[:1].abs().max() if dtype == torch.bfloat16 else torch.allclose(one, out[:1], rtol=1e-4, atol=1e-5)


def test_strides_and_rows_of_nobody():
    """Queries and results as slices of something wider; rows in front, behind and of sequences without rows stay as they were."""
    H, G, d = 4, 2, 64
    for n in (2, 100):
        counts, pos0 = [n, 0, n], [30, 5, 200]
        lens = [p + m for p, m in zip(pos0, counts)]
        c, table = cache_of(lens, 32, G, d, d)
        fill(c, table, lens)
        for pad in (0, 3, 8):
            wide = randn(2 * n + 6, H, d + pad, seed=3).to(torch.bfloat16)
            q = wide[..., pad:]
            out = torch.full((2 * n + 6, H, d + pad), 7.0, device="cuda", dtype=torch.bfloat16)
            c.attend(q, ints([2, 2 + n, 2 + n, 2 + 2 * n]), ints(pos0), table, max_new=n, max_len=max(lens), out=out[..., :d])
            check_attention(c, table, q[2:], counts, pos0, out[2:, :, :d])
            assert (out[:2] == 7).all() and (out[2 + 2 * n:] == 7).all() and (out[..., d:] == 7).all()


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_windows_and_first_positions_of_any_size(n, dtype):
    """The largest numbers that the arguments hold: everything is visible."""
    H, G, d, L, most = 4, 2, 64, 700, 2 ** 31 - 1
    c, table = cache_of([L], 64, G, d, d)
    fill(c, table, [L])
    q = randn(n, H, d, seed=3).to(dtype)
    for window, first in ((16, most), (16, most - 100), (most, 0), (most, most), (most - 5, 3)):
        options = dict(window=window, first=first)
        check_attention(c, table, q, [n], [L - n], c.attend(q, ints([0, n]), ints([L - n]), table, max_new=n, max_len=L, **options), **options)


def test_host_numbers_that_are_too_small():
    """A longer sequence than max_len is attended to as a whole; rows beyond max_new are left as they were."""
    H, G, d = 4, 2, 64
    c, table = cache_of([3000], 64, G, d, d)
    fill(c, table, [3000])
    q = randn(1, H, d, seed=3)
    check_attention(c, table, q, [1], [2999], c.attend(q, ints([0, 1]), ints([2999]), table, max_new=1, max_len=10))
    q = randn(5, H, d, seed=3)
    out = torch.full((5, H, d), 7.0, device="cuda")
    c.attend(q, ints([0, 5]), ints([2995]), table, max_new=3, max_len=3000, out=out)
    check_attention(c, table, q[:3], [3], [2995], out[:3])
    assert (out[3:] == 7).all()


def test_pages_outside_the_cache_are_reported_and_not_touched():
    from smoltts_b200._errors import SmolError

    H, G, d = 4, 2, 64
    c, table = cache_of([100], 32, G, d, d)
    fill(c, table, [100])
    bad = table.clone()
    bad[0, 1] = c.n_pages
    before = c.k.view(torch.uint8).clone()
    q = randn(1, H, d, seed=3)
    assert torch.isfinite(c.attend(q, ints([0, 1]), ints([99]), bad, max_new=1, max_len=100)).all()
    with pytest.raises(SmolError):
        c.check_device_errors()
    c._err.zero_()
    k = randn(1, G, d)
    c.append(k, k, ints([0, 1]), ints([40]), bad, max_new=1)
    assert torch.equal(before, c.k.view(torch.uint8))
    with pytest.raises(SmolError):
        c.check_device_errors()
    c._err.zero_()
    c.append(k, k, ints([0, 1]), ints([200]), table, max_new=1)      # behind the table's last page
    with pytest.raises(SmolError):
        c.check_device_errors()


# ---------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_portions_then_tokens(dtype):
    """As a layer is served: portions of two prompts, then tokens of both, rotation on the way, a window with first tokens; each step against the
    cache's own contents, and the contents against what was appended."""
    H, G, d, page = 8, 2, 64, 32
    c, table = cache_of([400, 400], page, G, d, d)
    freq = (10000.0 ** (-torch.arange(d // 2, device="cuda") / (d // 2))).float()
    pos0, seen_k = [0, 0], [[], []]
    for step, counts in enumerate([[100, 1], [37, 150], [1, 1], [1, 1], [60, 3], [1, 0], [5, 1]]):
        T = sum(counts)
        q, k, v = (randn(T, h, d, seed=10 * step + i).to(dtype) for i, h in enumerate((H, G, G)))
        qr = c.append(k, v, ints(starts(counts)), ints(pos0), table, max_new=max(counts), q=q, freq=freq)
        o = dict(window=64, first=4)
        out = c.attend(qr, ints(starts(counts)), ints(pos0), table, max_new=max(counts), max_len=max(p + n for p, n in zip(pos0, counts)), **o)
        check_attention(c, table, qr, counts, pos0, out, **o)
        for s, n in enumerate(counts):
            at = starts(counts)[s]
            seen_k[s].append(rotated(k[at:at + n], torch.arange(pos0[s], pos0[s] + n, device="cuda"), freq, True))
            pos0[s] += n
    for s in range(2):
        want, (got, _) = torch.cat(seen_k[s]), held(c, table, s, pos0[s])
        # codes of a block that grew were rounded twice: at most a whole step
        scale = c.k_scale[table[s].clamp(min=0).long()].transpose(1, 2).reshape(-1, G)[:-(-pos0[s] // BLOCK)].repeat_interleave(BLOCK, 0)[:pos0[s]].double().unsqueeze(-1)
        assert ((got.double() - want).abs() <= 2.0 ** -3 * want.abs() + 2.0 ** -9 * scale + 1e-5).all()


def test_captured_and_on_other_streams():
    """Both calls in one graph, replayed on new contents, two graphs side by side on two streams, and an eager call beside them."""
    H, G, d, n = 8, 2, 128, 3
    jobs = []
    for j in range(2):
        c, table = cache_of([900, 500, 70], 64, G, d, d, seed=j)
        fill(c, table, [890, 490, 60], seed=j)
        q, k, v = (randn(n, h, d, seed=20 + 3 * j + i).to(torch.bfloat16) for i, h in enumerate((H, G, G)))
        start, pos0 = ints([0, 1, 2, 3]), ints([890, 490, 60])
        jobs.append((c, table, q, k, v, start, pos0))

    def step(job):
        c, table, q, k, v, start, pos0 = job
        c.append(k, v, start, pos0, table, max_new=1)
        return c.attend(q, start, pos0, table, max_new=1, max_len=900)

    eager = [step(j).clone() for j in jobs]
    graphs, outs = [], []
    for j in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(j))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, outs))
    for j in jobs:
        j[2].copy_(-j[2])
        j[3].mul_(2)
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        again = [step(j) for j in jobs]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, outs))


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes of key codes: the pages at its end."""
    from smoltts_b200.kv_cache import KVCache8

    G, d, page = 8, 128, 128
    n = (1 << 32) // (G * d * page) + 64
    k = torch.zeros(n, G, page, d, dtype=torch.float8_e4m3fn, device="cuda")
    v = torch.zeros(n, G, page, d, dtype=torch.float8_e4m3fn, device="cuda")
    s = [torch.zeros(n, G, page // BLOCK, device="cuda") for _ in range(2)]
    c = KVCache8(k, v, s[0], s[1])
    for rows in (1, 200):
        table = torch.tensor([[n - 1, n - 3, n - 2]], dtype=torch.int32, device="cuda")
        fill(c, table, [300])
        assert not c.k.view(torch.uint8)[:n - 3].any()
        q = randn(rows, 16, d, seed=3).to(torch.bfloat16)
        out = c.attend(q, ints([0, rows]), ints([300 - rows]), table, max_new=rows, max_len=300)
        check_attention(c, table, q, [rows], [300 - rows], out)


def test_refusals():
    from smoltts_b200._errors import SmolError
    from smoltts_b200.kv_cache import KVCache8

    H, G, d = 4, 2, 64
    c, table = cache_of([64], 32, G, d, d)
    start, pos0, k, q = ints([0, 1]), ints([0]), randn(1, G, d), randn(1, H, d)

    def refused(call, *a, **o):
        with pytest.raises((ValueError, SmolError)):
            call(*a, **o)

    for bad in (k.half(), k.cpu(), randn(1, G, d + 1), randn(1, G + 1, d), randn(1, d, G).transpose(1, 2), k[0]):
        refused(c.append, bad, k, start, pos0, table, max_new=1)
        refused(c.append, k, bad, start, pos0, table, max_new=1)
    refused(c.append, k, k.bfloat16(), start, pos0, table, max_new=1)
    refused(c.append, k, k, start.long(), pos0, table, max_new=1)
    refused(c.append, k, k, start, ints([0, 0]), table, max_new=1)
    refused(c.append, k, k, start, pos0, table[0], max_new=1)
    refused(c.append, k, k, start, pos0, table, max_new=0)
    refused(c.append, k, k, start, pos0, table, max_new=1, q_out=q)
    refused(c.append, k, k, start, pos0, table, max_new=1, q=q, q_out=q)
    refused(c.append, k, k, start, pos0, table, max_new=1, q=q.bfloat16())
    refused(c.append, k, k, start, pos0, table, max_new=1, freq=torch.ones(33, device="cuda"))
    refused(c.append, k, k, start, pos0, table, max_new=1, freq=torch.ones(3, device="cuda").double())
    for o in (dict(window=-1), dict(first=-1), dict(softcap=-1.0), dict(softcap=math.nan), dict(sink=torch.ones(3, device="cuda")), dict(slope=torch.ones(H)), dict(max_len=0),
              dict(out=torch.empty(1, H, d, device="cuda", dtype=torch.bfloat16)), dict(out=torch.empty(2, H, d, device="cuda")), dict(kv_len=ints([1, 2])),
              dict(out=torch.empty(1, 1, d, device="cuda").expand(1, H, d))):
        refused(c.attend, q, start, pos0, table, **{"max_new": 1, "max_len": 64, **o})
    refused(c.attend, randn(1, 3, d), start, pos0, table, max_new=1, max_len=64)
    refused(c.attend, q.half(), start, pos0, table, max_new=1, max_len=64)
    refused(KVCache8.allocate, 4, 24, G, d)
    refused(KVCache8.allocate, 0, 32, G, d)
    refused(KVCache8, c.k, c.v, c.k_scale[..., :1], c.v_scale)
    refused(KVCache8, c.k, c.v, c.k_scale, c.v_scale, dim=32)
    refused(KVCache8, c.k.view(torch.uint8), c.v, c.k_scale, c.v_scale)
    wide = KVCache8.allocate(4, 16, 1, 272)
    refused(wide.append, randn(1, 1, 272), randn(1, 1, 272), start, pos0, ints([[0]]), max_new=1)
    refused(wide.attend, randn(1, 1, 272), start, pos0, ints([[0]]), max_new=1, max_len=1)


@pytest.mark.parametrize("n", [2, 40])
def test_results_that_overlap_what_is_read_or_themselves_are_refused(n):
    H, G, d = 4, 2, 64
    c, table = cache_of([64], 32, G, d, d)
    fill(c, table, [64])
    batch, room = (ints([0, n]), ints([64 - n]), table), torch.zeros(4 * n * H * d, device="cuda", dtype=torch.bfloat16)
    cut = lambda at, *stride: room.as_strided((n, H, d), stride or (H * d, d, 1), at)  # noqa: E731
    q, k, v = cut(0), randn(n, G, d, seed=4).to(torch.bfloat16), randn(n, G, d, seed=5).to(torch.bfloat16)
    q.copy_(randn(n, H, d, seed=3))
    far = n * H * d
    for out in (q, cut(d), cut(far - 1), cut(far, d, d, 1), cut(far, H * d, d - 1, 1), cut(far, (H - 1) * d, d, 1), cut(far, d, (n - 1) * d, 1)):
        with pytest.raises(ValueError):
            c.attend(q, *batch, max_new=n, max_len=64, out=out)
        with pytest.raises(ValueError):
            c.append(k, v, *batch, max_new=n, q=q, q_out=out)
    with pytest.raises(ValueError):
        c.append(k, v, *batch, max_new=n, q=randn(n, G, d).to(torch.bfloat16), q_out=k)
    # what lies apart in the same memory, and heads in front of rows, are served
    for out in (cut(far), cut(far, d, n * d, 1), cut(far, H * d + 24, d + 8, 1)):
        if n == 2 or out.stride(0) != H * d + 24:
            check_attention(c, table, q, [n], [64 - n], c.attend(q, *batch, max_new=n, max_len=64, out=out).contiguous())
            want = c.append(k, v, *batch, max_new=n, q=q)
            assert torch.equal(c.append(k, v, *batch, max_new=n, q=q, q_out=out), want)


def test_softcap_must_be_finite():
    c, table = cache_of([64], 32, 2, 64, 64)
    with pytest.raises(ValueError):
        c.attend(randn(1, 4, 64), ints([0, 1]), ints([63]), table, max_new=1, max_len=64, softcap=math.inf)


def test_device_words_are_told_apart():
    from smoltts_b200._errors import SmolError

    c, _ = cache_of([64], 32, 2, 64, 64)
    for word, text in ((1, "page outside"), (2, "do not fit"), (3, "ran out")):
        c._err.fill_(word)
        with pytest.raises(SmolError, match=text):
            c.check_device_errors()
