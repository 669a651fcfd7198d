"""The 8-bit key/value cache where magnitudes differ: a row's result depends on what it sees alone, however large or small what lies beside it is."""
from __future__ import annotations

import math

import pytest
import torch

from cache8_util import BLOCK, ints, tolerance
from test_gpu_cache8 import cache_of, randn

pytestmark = pytest.mark.gpu

# A weight's last bit, relative to the largest product of a weight and its block's scale that the row sees in the step.  Tiles of many rows: the second e4m3 part
# has the first one's unit, so half of its least code, 2^-10, on 256.  Few rows: the second part is 16 times finer.  float32: half of f16's least number, 2^-25, on
# at least 128.
LEAST_TILES, LEAST_FEW, LEAST_F32 = 2.0 ** -18, 2.0 ** -22, 2.0 ** -32


def check(c, table, q, pos0, out, least, scale=None, window=0, first=0, kv_len=None, sink=None, softcap=0.0):
    """One sequence's rows against 64 bits.  On top of `tolerance`: the weights' last bit times the codes it multiplies; and for bf16 2^-15 of the weights, from three roundings
    of a sum of a score and a block's exponent of at most 110, each 2^-24 of at most 160 (scores below 50 in units of log2) in units of log2."""
    n, H, d = q.shape
    G, page, pages = c.kv_heads, c.page_size, table[0][table[0] >= 0].long()
    L = pos0 + n
    k, _ = c.values(pages)
    k = k.double().transpose(1, 2).reshape(-1, G, d)[:L]
    codes = c.v.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double().transpose(1, 2).reshape(-1, G, c.v.shape[3])[:L, :, :c.vdim]
    unit = c.v_scale[pages].abs().double().transpose(1, 2).reshape(-1, G).repeat_interleave(BLOCK, 0)[:L]
    j = torch.arange(L, device="cuda")
    dist = torch.arange(pos0, L, device="cuda").view(n, 1) - j
    seen = dist >= 0
    if window:
        seen &= (dist < window) | (j < first)
    if kv_len is not None:
        seen &= j < kv_len
    some = seen.any(1, keepdim=True)
    for h in range(H):
        g = h // (H // G)
        scale_ = d ** -0.5 if scale is None else scale
        s = q[:, h].double() @ k[:, g].T * scale_
        s = (softcap * torch.tanh(s / softcap) if softcap else s).masked_fill(~seen, -math.inf)
        size = (q[:, h].double().abs() @ k[:, g].abs().T * scale_).masked_fill(~seen, 0.0).amax(1, keepdim=True)
        top = s.amax(1, keepdim=True).masked_fill(~some, 0.0)
        if sink is not None:
            top = top.clamp(min=sink[h].item())
        w = torch.exp(s - top)
        total = w.sum(1, keepdim=True) + (torch.exp(sink[h].double() - top) if sink is not None else 0.0)
        total = total.masked_fill(total == 0, 1.0)
        v = codes[:, g] * unit[:, g, None]
        want, spread = w @ v / total, w @ v.abs() / total
        floor = (w * unit[:, g]).amax(1, keepdim=True) * (seen.double() @ codes[:, g].abs()) / total
        tol = tolerance(q.dtype, want, spread, size) + least * floor + (2.0 ** -15 * spread if q.dtype == torch.bfloat16 else 0.0)
        far = ((out[:, h].double() - want).abs() - tol) / (spread + 1e-30)
        assert far.max().item() <= 0, (h, far.max().item(), (far > 0).any(1).nonzero().flatten().tolist()[:20])


def ones_column(q, k, at=8.0, key=0.0):
    """Coordinate 0 as a score of its own: with a scale of 1/8 a key's is its coordinate."""
    q[..., 0], k[..., 0] = at, key


KERNELS = [(torch.bfloat16, 1, LEAST_FEW), (torch.bfloat16, 7, LEAST_FEW), (torch.bfloat16, 150, LEAST_TILES), (torch.float32, 1, LEAST_F32),
           (torch.float32, 7, LEAST_F32), (torch.float32, 150, LEAST_F32)]


@pytest.mark.parametrize("dtype,n,least", KERNELS)
@pytest.mark.parametrize("power", [12, 30, 100])
@pytest.mark.parametrize("where", ["later", "behind_the_window", "behind_kv_len", "little_weight", "infinity", "between"])
def test_a_row_depends_on_what_it_sees_alone(dtype, n, least, power, where):
    """Values 2^power larger at positions that some or all rows do not see, or that weigh next to nothing (a score 40 lower, 2^-58)."""
    H, G, d, pos0 = 4, 2, 64, 246
    L = pos0 + n
    c, table = cache_of([L], 32, G, d, d, seed=3)
    k, v, q = randn(L, G, d, seed=1), randn(L, G, d, seed=2), randn(n, H, d, seed=3)
    ones_column(q, k)
    v *= 2.0 ** (-power / 2 if where == "between" else 0.0)
    big = torch.zeros(L, dtype=torch.bool, device="cuda")
    options = {}
    if where in ("later", "infinity"):
        big[pos0 + 1 if n == 1 else pos0 + n // 2:] = True
        if n == 1:      # (hidden in the last step all the same)
            big[pos0 - 10:], options["kv_len"] = True, pos0 - 16
    elif where == "behind_the_window":
        big[192:208], options["window"] = True, 40      # (the first row sees one of them)
        big[272:288] = True
    elif where == "behind_kv_len":
        big[240:], options["kv_len"] = True, 240 - 10
    elif where == "little_weight":
        big[224:240] = True
        k[224:240, :, 0] = -40.0
    else:
        big[192:208] = True
    v[big] *= 2.0 ** power
    if where == "infinity":
        v[big.nonzero()[-1].item(), :, 5] = math.inf
    q = q.to(dtype)
    c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
    o = {x: (ints([y]) if x == "kv_len" else y) for x, y in options.items()}
    out = c.attend(q, ints([0, n]), ints([pos0]), table, max_new=n, max_len=L, **o)
    check(c, table, q, pos0, out, least, **options)
    sink = torch.linspace(-1.0, 3.0, H, device="cuda")
    out = c.attend(q, ints([0, n]), ints([pos0]), table, max_new=n, max_len=L, sink=sink, **o)
    check(c, table, q, pos0, out, least, sink=sink, **options)
    c.check_device_errors()


@pytest.mark.parametrize("dtype,n,least", KERNELS)
@pytest.mark.parametrize("low", [0.0, 2.0 ** -90])
def test_blocks_of_zeros_and_of_everything(dtype, n, least, low):
    """Blocks of zeros (scale 2^-110) or next to nothing beside ordinary ones, and blocks near the largest there is: the denominator counts them all."""
    H, G, d, pos0 = 4, 2, 64, 250
    L = pos0 + n
    c, table = cache_of([L], 32, G, d, d, seed=3)
    k, v, q = randn(L, G, d, seed=1), randn(L, G, d, seed=2), randn(n, H, d, seed=3).to(dtype)
    for b in range(0, L, 2 * BLOCK):
        v[b:b + BLOCK] *= low
    c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
    check(c, table, q, pos0, c.attend(q, ints([0, n]), ints([pos0]), table, max_new=n, max_len=L), least)
    v[96:112] *= 2.0 ** 88      # (ordinary, tiny and huge in one step)
    c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
    for options in (dict(), dict(window=120)):
        check(c, table, q, pos0, c.attend(q, ints([0, n]), ints([pos0]), table, max_new=n, max_len=L, **options), least, **options)


@pytest.mark.parametrize("n", [1, 7, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shares_of_the_keys_whose_values_differ(dtype, n):
    """A long context in several shares, joined in a cluster or by a kernel of its own: values grow by 2^20 every 700 positions, scores fall by 12 meanwhile."""
    H, G, d = 4, 2, 64
    for L in (2100, 9000 if n < 9 else 3000):
        pos0 = L - n
        c, table = cache_of([L], 64, G, d, d, seed=3)
        k, v, q = randn(L, G, d, seed=1), randn(L, G, d, seed=2), randn(n, H, d, seed=3)
        ones_column(q, k)
        steps = (torch.arange(L, device="cuda") // 700).float()
        k[:, :, 0] = -12.0 * (steps % 4).view(-1, 1)
        v *= torch.exp2(20.0 * (steps % 4) - 30.0).view(-1, 1, 1)
        q = q.to(dtype)
        c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
        out = c.attend(q, ints([0, n]), ints([pos0]), table, max_new=n, max_len=L)
        check(c, table, q, pos0, out, LEAST_F32 if dtype == torch.float32 else LEAST_FEW if n < 9 else LEAST_TILES)


@pytest.mark.parametrize("n", [1, 150])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rise", [30.0, 40.0, 44.0])
def test_rising_scores_of_large_values(dtype, n, rise):
    """Scores that rise by 30 to 44 from one step of 128 positions to the next, values near 2^90 and a clamped infinity."""
    H, G, d, pos0 = 4, 2, 64, 500
    L = pos0 + n
    c, table = cache_of([L], 64, G, d, d, seed=3)
    k, v, q = randn(L, G, d, seed=1), randn(L, G, d, seed=2) * 2.0 ** 88, randn(n, H, d, seed=3)
    ones_column(q, k)
    k[:, :, 0] = ((torch.arange(L, device="cuda") // 128).float() * rise - 2 * rise).view(-1, 1)
    v[400, 0, 3], v[L - 1, 1, 9] = math.inf, -math.inf
    q = q.to(dtype)
    c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
    out = c.attend(q, ints([0, n]), ints([pos0]), table, max_new=n, max_len=L)
    assert torch.isfinite(out).all()
    check(c, table, q, pos0, out, LEAST_F32 if dtype == torch.float32 else LEAST_FEW if n == 1 else LEAST_TILES)


def test_a_sink_far_above_the_scores():
    """Scores 70 below the sink, values of 2^90: what is left is 2^-11."""
    H, G, d, L = 4, 2, 64, 300
    for dtype in (torch.bfloat16, torch.float32):
        for n in (1, 150):
            c, table = cache_of([L], 64, G, d, d, seed=3)
            k, v, q = randn(L, G, d, seed=1), randn(L, G, d, seed=2) * 2.0 ** 90, randn(n, H, d, seed=3).to(dtype)
            c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
            sink = torch.full((H,), 70.0, device="cuda")
            out = c.attend(q, ints([0, n]), ints([L - n]), table, max_new=n, max_len=L, sink=sink)
            check(c, table, q, L - n, out, LEAST_F32 if dtype == torch.float32 else LEAST_FEW if n == 1 else LEAST_TILES, sink=sink)


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 1), (torch.bfloat16, 150), (torch.float32, 150)])
@pytest.mark.parametrize("cap", [300.0, 1e4, 1e6, 1e9, 3.4e38])
@pytest.mark.parametrize("scale", [0.125, 60.0])
def test_soft_caps_far_above_the_scores(dtype, n, cap, scale):
    """Scores of up to 10 and 5000 under caps from below them to fp32's end: what a cap adds to a score's error is 2^-20 of the score, an eighth of what its size is given."""
    H, G, d, L = 4, 2, 64, 400
    c, table = cache_of([L], 32, G, d, d, seed=5)
    k, v, q = randn(L, G, d, seed=1), randn(L, G, d, seed=2), randn(n, H, d, seed=3).to(dtype)
    c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
    out = c.attend(q, ints([0, n]), ints([L - n]), table, max_new=n, max_len=L, scale=scale, softcap=cap)
    check(c, table, q, L - n, out, LEAST_F32 if dtype == torch.float32 else LEAST_FEW if n < 9 else LEAST_TILES, scale=scale, softcap=cap)


END = 2 ** 31 - 128      # positions are below this
BAD = [([0, 3], [2 ** 31 - 1]), ([0, 3], [2 ** 31 - 10]), ([0, 3], [END - 2]), ([2, 0], [5]), ([-1, 2], [5]), ([2 ** 31 - 1, -2 ** 31], [5]), ([1, 4], [5]), ([-2 ** 31, 3], [5])]


@pytest.mark.parametrize("start,pos0", BAD)
def test_append_to_arrays_that_do_not_fit(start, pos0):
    """Positions and rows outside their ranges, those whose sums pass 32 bits among them: reported, and nothing is written."""
    from smoltts_b200._errors import SmolError

    c, table = cache_of([40], 32, 2, 64, 64)
    before = [x.view(torch.uint8).clone() for x in (c.k, c.v, c.k_scale, c.v_scale)]
    k, v, q = randn(3, 2, 64, seed=1), randn(3, 2, 64, seed=2), randn(3, 4, 64, seed=3)
    out = torch.full((3, 4, 64), 7.0, device="cuda")
    c.append(k, v, ints(start), ints(pos0), table, max_new=3, q=q, q_out=out)
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, (c.k, c.v, c.k_scale, c.v_scale))) and (out == 7).all()
    with pytest.raises(SmolError, match="do not fit"):
        c.check_device_errors()


def test_append_behind_the_table():
    from smoltts_b200._errors import SmolError

    c, table = cache_of([40], 32, 2, 64, 64)
    k = randn(3, 2, 64, seed=1)
    before = c.k.view(torch.uint8).clone()
    c.append(k, k, ints([0, 3]), ints([END - 3]), table, max_new=3)
    assert torch.equal(before, c.k.view(torch.uint8))
    with pytest.raises(SmolError, match="page outside"):
        c.check_device_errors()


@pytest.mark.parametrize("dtype,n", [(torch.float32, 3), (torch.bfloat16, 3), (torch.bfloat16, 40)])
@pytest.mark.parametrize("L", [64, 3000])
def test_attention_of_arrays_that_do_not_fit(dtype, n, L):
    """A sequence that does not fit is left out, the other is served; positions behind the table are reported and the held ones attended to, without walking to them."""
    from smoltts_b200._errors import SmolError

    H, G, d = 4, 2, 64
    c, table = cache_of([L, L], 32, G, d, d)
    k, v = randn(2 * L, G, d, seed=1), randn(2 * L, G, d, seed=2)
    c.append(k, v, ints([0, L, 2 * L]), ints([0, 0]), table, max_new=L)
    q = randn(2 * n, H, d, seed=3).to(dtype)
    want = c.attend(q, ints([0, n, 2 * n]), ints([L - n, L - n]), table, max_new=n, max_len=L)
    c.check_device_errors()
    for first, pos in ((n, 2 ** 31 - 1), (n, 2 ** 31 - 10), (n, END - n + 1), (2 * n + 5, L - n)):
        out = torch.full((2 * n, H, d), 7.0, device="cuda", dtype=dtype)
        c.attend(q, ints([0, n, first + n if first == n else first]), ints([L - n, pos]), table, max_new=n, max_len=L, out=out)
        assert torch.equal(out[:n], want[:n]) and (out[n:] == 7).all()
        with pytest.raises(SmolError, match="do not fit"):
            c.check_device_errors()
        c._err.zero_()
    held = table.shape[1] * 32
    every = c.attend(q[n:], ints([0, n]), ints([held - n]), table[1:], max_new=n, max_len=L, kv_len=ints([held - n]))
    c.check_device_errors()
    far = c.attend(q[n:], ints([0, n]), ints([2 ** 30]), table[1:], max_new=n, max_len=L, kv_len=ints([held - n]))
    torch.testing.assert_close(far, every, rtol=0.0, atol=0.0, equal_nan=True)      # (behind the last held position lies what an earlier user left, NaNs too)
    c.check_device_errors()      # (hidden: nobody asks for the pages)
    c.attend(q[n:], ints([0, n]), ints([2 ** 30]), table[1:], max_new=n, max_len=L)
    with pytest.raises(SmolError, match="page outside"):
        c.check_device_errors()


@pytest.mark.parametrize("dtype,n", [(torch.float32, 8), (torch.bfloat16, 8), (torch.bfloat16, 40)])
def test_the_largest_window_and_rows_in_front_of_the_first_position(dtype, n):
    H, G, d, L = 4, 2, 64, n - 5
    c, table = cache_of([64], 32, G, d, d)
    k, v, q = randn(L, G, d, seed=1), randn(L, G, d, seed=2), randn(n, H, d, seed=3).to(dtype)
    c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
    want = c.attend(q, ints([0, n]), ints([-5]), table, max_new=n, max_len=L)
    assert (want[:5] == 0).all() and (want[5:] != 0).any()
    for window in (2 ** 31 - 1, 2 ** 31 - 4):
        assert torch.equal(c.attend(q, ints([0, n]), ints([-5]), table, max_new=n, max_len=L, window=window), want)


@pytest.mark.parametrize("n,context", [(300, 1000), (300, 12000), (420, 2000)])
def test_two_column_halves_share_the_keys(n, context):
    """Values of 200 columns take two blocks a tile: shares of the keys are counted for both, and few keys are not shared out beyond what the SMs hold."""
    H, G, d, dv, L = 4, 2, 128, 200, context + n
    c, table = cache_of([L], 64, G, d, dv, seed=3)
    k, v, q = randn(L, G, d, seed=1), randn(L, G, dv, seed=2), randn(n, H, d, seed=3).to(torch.bfloat16)
    c.append(k, v, ints([0, L]), ints([0]), table, max_new=L)
    out = c.attend(q, ints([0, n]), ints([context]), table, max_new=n, max_len=L)
    check(c, table, q, context, out, LEAST_TILES)


def test_shares_of_two_column_halves_fit_the_device():
    """A portion of 280 tokens of 16 and 8 heads: 40 tiles, 80 blocks with 200 columns.  Three shares of 80 would wait for one another; the keys are too few for that."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    H, G, d, L, n = 16, 8, 128, 1000, 280
    c, table = cache_of([L], 64, G, d, 200)
    c.append(randn(L, G, d, seed=1), randn(L, G, 200, seed=2), ints([0, L]), ints([0]), table, max_new=L)
    c.attend(randn(n, H, d, seed=3).to(torch.bfloat16), ints([0, n]), ints([L - n]), table, max_new=n, max_len=L)
    (need,) = c._need.values()
    shares = need // (n * H * (200 + 4) * 4) if need else 1
    assert shares * 80 <= sms


def test_numbers_that_their_types_do_not_hold_are_refused():
    c, table = cache_of([64], 32, 2, 64, 64)
    q, k, start, pos0 = randn(1, 4, 64), randn(1, 2, 64), ints([0, 1]), ints([63])
    for bad in (dict(window=2 ** 31), dict(first=2 ** 40), dict(max_len=2 ** 31), dict(max_new=2 ** 31), dict(scale=1e39), dict(softcap=1e39), dict(window=3.5)):
        with pytest.raises(ValueError, match="range"):
            c.attend(q, start, pos0, table, **{"max_new": 1, "max_len": 64, **bad})
    for bad in (dict(max_new=2 ** 31), dict(rot_mult=1e39, freq=torch.ones(4, device="cuda"))):
        with pytest.raises(ValueError, match="range"):
            c.append(k, k, start, pos0, table, **{"max_new": 1, **bad})
