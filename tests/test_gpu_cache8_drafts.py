"""Drafting and forking on the 8-bit key/value cache: trees, rotary positions of several axes, attention along paths, rows and pages that move, all of them as
they are used together, and what they refuse."""
from __future__ import annotations

import math

import pytest
import torch

from cache8_util import BLOCK, HALF_STEP, attention, ints, quantised, starts, tolerance
from drafts_util import kept, layout, parents_of, paths_of, tree_attention
from test_gpu_cache8 import OPTIONS, cache_of, check_attention, fill, gen, held, options_of, randn

pytestmark = pytest.mark.gpu

SHAPES = ["chain", "roots", "fan", "comb", "random"]


def tree_of(c, parents, pos0):
    """The tree of sequences' parents (lists), and its arrays on the device."""
    counts = [len(p) for p in parents]
    return c.draft_tree(ints(sum(parents, [])), ints(starts(counts)), ints(pos0), max_new=max(counts))


# ---------------------------------------------------------------------------------------------- trees

@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("counts", [[1], [25], [31, 0, 32, 33], [64] * 5, [100, 1, 257], [1025, 7], [4096]])
def test_trees(shape, counts):
    c, _ = cache_of([16], 16, 1, 16, 16, garbage=False)
    parents = [parents_of(shape, n, s) for s, n in enumerate(counts)]
    pos0 = [1000 * s + s for s in range(len(counts))]
    tree = tree_of(c, parents, pos0)
    words = (max(counts) + 31) // 32
    assert tree.sees.shape == (sum(counts), words)
    at = 0
    for p, first in zip(parents, pos0):
        depth, bits = layout(p, words)
        assert torch.equal(tree.positions[at:at + len(p)].cpu(), (first + depth).int()) and torch.equal(tree.sees[at:at + len(p)].cpu(), bits)
        at += len(p)
    c.check_device_errors()


def test_parents_that_cannot_be_are_reported_and_count_as_none():
    from smoltts_b200._errors import SmolError

    for bad in (3, 4, 100, -2, 2 ** 31 - 1, -2 ** 31):
        c, _ = cache_of([16], 16, 1, 16, 16, garbage=False)
        tree = tree_of(c, [[-1, 0, 1, bad, 3]], [10])
        depth, bits = layout([-1, 0, 1, -1, 3], 1)
        assert torch.equal(tree.positions.cpu(), (10 + depth).int()) and torch.equal(tree.sees.cpu(), bits)
        with pytest.raises(SmolError, match="word 2"):
            c.check_device_errors()


def test_sequences_that_do_not_fit_are_left_out():
    """More rows than max_new, positions below 0 or beyond the last, starts that go back: reported, the others laid out."""
    from smoltts_b200._errors import SmolError

    most = 2 ** 31 - 1
    for start, pos0 in (([0, 2, 7, 8], [1, 2, 3]), ([0, 2, 4, 6], [1, -1, 3]), ([0, 2, 4, 6], [1, most - 128, 3]), ([0, 2, 1, 3], [1, 2, 3]), ([0, 2, 90, 91], [1, 2, 3])):
        c, _ = cache_of([16], 16, 1, 16, 16, garbage=False)
        tree = c.draft_tree(ints([-1, 0] * 4), ints(start), ints(pos0), max_new=4)
        alone = min(2, start[2])      # rows of the first sequence that no other claims
        assert tree.positions[:alone].tolist() == [1, 2][:alone] and tree.sees[:alone, 0].tolist() == [1, 3][:alone]
        with pytest.raises(SmolError, match="word 2"):
            c.check_device_errors()


def test_trees_of_other_arrays_are_refused():
    c, _ = cache_of([16], 16, 1, 16, 16, garbage=False)
    p, start, pos0 = ints([-1, 0]), ints([0, 2]), ints([5])
    for args in ((p.long(), start, pos0), (p.cpu(), start, pos0), (p.view(1, 2), start, pos0), (p, start[:1], pos0), (p, start, pos0.float()), (p[:0], start, pos0), (p, start, pos0[:0]),
                 (ints([-1, 9, 0, 9])[::2], start, pos0)):
        with pytest.raises(ValueError):
            c.draft_tree(*args, max_new=2)
    for most in (0, -1, 4097):
        with pytest.raises(ValueError):
            c.draft_tree(p, start, pos0, max_new=most)


# ---------------------------------------------------------------------------------------------- append at positions of their own

def turned(x, positions, axis, freq, half, mult=1.0):
    """x [rows, heads, d] in 64 bits, pair i by positions[axis[i]] * freq[i]."""
    y, n = x.double().clone(), freq.numel()
    for i in range(n):
        a, b = (i, i + n) if half else (2 * i, 2 * i + 1)
        t = (positions[int(axis[i])].double() * freq[i].double().item()).view(-1, 1)
        y[:, :, a] = mult * (x[:, :, a].double() * t.cos() - x[:, :, b].double() * t.sin())
        y[:, :, b] = mult * (x[:, :, b].double() * t.cos() + x[:, :, a].double() * t.sin())
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,pairs,half,axes,mult", [(64, 32, True, 1, 1.0), (128, 64, True, 3, 1.0), (128, 64, False, 3, 1.25), (96, 16, True, 2, 1.0), (33, 5, True, 3, 1.0), (33, 5, False, 4, 1.0), (256, 128, True, 4, 1.0)])
def test_rotation_by_positions_of_several_axes(dtype, d, pairs, half, axes, mult):
    """Rows lie where they lie; they are turned by what is given, anywhere from -2^31 to 2^31 - 1.  Tolerances as where positions are places: 2^-22 of both terms, then half a step."""
    lens, pos0, H = [5, 37], [0, 21], 6
    c, table = cache_of([5, 21 + 37], 64, 2, d, 16, garbage=False)
    freq = (10000.0 ** (-torch.arange(pairs, device="cuda") / pairs)).float()
    T = sum(lens)
    positions = torch.randint(0, 5000, (axes, T), generator=gen(9), device="cuda").int()
    positions[0, :4] = ints([2 ** 31 - 1, -2 ** 31, -7, 0])
    axis = torch.randint(0, axes, (pairs,), generator=gen(10), device="cuda").int()
    k, v, q = randn(T, 2, d, seed=1).to(dtype), randn(T, 2, 16, seed=2).to(dtype), randn(T, H, d, seed=3).to(dtype)
    got = c.append(k, v, ints(starts(lens)), ints(pos0), table, max_new=37, q=q, freq=freq, rot_half=half, rot_mult=mult, positions=positions, axis=axis)
    size, at = 2.0 * mult * 2.0 ** -22, starts(lens)
    want = turned(q, positions, axis, freq, half, mult)
    err = (got.double() - want).abs()
    assert (err <= HALF_STEP[dtype] * want.abs() * 1.01 + size * q.abs().max().item()).all(), err.max()
    want = turned(k, positions, axis, freq, half, mult)
    for s, n in enumerate(lens):
        k8, v8 = held(c, table, s, pos0[s] + n)
        place = torch.arange(pos0[s], pos0[s] + n, device="cuda")
        scale = c.k_scale[table[s].clamp(min=0).long()].transpose(1, 2).reshape(-1, 2)[place // BLOCK].double().unsqueeze(-1)
        err = (k8[pos0[s]:].double() - want[at[s]:at[s] + n]).abs()
        assert (err <= 2.0 ** -4 * want[at[s]:at[s] + n].abs() * 1.01 + 2.0 ** -10 * scale + size * k.abs().max().item()).all(), err.max()
        assert pos0[s] or torch.equal(v8.double(), quantised(v[at[s]:at[s] + n])[0])
    c.check_device_errors()


def test_positions_that_are_the_places_change_nothing():
    """To the bit, whether one axis or three that agree, with a map of axes or without."""
    lens, pos0, H, G, d = [5, 37], [3, 21], 4, 2, 64
    freq = (10000.0 ** (-torch.arange(32, device="cuda") / 32)).float()
    T = sum(lens)
    k, v, q = randn(T, G, d, seed=1), randn(T, G, d, seed=2), randn(T, H, d, seed=3)
    places = ints([p + i for p, n in zip(pos0, lens) for i in range(n)])
    results = []
    for more in (dict(), dict(positions=places), dict(positions=places.repeat(3, 1).contiguous(), axis=torch.randint(0, 3, (32,), device="cuda").int()), dict(positions=places.view(1, T))):
        c, table = cache_of([p + n for p, n in zip(pos0, lens)], 32, G, d, d, garbage=False)
        out = c.append(k, v, ints(starts(lens)), ints(pos0), table, max_new=37, q=q, freq=freq, **more)
        results.append((out, c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale))
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))


def test_an_axis_that_there_is_not_is_reported_and_counts_as_the_first():
    from smoltts_b200._errors import SmolError

    for bad in (3, -1, 2 ** 31 - 1):
        outs = []
        for a in (bad, 0):
            c, table = cache_of([6], 16, 1, 16, 16, garbage=False)
            positions = torch.arange(18, device="cuda").int().view(3, 6)
            outs.append(c.append(randn(6, 1, 16), randn(6, 1, 16), ints([0, 6]), ints([0]), table, max_new=6, q=randn(6, 2, 16), freq=torch.ones(4, device="cuda"), positions=positions, axis=ints([0, 1, a, 2])))
            if a == bad:
                with pytest.raises(SmolError, match="word 2"):
                    c.check_device_errors()
        assert torch.equal(*outs)


def test_positions_that_do_not_fit_are_refused():
    c, table = cache_of([6], 16, 1, 16, 16, garbage=False)
    x, f, p = randn(6, 1, 16), torch.ones(4, device="cuda"), torch.zeros(3, 6, device="cuda").int()
    for more in (dict(positions=p[0]), dict(freq=f, axis=ints([0] * 4)), dict(freq=f, positions=p.long()), dict(freq=f, positions=p[:, :5].contiguous()), dict(freq=f, positions=p.T), dict(freq=f, positions=p[:0]),
                 dict(freq=f, positions=p, axis=ints([0] * 3)), dict(freq=f, positions=p, axis=torch.zeros(4, device="cuda")), dict(freq=f, positions=p.cpu()), dict(freq=f, positions=p.view(3, 6, 1))):
        with pytest.raises(ValueError):
            c.append(x, x, ints([0, 6]), ints([0]), table, max_new=6, **more)


# ---------------------------------------------------------------------------------------------- attention along paths

def check_tree(c, table, q, counts, pos0, tree, out, at=0, **options):
    first = starts(counts)
    kv_len = options.pop("kv_len", None)
    for s, n in enumerate(counts):
        if n == 0:
            continue
        rows = slice(at + first[s], at + first[s] + n)
        k, v = held(c, table, s, pos0[s] + n)
        want, spread, size = tree_attention(q[rows], k, v, pos0[s], tree.positions[rows].clamp(0, 2 ** 31 - 129), tree.sees[rows], options.get("scale", c.dim ** -0.5), kv_len=None if kv_len is None else kv_len[s],
                                            **{x: options[x] for x in ("window", "first", "softcap", "sink", "slope", "penalty") if x in options})
        far = max(pos0[s] + n, int(tree.positions[rows].max()))
        bent = options.get("softcap", 0.0) + (options["slope"].max().item() * far if options.get("slope") is not None else 0.0)
        if options.get("penalty") is not None:
            bent += options["penalty"][0].abs().max().item() * math.log1p(options["penalty"][1].max().item() * far)
        off = (out[rows].double() - want).abs() - tolerance(q.dtype, want, spread, size, bent)
        assert off.max().item() <= 0, (s, off.max().item(), (off > 0).float().mean().item())


ROWS = [
    # heads, kv_heads, d, dv, page, counts, pos0: few rows, many, both
    (12, 4, 64, 64, 64, [1], [0]),
    (12, 4, 64, 64, 64, [1, 4, 2, 5], [2047, 15, 16, 700]),
    (8, 8, 128, 128, 16, [3, 7], [63, 4000]),
    (3, 1, 80, 72, 48, [3, 1], [50, 333]),
    (40, 2, 33, 7, 16, [1, 2], [1, 70]),
    (4, 2, 256, 200, 64, [1, 3], [129, 20]),
    (1, 1, 64, 64, 128, [9], [20000]),
    (4, 4, 64, 64, 64, [64], [0]),
    (8, 2, 128, 128, 64, [64, 31, 100], [500, 0, 127]),
    (12, 4, 64, 64, 16, [33, 129], [128, 77]),
    (4, 2, 33, 7, 16, [65, 66], [1, 250]),
    (4, 2, 256, 200, 64, [90], [129]),
    (8, 2, 64, 64, 64, [150, 0, 3, 1], [100, 7, 2500, 3000]),
    (2, 1, 128, 64, 32, [520], [300]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,d,dv,page,counts,pos0", ROWS)
def test_attention_along_paths(dtype, H, G, d, dv, page, counts, pos0):
    lens = [p + n for p, n in zip(pos0, counts)]
    c, table = cache_of(lens, page, G, d, dv, seed=H)
    fill(c, table, lens, seed=H)
    q = randn(sum(counts), H, d, seed=4).to(dtype)
    for shape in ("random", "fan", "chain"):
        tree = tree_of(c, [parents_of(shape, n, s) for s, n in enumerate(counts)], pos0)
        out = c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=max(counts), max_len=max(lens), tree=tree)
        check_tree(c, table, q, counts, pos0, tree, out)
    # a chain is the ordinary thing
    plain = c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=max(counts), max_len=max(lens))
    assert (plain.double() - out.double()).abs().max() <= 4 * HALF_STEP[dtype] * plain.abs().max() if dtype == torch.bfloat16 else torch.allclose(plain, out, rtol=1e-4, atol=1e-5)
    c.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", list(OPTIONS))
@pytest.mark.parametrize("counts,pos0", [([3, 1, 5], [200, 36, 1]), ([40, 3], [150, 90]), ([70], [0])])
def test_masks_and_scores_of_trees(dtype, name, counts, pos0):
    H, G, d = 6, 2, 64
    lens = [p + n for p, n in zip(pos0, counts)]
    c, table = cache_of(lens, 32, G, d, d, seed=2)
    fill(c, table, lens, seed=2)
    q = randn(sum(counts), H, d, seed=4).to(dtype)
    o = options_of(name, H)
    tree = tree_of(c, [parents_of("random", n, s) for s, n in enumerate(counts)], pos0)
    out = c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=max(counts), max_len=max(lens), tree=tree, **o)
    check_tree(c, table, q, counts, pos0, tree, out, **o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [3, 17, 45])
def test_any_mask_and_any_positions(dtype, n):
    """Bits at random (rows that see later ones, that do not see themselves, that see none), positions that agree, go back, lie far away or outside their range, with and
    without options; words for fewer rows than there are."""
    from smoltts_b200.kv_cache import DraftTree

    H, G, d, counts, pos0 = 4, 2, 64, [n, n, n], [0, 100, 333]
    lens = [p + n for p in pos0]
    c, table = cache_of(lens, 32, G, d, d, seed=7)
    fill(c, table, lens, seed=7)
    q = randn(3 * n, H, d, seed=4).to(dtype)
    places = [p + i for p in pos0 for i in range(n)]
    near = torch.tensor(places, device="cuda") + torch.randint(-30, 31, (3 * n,), generator=gen(3), device="cuda")
    odd = near.clone()
    odd[::3] = ints([2 ** 31 - 1, -5, 2 ** 31 - 129, 10 ** 6, 0] * 20)[:odd[::3].numel()]
    slope = torch.full((H,), 0.01, device="cuda")
    for words in ((n + 31) // 32, (n + 31) // 32 + 2, 1):
        sees = torch.randint(-2 ** 31, 2 ** 31, (3 * n, words), generator=gen(words), device="cuda").int()
        sees[1] = sees[n + 1] = 0
        for positions, options in ((near, (dict(), dict(window=25), dict(window=25, first=3), dict(slope=slope), dict(sink=slope))), (odd, (dict(), dict(window=40), dict(window=40, first=60), dict(window=1)))):
            tree = DraftTree(positions.int(), sees)
            for o in options:
                out = c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=n, max_len=max(lens), tree=tree, **o)
                check_tree(c, table, q, counts, pos0, tree, out, **o)
                assert (out[1] == 0).all()      # no context, no bits
    c.check_device_errors()


@pytest.mark.parametrize("n", [1, 12, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_hidden_keys_and_rows_of_nobody(n, dtype):
    """kv_len counts places; rows in front of, behind and between the sequences stay as they were; queries and results are slices."""
    H, G, d = 4, 2, 128
    pos0, counts, kv_len = [100, 5, 50, 300], [n, 0, n, n], [0, 9, 20, 300 + n // 2]
    lens = [p + m for p, m in zip(pos0, counts)]
    c, table = cache_of(lens, 64, G, d, d)
    fill(c, table, lens)
    start = [s + 2 for s in starts(counts)]
    wide = randn(3 * n + 5, H, d + 8, seed=4).to(dtype)
    q = wide[..., 8:]
    parents = [-9, 77] + sum([parents_of("fan", m) for m in counts], []) + [5, 5, 5]
    tree = c.draft_tree(ints(parents), ints(start), ints(pos0), max_new=n)
    c.check_device_errors()
    for o in (dict(), dict(sink=torch.ones(H, device="cuda")), dict(window=10), dict(window=10, first=3)):
        out = torch.full((3 * n + 5, H, d + 3), 7.0, device="cuda", dtype=dtype)
        c.attend(q, ints(start), ints(pos0), table, max_new=n, max_len=max(lens), kv_len=ints(kv_len), tree=tree, out=out[..., :d], **o)
        assert (out[2:2 + n, :, :d] == 0).all() and (out[:2] == 7).all() and (out[2 + 3 * n:] == 7).all() and (out[..., d:] == 7).all()
        check_tree(c, table, q, counts, pos0, tree, out[..., :d], at=2, kv_len=kv_len, **o)


@pytest.mark.parametrize("n", [4, 24, 90])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_on_one_branch_is_not_seen_on_another(n, dtype):
    H, G, d, L = 4, 2, 64, 200
    c, table = cache_of([L + n], 32, G, d, d)
    k, v = randn(L + n, G, d, seed=1), randn(L + n, G, d, seed=2)
    k[L + 1, 0, 3], v[L + 2, 1, 9], v[70, 1, 5] = math.nan, math.nan, math.nan
    c.append(k, v, ints([0, L + n]), ints([0]), table, max_new=L + n)
    q = randn(n, H, d, seed=3).to(dtype)
    parents = parents_of("fan", n)
    ways = paths_of(parents)
    tree = tree_of(c, [parents], [L])
    for window in (0, 60):
        out = c.attend(q, ints([0, n]), ints([L]), table, max_new=n, max_len=L + n, window=window, tree=tree)
        want = torch.zeros(n, H, d, dtype=torch.bool, device="cuda")
        for i, way in enumerate(ways):
            want[i, :2] |= 1 in way
            want[i, 2:, 9] |= 2 in way
            want[i, 2:, 5] |= not window
        assert torch.equal(torch.isnan(out), want) and torch.isfinite(out[~want]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_trees_of_few_and_many_rows_in_one_batch(dtype):
    """Long contexts, so that sequences of few rows go their own way; rows behind max_new are left alone, and seen all the same."""
    H, G, d, counts, pos0 = 8, 2, 64, [1, 150, 0, 3, 9, 1], [5000, 100, 7, 2500, 3000, 0]
    lens = [p + n for p, n in zip(pos0, counts)]
    c, table = cache_of(lens, 64, G, d, d, seed=1)
    fill(c, table, lens, seed=1)
    q = randn(sum(counts) + 2, H, d, seed=4).to(dtype)
    parents = sum([parents_of("random", n, s) for s, n in enumerate(counts)], []) + [-1, -1]
    tree = c.draft_tree(ints(parents), ints(starts(counts)), ints(pos0), max_new=150)
    for o in (dict(), dict(window=700, first=5)):
        out = torch.full((sum(counts) + 2, H, d), 7.0, device="cuda", dtype=dtype)
        c.attend(q, ints(starts(counts)), ints(pos0), table, max_new=150, max_len=max(lens), out=out, tree=tree, **o)
        check_tree(c, table, q, counts, pos0, tree, out, **o)
        assert (out[sum(counts):] == 7).all()


def test_rows_behind_max_new_are_left_alone_and_seen():
    from smoltts_b200.kv_cache import DraftTree

    H, G, d = 4, 2, 64
    c, table = cache_of([300], 64, G, d, d)
    fill(c, table, [300])
    q = randn(20, H, d, seed=3)
    tree = DraftTree(ints([280] * 20), ints([[2 ** 20 - 1]] * 20))
    out = torch.full((20, H, d), 7.0, device="cuda")
    c.attend(q, ints([0, 20]), ints([280]), table, max_new=3, max_len=300, out=out, tree=tree)
    k, v = held(c, table, 0, 300)
    want, spread, size = tree_attention(q[:3], k, v, 280, tree.positions, tree.sees[:3], d ** -0.5)
    assert ((out[:3].double() - want).abs() <= tolerance(q.dtype, want, spread, size)).all() and (out[3:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("most", [2, 9, 30, 40])
def test_host_numbers_that_are_too_small(dtype, most):
    """max_len sizes the grid and nothing else; rows beyond max_new are left as they were, and seen by the others where bits name them."""
    H, G, d, n, L = 4, 2, 64, 45, 3000
    c, table = cache_of([L, 100 + n], 64, G, d, d)
    fill(c, table, [L, 100 + n])
    q = randn(2 * n, H, d, seed=3).to(dtype)
    pos0 = [L - n, 100]
    tree = tree_of(c, [parents_of("fan", n), [-1] * n], pos0)
    tree.sees[:, 1] |= 1 << 12      # everybody sees row 44
    out = torch.full((2 * n, H, d), 7.0, device="cuda", dtype=dtype)
    c.attend(q, ints([0, n, 2 * n]), ints(pos0), table, max_new=most, max_len=10, out=out, tree=tree)
    for s, p in enumerate(pos0):
        k, v = held(c, table, s, p + n)
        rows = slice(s * n, s * n + most)
        want, spread, size = tree_attention(q[rows], k, v, p, tree.positions[s * n:(s + 1) * n], tree.sees[rows], d ** -0.5)
        assert ((out[rows].double() - want).abs() <= tolerance(dtype, want, spread, size)).all()
        assert (out[s * n + most:(s + 1) * n] == 7).all()
    c.check_device_errors()


def test_pages_whose_bytes_pass_32_bits():
    """The same step in a pool of a few pages and at the end of one of 4.6 GB of keys: equal to the bit."""
    from smoltts_b200.kv_cache import KVCache8, copy_pages, keep_rows

    G, H, d, page, n, far = 8, 16, 128, 64, 20, 70000
    small, big = KVCache8.allocate(12, page, G, d), KVCache8.allocate(far, page, G, d)
    assert big.k.numel() > 2 ** 32
    freq = (10000.0 ** (-torch.arange(64, device="cuda") / 64)).float()
    got = []
    for c, base in ((small, 0), (big, far - 12)):
        table = ints([[base + p for p in (5, 2, 9)], [base + p for p in (7, 0, 11)]])
        k, v = randn(300, G, d, seed=1).to(torch.bfloat16), randn(300, G, d, seed=2).to(torch.bfloat16)
        c.append(k, v, ints([0, 150, 300]), ints([0, 0]), table, max_new=150)
        results = []
        for dtype, m in ((torch.bfloat16, 2), (torch.bfloat16, n), (torch.bfloat16, 40), (torch.float32, 4)):
            tree = c.draft_tree(ints(parents_of("fan", m) * 2), ints([0, m, 2 * m]), ints([140, 130]), max_new=m)
            q = c.append(randn(2 * m, G, d, seed=3).to(dtype), randn(2 * m, G, d, seed=4).to(dtype), ints([0, m, 2 * m]), ints([140, 130]), table, max_new=m, q=randn(2 * m, H, d, seed=5).to(dtype), freq=freq,
                         positions=tree.positions)
            results.append(c.attend(q, ints([0, m, 2 * m]), ints([140, 130]), table, max_new=m, max_len=180, tree=tree))
        keep_rows(c, ints([140, 130]), table, ints([[0, 3, 17], [1, 2, 30]]), ints([3, 3]))
        copy_pages(c, [base + 9, base + 11], [base + 1, base + 3])
        c.check_device_errors()
        at = torch.arange(base, base + 12, device="cuda")
        got.append([*results, *(x.view(torch.uint8)[at] for x in (c.k, c.v)), *(x[at] for x in (c.k_scale, c.v_scale))])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and (big.k.view(torch.uint8)[:far - 12].amax() == 0)


def test_trees_that_do_not_fit_are_refused():
    from smoltts_b200._errors import SmolError
    from smoltts_b200.kv_cache import DraftTree

    c, table = cache_of([40], 16, 1, 16, 16)
    fill(c, table, [40])
    q, pos, sees = randn(6, 2, 16), ints([34] * 6), ints([[1]] * 6)
    for tree in (DraftTree(pos[:5], sees), DraftTree(pos, sees[:5]), DraftTree(pos, sees[:, 0]), DraftTree(pos, sees[:, :0]), DraftTree(pos.long(), sees), DraftTree(pos, sees.cpu()), DraftTree(pos.view(6, 1), sees),
                 DraftTree(pos, ints([[1, 2]] * 6)[:, ::2])):
        with pytest.raises(ValueError):
            c.attend(q, ints([0, 6]), ints([34]), table, max_new=6, max_len=40, tree=tree)
    room = torch.zeros(6 * 2 * 16 + 12, device="cuda")
    with pytest.raises(ValueError):      # a result over the tree's arrays
        c.attend(q, ints([0, 6]), ints([34]), table, max_new=6, max_len=40, tree=DraftTree(room[180:186].view(torch.int32), sees), out=room[:192].view(6, 2, 16))
    out = torch.full((6, 2, 16), 7.0, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):      # a sequence that begins in front of its first position
        res = out.to(dtype)
        c.attend(q.to(dtype), ints([0, 6]), ints([-1]), table, max_new=6, max_len=40, tree=DraftTree(pos, sees), out=res)
        with pytest.raises(SmolError, match="word 2"):
            c.check_device_errors()
        c._err.zero_()


@pytest.mark.parametrize("n,context", [(2, 100), (3, 5000), (9, 40), (9, 900), (20, 5000), (40, 100)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gates_and_factors_of_results(dtype, n, context):
    """What the C entry takes beyond the class: results times out_scale and sigmoid(gate), whoever writes them (one block, a cluster, the kernel that joins shares)."""
    import ctypes as C

    from smoltts_b200 import _capi_lm as cl

    H, G, d = 4, 2, 72
    c, table = cache_of([context + n], 32, G, d, d)
    fill(c, table, [context + n])
    q, gate = randn(n, H, d, seed=3).to(dtype), randn(n, H * d + 5, seed=4)
    tree = tree_of(c, [parents_of("fan", n)], [context])
    want = c.attend(q, ints([0, n]), ints([context]), table, max_new=n, max_len=context + n, tree=tree).double() * 0.5 * torch.sigmoid(gate[:, :H * d].double()).view(n, H, d)
    out = torch.full((n, H, d), 7.0, device="cuda", dtype=dtype)
    start, pos0 = ints([0, n]), ints([context])
    cache = cl.SmolLmCache8(k=c.k.data_ptr(), v=c.v.data_ptr(), k_scale=c.k_scale.data_ptr(), v_scale=c.v_scale.data_ptr(), n_pages=c.n_pages, page_size=32, kv_heads=G, dim=d, vdim=d, err=c._err.data_ptr())
    batch = cl.SmolLmCache8Batch(n_tokens=n, n_seqs=1, max_pages=table.shape[1], max_new=n, max_len=context + n, seq_start=start.data_ptr(), seq_pos0=pos0.data_ptr(), block_table=table.data_ptr())
    a = cl.SmolLmCache8Attend(dtype=0 if dtype == torch.bfloat16 else 1, heads=H, q=q.data_ptr(), out=out.data_ptr(), q_row=H * d, q_head=d, out_row=H * d, out_head=d, scale=d ** -0.5, out_scale=0.5,
                              gate=gate.data_ptr(), gate_row=H * d + 5, tree_positions=tree.positions.data_ptr(), tree_sees=tree.sees.data_ptr(), tree_words=tree.sees.shape[1])
    lib, need = cl.load(), C.c_size_t()
    cl.check(lib.smol_lm_cache8_workspace_bytes(C.byref(cache), C.byref(batch), C.byref(a), C.byref(need)))
    work = torch.empty(max(need.value, 16), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    cl.check(lib.smol_lm_cache8_attend(C.byref(cache), C.byref(batch), C.byref(a), work.data_ptr(), need.value, stream))
    # the result without a gate is rounded once, that with one after the product: half a step each, and four roundings of fp32 between
    assert ((out.double() - want).abs() <= 2.01 * HALF_STEP[dtype] * want.abs() + 2.0 ** -21 * want.abs() + 1e-30).all()
    c.check_device_errors()


# ---------------------------------------------------------------------------------------------- rows that are kept

def check_kept(c, before, table, pos0, rows):
    """Every sequence against the definition, and everything else as it was."""
    old_k, old_v, old_ks, old_vs = before
    per = c.page_size // BLOCK
    for old, old_scale, codes, scale, width in ((old_k, old_ks, c.k, c.k_scale, c.dim), (old_v, old_vs, c.v, c.v_scale, c.vdim)):
        free = torch.ones(c.n_pages, c.page_size, dtype=torch.bool, device="cuda")
        blocks = torch.ones(c.n_pages, per, dtype=torch.bool, device="cuda")
        for s, (p, r) in enumerate(zip(pos0, rows)):
            if not r:
                continue
            pages = table[s][table[s] >= 0].long()
            for g in range(c.kv_heads):
                exps = torch.log2(old_scale[pages, g].abs().double()).round().flatten()
                x = old[pages, g].contiguous().view(torch.float8_e4m3fn).double().reshape(-1, old.shape[3]) * torch.exp2(exps).repeat_interleave(BLOCK).unsqueeze(1)
                want, want_exps = kept(x, int(exps[p // BLOCK]), r, p)
                first, last = p // BLOCK, (p + len(r) - 1) // BLOCK
                got_scale = scale[pages, g].flatten()[first:last + 1]
                assert got_scale.abs().tolist() == [2.0 ** e for e in want_exps]
                got = codes.view(torch.uint8)[pages, g].contiguous().view(torch.float8_e4m3fn).double().reshape(-1, old.shape[3]) * scale[pages, g].abs().double().flatten().repeat_interleave(BLOCK).unsqueeze(1)
                assert torch.equal(got[first * BLOCK:p + len(r)].nan_to_num(1e30), want[first * BLOCK:].nan_to_num(1e30))
                for b in range(first, last + 1):      # the mark of a block that holds a NaN
                    lo, hi = max(b * BLOCK, p), min((b + 1) * BLOCK, p + len(r))
                    marked = bool(torch.isnan(want[lo:hi]).any()) or (b * BLOCK < p and bool(old_scale[pages, g].flatten()[b] < 0))
                    assert bool(got_scale[b - first] < 0) == marked
            for at in range(p // BLOCK * BLOCK, p + len(r)):
                free[pages[at // c.page_size], at % c.page_size] = False
                blocks[pages[at // c.page_size], at % c.page_size // BLOCK] = False
        assert torch.equal(old.transpose(1, 2)[free], codes.view(torch.uint8).transpose(1, 2)[free]) and torch.equal(old_scale.transpose(1, 2)[blocks], scale.transpose(1, 2)[blocks])
        assert (codes.view(torch.uint8)[..., width:] == 0).all()


def contents(c):
    return [x.clone() for x in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale)]


def arrays(rows):
    most = max(1, max(len(r) for r in rows))
    return ints([r + [10 ** 6] * (most - len(r)) for r in rows]), ints([len(r) for r in rows])


def uneven(c, table, lens, seed=0):
    """Rows of very different magnitude, some blocks of zeros, NaNs here and there."""
    T = sum(lens)
    size = torch.exp2(torch.randint(-12, 13, (T, 1, 1), generator=gen(seed + 3), device="cuda").float())
    k, v = randn(T, c.kv_heads, c.dim, seed=seed) * size, randn(T, c.kv_heads, c.vdim, seed=seed + 1) * size.flip(0)
    k[40:60] = 0
    v[5, 0, 0] = k[T // 2, -1, -1] = k[T - 1, 0, 0] = math.nan
    c.append(k, v, ints(starts(lens)), ints([0] * len(lens)), table, max_new=max(lens))


@pytest.mark.parametrize("G,d,dv,page", [(2, 64, 64, 16), (4, 128, 128, 64), (1, 16, 48, 32), (3, 80, 72, 48), (2, 33, 7, 16), (1, 256, 200, 16), (2, 1, 3, 32)])
def test_rows_are_kept_as_an_append_would_write_them(G, d, dv, page):
    lens = [30, 100, 16, 17, 64, 5, 150, 33]
    pos0 = [7, 50, 0, 16, 31, 4, 0, 15]
    rows = [[0, 1, 5], [1, 3, 20, 21, 22, 49], [15], [0], [], [0], sorted({*range(0, 120, 3), 119, 149}), list(range(17))]
    cs = [cache_of(lens, page, G, d, dv, seed=i)[0] for i in range(3)]
    table = cache_of(lens, page, G, d, dv, seed=0)[1]
    for i, c in enumerate(cs):
        uneven(c, table, lens, seed=10 * i)
    from smoltts_b200.kv_cache import keep_rows

    before = [contents(c) for c in cs]
    keep_rows(cs, ints(pos0), table, *arrays(rows))
    for c, b in zip(cs, before):
        check_kept(c, b, table, pos0, rows)
        c.check_device_errors()


def test_a_kept_prefix_changes_nothing_in_a_block_begun_before():
    from smoltts_b200.kv_cache import keep_rows

    c, table = cache_of([20], 16, 2, 64, 64)
    uneven(c, table, [20])
    before = contents(c)
    keep_rows(c, ints([3]), table, *arrays([[0, 1, 2, 3, 4]]))
    assert all(torch.equal(a, b) for a, b in zip(before, contents(c)))


def test_more_layers_than_a_launch_takes():
    from smoltts_b200.kv_cache import keep_rows

    made = [cache_of([60], 32, 1, 16, 32, seed=0) for _ in range(70)]
    cs, table = [c for c, _ in made], made[0][1]
    for i, c in enumerate(cs):
        uneven(c, table, [60], seed=i)
    before = [contents(c) for c in cs]
    keep_rows(cs, ints([9]), table, *arrays([[2, 3, 9, 30, 50]]))
    for c, b in zip(cs, before):
        check_kept(c, b, table, [9], [[2, 3, 9, 30, 50]])


def test_rows_that_do_not_fit_are_reported_and_nothing_of_their_sequence_moves():
    from smoltts_b200._errors import SmolError
    from smoltts_b200.kv_cache import keep_rows

    lens, pos0 = [60, 60], [9, 9]
    good = [1, 4, 8, 20]
    for bad, count, p, word in (([4, 4, 8, 20], 4, 9, 2), ([4, 3, 8, 20], 4, 9, 2), ([-1, 4, 8, 20], 4, 9, 2), (good, 5, 9, 2), (good, -1, 9, 2), (good, 4, -1, 2), ([1, 4, 8, 90], 4, 9, 1),
                                ([1, 4, 8, 2 ** 31 - 1], 4, 9, 2), (good, 4, 2 ** 31 - 1, 2), (good, 4, 2 ** 31 - 140, 2), (good, 4, 100, 1)):
        c, table = cache_of(lens, 16, 2, 32, 16)
        uneven(c, table, lens)
        before = contents(c)
        keep_rows(c, ints([p, 9]), table, ints([bad, good]), ints([count, 4]))
        check_kept(c, before, table, pos0, [[], good])
        with pytest.raises(SmolError, match=f"word {word}"):
            c.check_device_errors()
    for at, page in ((0, 10 ** 6), (1, -5)):      # a page that there is not, under a row that goes or comes
        c, table = cache_of(lens, 16, 2, 32, 16)
        uneven(c, table, lens)
        before, wrong = contents(c), table.clone()
        wrong[0, at] = page
        keep_rows(c, ints(pos0), wrong, ints([good, good]), ints([4, 4]))
        check_kept(c, before, table, pos0, [[], good])
        with pytest.raises(SmolError, match="word 1"):
            c.check_device_errors()


def test_kept_rows_of_other_arrays_are_refused():
    from smoltts_b200.kv_cache import KVCache8, keep_rows

    c, table = cache_of([40], 16, 2, 32, 16)
    rows, counts, p = ints([[0, 1]]), ints([2]), ints([5])
    other = KVCache8.allocate(c.n_pages, 32, 2, 32, 16)
    for caches, args in (([c, c], (p, table, rows, counts)), ([c, other], (p, table, rows, counts)), ([], (p, table, rows, counts)), (c, (p, table, rows[0], counts)), (c, (p, table[0], rows, counts)),
                         (c, (p, table, rows[:, :0], counts)), (c, (p.long(), table, rows, counts)), (c, (p, table, rows, counts.cpu())), (c, (p, table, rows, ints([2, 2]))), (c, (ints([5, 5]), table, rows, counts)),
                         (c, (p, table, ints([[0, 9, 1, 9]])[:, ::2], counts))):
        with pytest.raises(ValueError):
            keep_rows(caches, *args)


# ---------------------------------------------------------------------------------------------- pages

@pytest.mark.parametrize("G,d,dv,page", [(1, 16, 16, 16), (2, 33, 7, 16), (4, 128, 128, 64), (3, 80, 72, 48), (8, 256, 200, 128)])
@pytest.mark.parametrize("layers,pairs", [(1, 1), (3, 5), (2, 700), (40, 2)])
def test_pages_are_copied(G, d, dv, page, layers, pairs):
    from smoltts_b200.kv_cache import copy_pages

    if pairs * layers * G * page * (d + dv) > 1 << 29:
        pairs = 30
    n = 2 * pairs + 1
    cs = [cache_of([n * page], page, G, d, dv, seed=i)[0] for i in range(layers)]
    order = torch.randperm(n, generator=torch.Generator().manual_seed(pairs)).tolist()
    src, dst = order[:pairs], order[pairs:2 * pairs]
    src[-1] = src[0]
    before = [contents(c) for c in cs]
    copy_pages(cs if layers > 1 else cs[0], src, dst)
    for c, b in zip(cs, before):
        for x, y in zip(b, contents(c)):
            x[dst] = x[src]
            assert torch.equal(x, y)


def test_pages_that_cannot_be_copied_are_refused():
    from smoltts_b200.kv_cache import KVCache8, copy_pages

    c, _ = cache_of([100], 16, 1, 16, 16)
    other = KVCache8.allocate(c.n_pages, 16, 1, 32, 16)
    before = contents(c)
    for caches, src, dst in ((c, [0], [c.n_pages]), (c, [-1], [0]), (c, [0, 1], [2, 2]), (c, [0, 1], [1, 2]), (c, [3], [3]), (c, [0, 1], [2]), (c, [2 ** 31], [0]), ([c, c], [0], [1]), ([c, other], [0], [1]), ([], [0], [1]),
                             (c, list(range(3)) * 20, [4] * 60)):
        with pytest.raises(ValueError):
            copy_pages(caches, src, dst)
    for src in ([0.5], torch.zeros(1, device="cuda").int(), ["0"]):
        with pytest.raises((ValueError, TypeError)):
            copy_pages(c, src, [1])
    copy_pages(c, [], [])
    assert all(torch.equal(a, b) for a, b in zip(before, contents(c)))
    copy_pages(c, torch.tensor([0]), torch.tensor([1]))
    assert torch.equal(c.k.view(torch.uint8)[1], before[0][0])


# ---------------------------------------------------------------------------------------------- as they are used

def layers_of(n, lens, page, G, d):
    made = [cache_of(lens, page, G, d, d, seed=i) for i in range(n)]
    return [c for c, _ in made], cache_of(lens, page, G, d, d, seed=0)[1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [7, 40])
def test_draft_verify_keep_and_fork(dtype, n):
    """Two layers, three sequences: prompts, a drafted tree at its depths' positions, a path kept, a fork that goes on by itself, a token of all of them.  Every attention against
    the cache's own contents; kept rows give what their path gave in the tree; the fork's pages are its own."""
    from smoltts_b200.kv_cache import copy_pages, keep_rows

    H, G, d, page = 8, 2, 64, 32
    pos0, counts = [50, 31, 130], [n, n - 2, n]
    lens = [p + m + 40 for p, m in zip(pos0, counts)]
    caches, table = layers_of(2, lens + [130 + n + 40], page, G, d)
    freq = (10000.0 ** (-torch.arange(d // 2, device="cuda") / (d // 2))).float()
    for i, c in enumerate(caches):
        T = sum(pos0)
        c.append(randn(T, G, d, seed=i).to(dtype), randn(T, G, d, seed=i + 9).to(dtype), ints(starts(pos0)), ints([0] * 3), table[:3].contiguous(), max_new=130, freq=freq)
    parents = [parents_of("random", m, s) for s, m in enumerate(counts)]
    tree = caches[0].draft_tree(ints(sum(parents, [])), ints(starts(counts)), ints(pos0), max_new=n)
    T, at = sum(counts), starts(counts)
    drafted = []
    for i, c in enumerate(caches):
        q, k, v = randn(T, H, d, seed=i + 20).to(dtype), randn(T, G, d, seed=i + 30).to(dtype), randn(T, G, d, seed=i + 40).to(dtype)
        q = c.append(k, v, ints(at), ints(pos0), table[:3].contiguous(), max_new=n, q=q, freq=freq, positions=tree.positions)
        out = c.attend(q, ints(at), ints(pos0), table[:3].contiguous(), max_new=n, max_len=max(lens), tree=tree)
        check_tree(c, table, q, counts, pos0, tree, out)
        drafted.append((q, out))
    rows = [sorted(paths_of(p)[-1]) for p in parents]      # the way to the last row
    keep_rows(caches, ints(pos0), table[:3].contiguous(), *arrays(rows))
    m = [len(r) for r in rows]
    for c, (q, out) in zip(caches, drafted):      # the path's rows again, as ordinary ones
        mine = torch.cat([torch.tensor([at[s] + r for r in rows[s]]) for s in range(3)]).cuda()
        again = c.attend(q[mine], ints(starts(m)), ints(pos0), table[:3].contiguous(), max_new=max(m), max_len=max(lens))
        k, v = zip(*(held(c, table, s, pos0[s] + m[s]) for s in range(3)))
        # two results of the same values, each within 2^-8 of itself and 2^-9 of its weights; codes below the smallest normal one may have lost their last bit on the way, 2^-17 of a block
        assert (again.double() - out[mine].double()).abs().max() <= 0.02 * out.abs().max()
        first = starts(m)
        for s in range(3):
            want, spread, size = attention(q[mine[first[s]:first[s + 1]]], k[s], v[s], torch.arange(pos0[s], pos0[s] + m[s], device="cuda"), d ** -0.5)
            assert ((again[first[s]:first[s + 1]].double() - want).abs() <= tolerance(dtype, want, spread, size)).all()
    # the last sequence is forked: whole pages are shared, the one that goes on filling is copied
    length = pos0[2] + m[2]
    whole = length // page
    fork = torch.cat([table[2, :whole], table[3, whole:]])
    table[3] = fork
    if length % page:
        copy_pages(caches, [int(table[2, whole])], [int(table[3, whole])])
    pos = [p + x for p, x in zip(pos0, m)] + [length]
    for i, c in enumerate(caches):
        before = held(c, table, 2, length)
        q, k, v = randn(4, H, d, seed=i + 50).to(dtype), randn(4, G, d, seed=i + 60).to(dtype), randn(4, G, d, seed=i + 70).to(dtype)
        c.append(k, v, ints(range(5)), ints(pos), table, max_new=1, freq=freq)
        assert all(torch.equal(a[:length // BLOCK * BLOCK], b[:length // BLOCK * BLOCK]) for a, b in zip(before, held(c, table, 3, length)))
        assert not torch.equal(held(c, table, 2, length + 1)[0][-1], held(c, table, 3, length + 1)[0][-1])
        check_attention(c, table, q, [1] * 4, pos, c.attend(q, ints(range(5)), ints(pos), table, max_new=1, max_len=max(lens)))
        c.check_device_errors()


def test_calls_on_several_streams_at_once():
    """Kernels for few, 32 and many rows, in clusters and with shares through memory, beside kept rows and copied pages: each as it is alone."""
    from smoltts_b200.kv_cache import copy_pages, keep_rows

    H, G, d = 8, 2, 128
    calls = []
    for i, (n, context, dtype) in enumerate([(1, 3000, torch.bfloat16), (5, 2100, torch.bfloat16), (16, 9000, torch.bfloat16), (70, 3000, torch.bfloat16), (9, 700, torch.float32)]):
        c, table = cache_of([context + n, 300 + n], 64, G, d, d, seed=i)
        fill(c, table, [context + n, 300 + n], seed=i)
        q = randn(2 * n, H, d, seed=i + 50).to(dtype)
        tree = tree_of(c, [parents_of("random", n, 1), parents_of("fan", n)], [context, 300])
        args = (q, ints([0, n, 2 * n]), ints([context, 300]), table)
        calls.append((c, lambda c=c, args=args, n=n, context=context, tree=tree: c.attend(*args, max_new=n, max_len=context + n, tree=tree)))
    moved, table = cache_of([400], 64, G, d, d, seed=9)
    fill(moved, table, [400], seed=9)
    want = [call() for _, call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(len(calls) + 1)]
    rows, counts, pos0, page = ints([[0, 20, 30]]), ints([3]), ints([350]), int(table[0, 0])
    spare = next(p for p in range(moved.n_pages) if p not in table.flatten().tolist())
    for _ in range(30):
        got = []
        for (_, call), stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                got.append(call())
        with torch.cuda.stream(streams[-1]):
            keep_rows(moved, pos0, table, rows, counts)
            copy_pages(moved, [page], [spare])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert torch.equal(moved.k.view(torch.uint8)[page], moved.k.view(torch.uint8)[spare])
    for c, _ in calls:
        c.check_device_errors()


def test_a_captured_step_is_replayed_beside_another():
    """Tree, append, attention, rows and pages in two graphs on two streams, replayed in turn and at once with new inputs: as the calls themselves on the same contents."""
    from smoltts_b200.kv_cache import copy_pages, keep_rows

    H, G, d, n = 8, 2, 64, 24
    steps = []
    for which in range(2):
        torch.manual_seed(which)
        c, table = cache_of([3000 + n, 200 + n], 32, G, d, d, seed=which)
        fill(c, table, [3000, 200], seed=which)
        spare = [p for p in range(c.n_pages) if p not in set(table.flatten().tolist())][:1]
        state = dict(parents=ints([-1] * (2 * n)), q=randn(2 * n, H, d).to(torch.bfloat16), k=randn(2 * n, G, d).to(torch.bfloat16), v=randn(2 * n, G, d).to(torch.bfloat16), pos0=ints([3000, 200]), start=ints([0, n, 2 * n]),
                     rows=ints([[0, 3, 7]] * 2), counts=ints([3, 3]), freq=torch.ones(d // 2, device="cuda"))

        def step(c=c, table=table, s=state, first=[int(table[0, 0])], spare=spare):
            tree = c.draft_tree(s["parents"], s["start"], s["pos0"], max_new=n)
            q = c.append(s["k"], s["v"], s["start"], s["pos0"], table, max_new=n, q=s["q"], freq=s["freq"], positions=tree.positions)
            out = c.attend(q, s["start"], s["pos0"], table, max_new=n, max_len=3000 + n, tree=tree)
            keep_rows(c, s["pos0"], table, s["rows"], s["counts"])
            copy_pages(c, first, spare)
            return out

        steps.append((c, state, step))
    graphs = []
    for c, state, step in steps:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, stream))
    for round_ in range(3):
        starts_ = []
        for (c, state, step), (graph, out, stream) in zip(steps, graphs):
            state["parents"].copy_(ints(parents_of("random", n, round_) + parents_of("fan", n)))
            state["q"].copy_(randn(2 * n, H, d, seed=round_))
            starts_.append(contents(c))
        torch.cuda.synchronize()
        for graph, out, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (c, state, step), (graph, out, stream), before in zip(steps, graphs, starts_):
            after, got = contents(c), out.clone()
            for x, y in zip((c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale), before):
                x.copy_(y)
            want = step()
            assert torch.equal(want, got) and all(torch.equal(a, b) for a, b in zip(after, contents(c)))
            c.check_device_errors()
