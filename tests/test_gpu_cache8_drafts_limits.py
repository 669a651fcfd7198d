"""Drafting and forking on the 8-bit key/value cache: arrays that are wrong anywhere, magnitudes at the ends of their range, rows that must be left alone."""
from __future__ import annotations

import pytest
import torch

from cache8_util import exponent, ints, starts
from drafts_util import parents_of
from test_gpu_cache8 import cache_of, fill, held, randn
from test_gpu_cache8_drafts import arrays, check_kept, check_tree, contents, uneven

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- append

@pytest.mark.parametrize("name", ["positions", "axis", "freq"])
def test_queries_over_the_arrays_that_angles_are_made_of_are_refused(name):
    """Every block of threads reads them while others write queries.  Beside them, within the same memory, there is room."""
    c, table = cache_of([6], 16, 1, 16, 16, garbage=False)
    T, H, pairs = 6, 2, 4
    room = torch.zeros(T * H * 16 + 64, device="cuda")
    sizes = {"positions": 3 * T, "axis": pairs, "freq": pairs}
    x, q = randn(T, 1, 16), randn(T, H, 16, seed=1)
    want = None
    for at in (8, T * H * 16 - 3, T * H * 16 + 8):      # inside, over the end, behind
        arrays = {"positions": torch.arange(3 * T, device="cuda").int(), "axis": ints([0, 1, 2, 0]), "freq": torch.ones(pairs, device="cuda")}
        here = room[at:at + sizes[name]].view(arrays[name].dtype)
        here.copy_(arrays[name].flatten())
        arrays[name] = here
        arrays["positions"] = arrays["positions"].view(3, T)
        args = dict(q=q, q_out=room[:T * H * 16].view(T, H, 16), **arrays)
        if at < T * H * 16:
            with pytest.raises(ValueError, match=name):
                c.append(x, x, ints([0, T]), ints([0]), table, max_new=T, **args)
            assert (room[:8] == 0).all()
        else:
            got = c.append(x, x, ints([0, T]), ints([0]), table, max_new=T, **args)
            want = c.append(x, x, ints([0, T]), ints([0]), table, max_new=T, **{**args, "q_out": None})
            assert torch.equal(got, want)
    none = torch.zeros(0, device="cuda")      # no pairs, nothing that is read
    assert torch.equal(c.append(x, x, ints([0, T]), ints([0]), table, max_new=T, q=q, q_out=torch.empty_like(q), freq=none), q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,pairs,half", [(33, 5, True), (64, 20, False), (96, 12, True), (128, 60, True), (256, 100, False), (64, 24, True)])
def test_positions_that_are_the_places_change_nothing_whatever_the_pairs(dtype, d, pairs, half):
    lens, pos0, H, G = [5, 37, 1], [3, 21, 16], 6, 2
    freq = (10000.0 ** (-torch.arange(pairs, device="cuda") / pairs)).float()
    T = sum(lens)
    k, v, q = randn(T, G, d, seed=1).to(dtype), randn(T, G, d, seed=2).to(dtype), randn(T, H, d, seed=3).to(dtype)
    places = ints([p + i for p, n in zip(pos0, lens) for i in range(n)])
    results = []
    for more in (dict(), dict(positions=places), dict(positions=places.repeat(3, 1).contiguous(), axis=torch.randint(0, 3, (pairs,), device="cuda").int())):
        c, table = cache_of([p + n for p, n in zip(pos0, lens)], 32, G, d, d, garbage=False)
        out = c.append(k, v, ints(starts(lens)), ints(pos0), table, max_new=37, q=q, freq=freq, rot_half=half, **more)
        results.append((out, c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale))
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))


# ---------------------------------------------------------------------------------------------- kept rows

# (rows, pos0 of the sequence; 64 positions in four pages): entries behind the first wrong one that ascend among themselves, and destinations behind the table's last page
UNORDERED = [
    ([5, -40, -39], 9), ([5, -2000000000, -1999999999], 9), ([-2 ** 31, -2 ** 31 + 1, -5], 9), ([-1, 0, 1], 9), ([-3, -2, -1, 0, 1, 2], 20), ([0, 1, 1, 2, 3], 9), ([9, 0, 1, 2], 61), ([2, 0, 1, 2, 3], 60),
    ([40] + list(range(-30, 30)), 3), (list(range(33)) + [2, 3, 4, 5], 28), (list(range(32)) + [-2 ** 31, -2 ** 31 + 1], 3),
]


@pytest.mark.parametrize("rows,pos0", UNORDERED)
def test_rows_in_no_order_are_reported_wherever_they_are(rows, pos0):
    """The block table is a piece of a larger tensor whose other rows name pages too.  Nothing of the sequence moves; the one beside it is served."""
    from smoltts_b200._errors import SmolError
    from smoltts_b200.kv_cache import keep_rows

    good = [1, 4, 8, 20]
    lens = [64, 64]
    c, table = cache_of(lens, 16, 2, 32, 16)
    uneven(c, table, lens)
    before = contents(c)
    around = table.flip(0).repeat(3, 1)
    around[2:4] = table
    most = max(len(rows), len(good))
    given = ints([rows + [0] * (most - len(rows)), good + [10 ** 6] * (most - len(good))])
    keep_rows(c, ints([pos0, 9]), around[2:4], given, ints([len(rows), len(good)]))
    check_kept(c, before, table, [pos0, 9], [[], good])
    with pytest.raises(SmolError, match="word 2"):
        c.check_device_errors()


@pytest.mark.parametrize("d,dv", [(64, 64), (128, 80), (256, 33)])
@pytest.mark.parametrize("power", [16, 40, 99])
def test_rows_of_zeros_from_blocks_of_any_scale(d, dv, power):
    """Rows that are zeros, or far below what lies beside them, are kept from a block of a large scale: into a block of zeros, of small numbers, and behind older rows of either.  No code of
    them may come out as anything but what its value is."""
    from smoltts_b200.kv_cache import keep_rows

    lens, pos0 = [64, 64, 64, 64], [16, 20, 16, 20]
    rows = [[0, 3, 17], [1, 3, 17], [0, 3, 17], [1, 3, 17]]
    c, table = cache_of(lens, 32, 2, d, dv)
    T = sum(lens)
    k, v = torch.zeros(T, 2, d, device="cuda"), torch.zeros(T, 2, dv, device="cuda")
    for x in (k, v):
        x = x.view(4, 64, *x.shape[1:])
        x[2:, 16:32] = 2.0 ** -99      # (the smallest that a scale of its own holds is 2^-110 times the least code)
        x[:, 34] = 2.0 ** power        # beside the last of the kept rows, and far above it
        x[2:, 19] = 2.0 ** -80
        x[1:, 36] = 2.0 ** (power - 12)
    c.append(k, v, ints(starts(lens)), ints([0] * 4), table, max_new=64)
    before = contents(c)
    keep_rows(c, ints(pos0), table, *arrays(rows))
    check_kept(c, before, table, pos0, rows)
    for x in c.values(table.flatten().long()):
        assert torch.isfinite(x).all()


def rounded(x, e):
    """x as codes of scale 2^e hold it, in 64 bits."""
    return (x.double() * 2.0 ** -e).float().to(torch.float8_e4m3fn).double() * 2.0 ** e


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("context", [16, 21])
def test_a_rejected_row_leaves_its_scale_behind(dtype, context):
    """One of six drafted rows is 2^12 larger than the others and rejected.  In a block that the context began, its rows and the kept ones hold what the raised scale leaves of them (2^-4 of
    themselves, twice for the older ones, and 2^-10 of the scale); in a block of kept rows alone the scale is made anew, for codes that were rounded under the raised one."""
    from smoltts_b200.kv_cache import keep_rows

    G, d, accepted = 2, 64, [0, 1, 4]
    c, table = cache_of([32], 32, G, d, d, garbage=False)
    x = randn(context + 6, G, d, seed=1).clamp(-3, 3)
    x[context + 3] *= 2.0 ** 12
    x = x.to(dtype)
    c.append(x[:context], x[:context], ints([0, context]), ints([0]), table, max_new=context)
    first = held(c, table, 0, 16)
    c.append(x[context:], x[context:], ints([0, 6]), ints([context]), table, max_new=6)
    keep_rows(c, ints([context]), table, ints([accepted]), ints([3]))
    for got, old in zip(held(c, table, 0, context + 3), first):
        assert torch.equal(got[:16], old)      # (the block in front of the drafted rows')
        for g in range(G):
            older, new = x[16:context, g].double(), x[[context + r for r in accepted], g].double()
            alone, raised = exponent(torch.cat([older, new]).abs().max().item()), exponent(x[16:, g].abs().max().item())
            assert raised - alone in (11, 12, 13)
            if context == 16:
                want = rounded(new, raised)
                want = rounded(want, exponent(want.abs().max().item()))
            else:
                want = torch.cat([rounded(rounded(older, exponent(older.abs().max().item())), raised), rounded(new, raised)])
            assert torch.equal(got[16:, g].double(), want)
            plain = torch.cat([older, new])
            # two roundings: 2 * 2^-4 + 2^-8 of the value; the second one's half step at the least codes, and the first one's, which is 2^-11 of that
            assert ((got[16:, g].double() - plain).abs() <= 0.1290 * plain.abs() + 1.001 * 2.0 ** (raised - 10)).all()
            assert (want == 0).sum() > (rounded(plain, alone) == 0).sum()
            assert c.k_scale[table[0, 0], g, 1].item() == 2.0 ** (exponent(want.abs().max().item()) if context == 16 else raised)
    c.check_device_errors()


# ---------------------------------------------------------------------------------------------- attention along paths

@pytest.mark.parametrize("dtype,rows", [(torch.bfloat16, [1, 2]), (torch.bfloat16, [6, 20]), (torch.bfloat16, [100, 40]), (torch.bfloat16, [90, 3]), (torch.float32, [1, 2]), (torch.float32, [30, 9])])
@pytest.mark.parametrize("context", [40, 600, 9000])
@pytest.mark.parametrize("first", [-1, -1000, -2 ** 31])
def test_a_tree_in_front_of_the_first_position_is_left_out(dtype, rows, context, first):
    """Few, 32 and many rows, both in one batch, and float32; keys in one share, in shares that a cluster joins, and in shares that go through memory.  The sequences beside it are served."""
    from smoltts_b200._errors import SmolError

    H, G, d = 4, 2, 64
    counts, pos0 = [rows[0], rows[1], rows[0]], [context, 50, 17]
    lens = [p + n for p, n in zip(pos0, counts)]
    c, table = cache_of(lens, 64, G, d, d)
    fill(c, table, lens)
    q = randn(sum(counts), H, d, seed=3).to(dtype)
    start = starts(counts)
    tree = c.draft_tree(ints(sum([parents_of("fan", n) for n in counts], [])), ints(start), ints(pos0), max_new=max(counts))
    c.check_device_errors()
    given = ints([context, first, 17])
    for _ in range(2):
        junk = [torch.full((1 << 22,), 3.0, device="cuda") for _ in range(3)]      # what a workspace may find
        del junk
        out = torch.full((sum(counts), H, d), 7.0, device="cuda", dtype=dtype)
        c.attend(q, ints(start), given, table, max_new=max(counts), max_len=context + max(counts), out=out, tree=tree)
        assert (out[start[1]:start[2]] == 7).all()
        out[start[1]:start[2]] = c.attend(q, ints(start), ints(pos0), table, max_new=max(counts), max_len=context + max(counts), tree=tree)[start[1]:start[2]]
        check_tree(c, table, q, counts, pos0, tree, out)
        with pytest.raises(SmolError, match="word 2"):
            c.check_device_errors()
        c._err.zero_()
