"""Rows of a tree where magnitudes differ.  A chain of drafted rows is an ordinary portion, so every check of one holds for it: the ones that look for what a row's result depends on are
run again with the rows as a chain, in the kernels for few, for 9 to 64 and for many rows, and in float32."""
from __future__ import annotations

import pytest
import torch

import test_gpu_cache8_ranges as ranges
from test_gpu_cache8_ranges import LEAST_F32, LEAST_FEW, LEAST_TILES

pytestmark = pytest.mark.gpu

# 4 query heads over 2: 2, 14, 40 and 300 rows.  (From 9 rows on both parts of a weight have one unit, as in the tiles.)
KERNELS = [(torch.bfloat16, 1, LEAST_FEW), (torch.bfloat16, 7, LEAST_TILES), (torch.bfloat16, 20, LEAST_TILES), (torch.bfloat16, 150, LEAST_TILES), (torch.float32, 7, LEAST_F32)]


@pytest.fixture
def as_a_chain(monkeypatch):
    """Every attention's rows as a chain: at their places, each seeing itself and those in front of it."""
    from smoltts_b200.kv_cache import DraftTree, KVCache8

    attend = KVCache8.attend

    def chained(self, q, seq_start, seq_pos0, block_table, max_new, max_len, **options):
        start, pos0, words = seq_start.tolist(), seq_pos0.tolist(), (max_new + 31) // 32
        positions = torch.zeros(q.shape[0], dtype=torch.int32)
        sees = torch.zeros(q.shape[0], words * 32, dtype=torch.bool)
        for s, p in enumerate(pos0):
            n = start[s + 1] - start[s]
            positions[start[s]:start[s + 1]] = p + torch.arange(n, dtype=torch.int32)
            sees[start[s]:start[s + 1], :n] = torch.ones(n, n, dtype=torch.bool).tril()
        bits = (sees.view(-1, words, 32).long() << torch.arange(32)).sum(-1)
        bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()
        return attend(self, q, seq_start, seq_pos0, block_table, max_new, max_len, tree=DraftTree(positions.to(q.device), bits.to(q.device)), **options)

    monkeypatch.setattr(KVCache8, "attend", chained)


@pytest.mark.parametrize("dtype,n,least", KERNELS)
@pytest.mark.parametrize("power", [12, 100])
@pytest.mark.parametrize("where", ["later", "behind_the_window", "behind_kv_len", "little_weight", "infinity", "between"])
def test_a_row_depends_on_what_it_sees_alone(as_a_chain, dtype, n, least, power, where):
    ranges.test_a_row_depends_on_what_it_sees_alone(dtype, n, least, power, where)


@pytest.mark.parametrize("dtype,n,least", KERNELS)
@pytest.mark.parametrize("low", [0.0, 2.0 ** -90])
def test_blocks_of_zeros_and_of_everything(as_a_chain, dtype, n, least, low):
    ranges.test_blocks_of_zeros_and_of_everything(dtype, n, least, low)


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 1), (torch.bfloat16, 20), (torch.bfloat16, 40), (torch.float32, 7)])
def test_shares_of_the_keys_whose_values_differ(as_a_chain, dtype, n):
    ranges.test_shares_of_the_keys_whose_values_differ(dtype, n)


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 1), (torch.bfloat16, 20), (torch.bfloat16, 150), (torch.float32, 20)])
@pytest.mark.parametrize("rise", [30.0, 40.0, 44.0])
def test_rising_scores_of_large_values(as_a_chain, dtype, n, rise):
    ranges.test_rising_scores_of_large_values(dtype, n, rise)


def test_a_sink_far_above_the_scores(as_a_chain):
    ranges.test_a_sink_far_above_the_scores()


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 1), (torch.bfloat16, 20), (torch.bfloat16, 150), (torch.float32, 20)])
@pytest.mark.parametrize("cap", [300.0, 1e6, 3.4e38])
@pytest.mark.parametrize("scale", [0.125, 60.0])
def test_soft_caps_far_above_the_scores(as_a_chain, dtype, n, cap, scale):
    ranges.test_soft_caps_far_above_the_scores(dtype, n, cap, scale)


@pytest.mark.parametrize("scale", [1e-30, 1e4, 1e20])
def test_queries_of_any_size(as_a_chain, scale):
    import test_gpu_cache8 as plain

    plain.test_queries_of_any_size(scale)


@pytest.mark.parametrize("n", [9, 24])
def test_nan_and_infinite_queries_stay_in_their_rows(n):
    """A row of the tree that is not finite is NaN as a whole, and no other is."""
    import math

    from cache8_util import ints
    from drafts_util import parents_of
    from test_gpu_cache8 import cache_of, fill, randn

    H, G, d, L = 4, 2, 64, 300
    c, table = cache_of([L + n], 32, G, d, d)
    fill(c, table, [L + n])
    tree = c.draft_tree(ints(parents_of("fan", n)), ints([0, n]), ints([L]), max_new=n)
    for bad in (math.nan, math.inf, -math.inf):
        q = randn(n, H, d, seed=3).to(torch.bfloat16)
        q[4, 1, 7] = bad
        out = c.attend(q, ints([0, n]), ints([L]), table, max_new=n, max_len=L + n, tree=tree)
        want = torch.zeros(n, H, d, dtype=torch.bool, device="cuda")
        want[4, 1] = True
        assert torch.equal(torch.isnan(out), want)
