"""Drafting and forking on the 8-bit key/value cache: arrays that are wrong anywhere, magnitudes at the ends of their range, rows that must be left alone."""
from __future__ import annotations

import pytest
import torch

from cache8_util import ints
from test_gpu_cache8 import cache_of
from test_gpu_cache8_drafts import check_kept, contents, uneven

pytestmark = pytest.mark.gpu


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
