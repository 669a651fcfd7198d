"""A refused call of the pools leaves owners and free indices as they were."""
import pytest

from smoltts_b200.pool import PagePool, SlotPool


def state(pool):
    return list(pool._free), bytes(pool._is_free), dict(getattr(pool, "_others", {}))


def test_a_refused_free_takes_no_owner_away():
    pool = PagePool(6, 16)
    a, b, c = pool.allocate(3)
    pool.share([a, b, b])
    before = state(pool)
    for bad in ([a, 5], [a, b, -1], [c, a, 6], [a, a, a], [b, a, b, b, b], [c, c], [a, c, c], [5, a]):
        with pytest.raises(ValueError):
            pool.free(bad)
        assert state(pool) == before, bad
    # each owner gives its pages back, and only then are they free
    pool.free([a, b])
    pool.free([b, a])
    assert len(pool) == 4
    pool.free([b, c])
    assert len(pool) == 6 and sorted(pool.allocate(6)) == list(range(6))


def test_a_page_that_a_fork_reads_is_not_handed_out_after_a_refused_free():
    pool = PagePool(3, 16)
    pages = pool.allocate(2)
    fork, src, dst = pool.fork(pages, 32)
    assert fork == pages and not src and not dst
    with pytest.raises(ValueError):
        pool.free([*pages, 2])
    pool.free(pages)      # the caller again, with its own pages
    assert len(pool) == 1 and pool.allocate(1) == [2]
    pool.free(fork)
    assert len(pool) == 2


def test_a_refused_free_loses_no_slot():
    pool = SlotPool(4)
    taken = pool.allocate(3)
    before = state(pool)
    for bad in ([taken[0], 3], [taken[0], taken[0]], [taken[1], 4], [taken[1], -1]):
        with pytest.raises(ValueError):
            pool.free(bad)
        assert state(pool) == before, bad
    pool.free(taken)
    assert len(pool) == 4
