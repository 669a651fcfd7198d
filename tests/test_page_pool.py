"""Pages with several owners: sharing, forking, giving back."""
import pytest

from smoltts_b200._errors import SmolError
from smoltts_b200.pool import PagePool


def test_a_fork_shares_whole_pages_and_copies_the_last_one():
    pool = PagePool(10, 32)
    pages = pool.allocate(4)
    for positions, whole, copied in ((0, 0, 0), (1, 0, 1), (32, 1, 0), (33, 1, 1), (100, 3, 1), (128, 4, 0)):
        free = len(pool)
        mine, src, dst = pool.fork(pages, positions)
        assert mine[:whole] == pages[:whole] and mine[whole:] == dst and src == pages[whole:whole + copied] and len(dst) == copied
        assert not set(dst) & set(pages) and len(pool) == free - copied
        pool.free(mine)
        assert len(pool) == free
    pool.free(pages)
    assert len(pool) == 10 and sorted(pool.allocate(10)) == list(range(10))


def test_a_page_is_free_when_its_last_owner_gives_it_back():
    pool = PagePool(3, 16)
    pages = pool.allocate(2)
    pool.share(pages)
    pool.share(pages[:1])
    pool.free(pages)
    assert len(pool) == 1
    pool.free(pages)
    assert len(pool) == 2      # (the first one has an owner left)
    with pytest.raises(ValueError):
        pool.free(pages[1:])
    pool.free(pages[:1])
    assert len(pool) == 3
    with pytest.raises(ValueError):
        pool.free(pages[:1])


def test_owners_in_any_order_and_the_same_page_twice():
    pool = PagePool(2, 16)
    (page,) = pool.allocate(1)
    pool.share([page, page])
    pool.free([page, page, page])
    assert len(pool) == 2


def test_what_cannot_be_shared_or_forked_is_refused_and_changes_nothing():
    pool = PagePool(4, 16)
    pages = pool.allocate(3)
    for bad in ([3], [-1], [4], [pages[0], 3]):
        with pytest.raises(ValueError):
            pool.share(bad)
    pool.free(pages[:1])      # (nobody else had it)
    assert len(pool) == 2
    with pytest.raises(ValueError):
        pool.fork(pages[1:], 33)
    with pytest.raises(ValueError):
        pool.fork(pages[1:], -1)
    with pytest.raises(ValueError):
        pool.fork(pages, 17)      # (the first page was given back)
    assert len(pool) == 2
    pool.allocate(2)
    with pytest.raises(SmolError):
        pool.fork(pages[1:], 17)
    pool.free(pages[1:])
    assert len(pool) == 2
