"""Host-side allocators of the engines' device pools: key/value pages and per-sequence state slots.

Both pools are index allocators over memory the engine owns; the device side sees only the indices (block tables,
slot arrays).  ``IndexPool`` hands out the lowest-numbered free index last (LIFO): an index freed by a finished
sequence is the first one reused, which keeps the working set of pages small and makes reuse bugs show early.
"""
from __future__ import annotations

from typing import Dict, Iterable, List, Sequence, Tuple

from ._errors import SMOL_ERR_CAPACITY, SmolError


class IndexPool:
    def __init__(self, n: int, what: str = "page"):
        self.n = int(n)
        self.what = what
        self._free: List[int] = list(range(self.n - 1, -1, -1))
        self._is_free = bytearray([1]) * self.n

    def __len__(self) -> int:
        """Indices currently free."""
        return len(self._free)

    def allocate(self, n: int = 1) -> List[int]:
        if n > len(self._free):
            raise SmolError(SMOL_ERR_CAPACITY, f"{self.what} pool exhausted: need {n}, {len(self._free)} of {self.n} free")
        got = [self._free.pop() for _ in range(n)]
        for i in got:
            self._is_free[i] = 0
        return got

    def _owners(self, i: int) -> int:
        return 1

    def _check(self, items: Iterable[int]) -> None:
        for i in items:
            if not 0 <= i < self.n or self._is_free[i]:
                raise ValueError(f"{self.what} {i} is not an allocated index of this pool")

    def _check_freed(self, items: List[int]) -> None:
        """Before anything is changed: all of them are allocated, and none comes more often than it has owners."""
        self._check(items)
        times: Dict[int, int] = {}
        for i in items:
            times[i] = times.get(i, 0) + 1
            if times[i] > self._owners(i):
                raise ValueError(f"{self.what} {i} is given back more often than it has owners")

    def free(self, items: Iterable[int]) -> None:
        items = list(items)
        self._check_freed(items)
        for i in items:
            self._is_free[i] = 1
        self._free.extend(reversed(items))


class PagePool(IndexPool):
    """Pages of ``page_size`` cached positions each.  A page may belong to several sequences, forks of one another, and is free when the last of them has given it back."""

    def __init__(self, n_pages: int, page_size: int):
        super().__init__(n_pages, "KV page")
        self.page_size = int(page_size)
        self._others: Dict[int, int] = {}      # owners of a page beside the first

    def share(self, items: Iterable[int]) -> None:
        """One owner more for every one of the pages, which are allocated."""
        items = list(items)
        self._check(items)
        for i in items:
            self._others[i] = self._others.get(i, 0) + 1

    def _owners(self, i: int) -> int:
        return 1 + self._others.get(i, 0)

    def free(self, items: Iterable[int]) -> None:
        """One owner less; a page without owners is free."""
        items, last = list(items), []
        self._check_freed(items)
        for i in items:
            if self._others.get(i, 0) > 0:
                self._others[i] -= 1
                if self._others[i] == 0:
                    del self._others[i]
            else:
                last.append(i)
        super().free(last)

    def fork(self, pages: Sequence[int], positions: int) -> Tuple[List[int], List[int], List[int]]:
        """Pages of a sequence that goes on from the first ``positions`` of one that has ``pages``: whole ones are shared, the last one, which both will go on filling, is a new
        one.  Returns the pages, and which are to be copied to which (``kv_cache.copy_pages``; at most one)."""
        need = self.pages_for(positions)
        if positions < 0 or need > len(pages):
            raise ValueError(f"{len(pages)} pages of {self.page_size} do not hold {positions} positions")
        whole = positions // self.page_size
        self._check(pages[:need])      # (in front of the allocation, which may hand out one that was given back)
        new = self.allocate(need - whole)
        self.share(pages[:whole])
        return [*pages[:whole], *new], list(pages[whole:need]), new

    def pages_for(self, positions: int) -> int:
        return (positions + self.page_size - 1) // self.page_size


class SlotPool(IndexPool):
    """Slots of per-sequence recurrent state."""

    def __init__(self, n_slots: int):
        super().__init__(n_slots, "state slot")
