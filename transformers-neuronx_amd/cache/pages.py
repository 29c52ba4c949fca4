"""Page and slot allocators: host-side bookkeeping only, no tensors.

The reference has no allocator: block tables and slot mappings come from the
caller (base.py:362-365, :386-398) and `kv_cache_manager.py` only moves whole
caches between devices. These are ours.
"""
from typing import Dict, Hashable, List, Optional


class OutOfPages(RuntimeError):
    """The pool cannot cover the request."""


class OutOfSlots(RuntimeError):
    """Every per-request state slot is taken."""


class PagePool:
    """A fixed number of pages with a LIFO free list, so that a page given back
    is the next one handed out and reuse shows early. Each page knows its holders:
    one, or several where requests share what it holds; it is free again when the
    last of them gives it back. Handing out a held page, or giving back a page
    twice or by one that does not hold it, raises."""

    def __init__(self, num_pages: int):
        if num_pages <= 0:
            raise ValueError(f"a page pool needs at least one page, got {num_pages}")
        self.num_pages = num_pages
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._holders: List[List[Hashable]] = [[] for _ in range(num_pages)]

    @property
    def num_free(self) -> int:
        return len(self._free)

    def allocate(self, n: int, holder: Hashable) -> List[int]:
        """`n` pages for `holder`, all or none."""
        if n > len(self._free):
            raise OutOfPages(f"{n} pages wanted, {len(self._free)} of {self.num_pages} free")
        pages = [self._free.pop() for _ in range(n)]
        for p in pages:
            if self._holders[p]:
                raise AssertionError(f"page {p} was on the free list while held by {self._holders[p][0]!r}")
            self._holders[p].append(holder)
        return pages

    def _held(self, pages: List[int], what: str) -> None:
        for p in pages:
            if not 0 <= p < self.num_pages:
                raise ValueError(f"page {p} is outside the pool")
            if not self._holders[p]:
                raise ValueError(f"page {p} is {what}")
        if len(set(pages)) != len(pages):
            raise ValueError("a page is named twice")

    def share(self, pages: List[int], holder: Hashable) -> None:
        """`holder` holds these pages too."""
        self._held(pages, "shared while nobody holds it")
        for p in pages:
            if holder in self._holders[p]:
                raise ValueError(f"page {p} is held by {holder!r} already")
        for p in pages:
            self._holders[p].append(holder)

    def free(self, pages: List[int], holder: Hashable) -> None:
        self._held(pages, "given back twice")
        for p in pages:
            if holder not in self._holders[p]:
                raise ValueError(f"page {p} is held by {self._holders[p][0]!r}, not by {holder!r}")
        for p in pages:
            self._holders[p].remove(holder)
            if not self._holders[p]:
                self._free.append(p)

    def rename(self, pages: List[int], holder: Hashable, name: Hashable) -> None:
        """What `holder` holds of these pages, `name` holds."""
        for p in pages:
            at = self._holders[p].index(holder)
            self._holders[p][at] = name

    def holder_of(self, page: int):
        """The page's holder (the first of several), None if it is free."""
        return self._holders[page][0] if self._holders[page] else None

    def holders_of(self, page: int) -> tuple:
        return tuple(self._holders[page])

    def packed(self, num_pages: int) -> Dict[int, int]:
        """{page: where it goes} of the held pages for a pool of `num_pages` that holds them as its first: a page stays where it
        is if it can, the others, lowest first, fill the places between."""
        held = [p for p in range(self.num_pages) if self._holders[p]]
        if len(held) > num_pages:
            raise OutOfPages(f"{len(held)} pages are held, a pool of {num_pages} was asked for")
        room = [p for p in range(len(held)) if not self._holders[p]]
        moves = iter(room)
        return {p: (p if p < len(held) else next(moves)) for p in held}

    def repack(self, where: Dict[int, int], num_pages: int) -> None:
        """Become a pool of `num_pages` whose held pages are `where` says they are."""
        holders: List[List[Hashable]] = [[] for _ in range(num_pages)]
        for p, q in where.items():
            holders[q] = self._holders[p]
        self.num_pages, self._holders = num_pages, holders
        self._free = [p for p in range(num_pages - 1, -1, -1) if not holders[p]]

    def check(self) -> None:
        """Every page is either free once or held."""
        free = sorted(self._free)
        if len(set(free)) != len(free):
            raise AssertionError("a page is on the free list twice")
        on_list = set(free)
        for p in range(self.num_pages):
            if bool(self._holders[p]) == (p in on_list):
                raise AssertionError(f"page {p} is {'both held and free' if self._holders[p] else 'lost'}")


class SlotPool:
    """Slots of fixed-size per-request state; a slot index is stable for the
    request's life."""

    def __init__(self, num_slots: int):
        self.num_slots = num_slots
        self._free = list(range(num_slots - 1, -1, -1))
        self._holder: Dict[int, Hashable] = {}

    @property
    def num_free(self) -> int:
        return len(self._free)

    def allocate(self, holder: Hashable) -> int:
        if not self._free:
            raise OutOfSlots(f"all {self.num_slots} request slots are taken")
        s = self._free.pop()
        self._holder[s] = holder
        return s

    def free(self, slot: int, holder: Hashable) -> None:
        if self._holder.get(slot) != holder:
            raise ValueError(f"slot {slot} is not held by {holder!r}")
        del self._holder[slot]
        self._free.append(slot)

    def rename(self, slot: int, holder: Hashable, name: Hashable) -> None:
        if self._holder.get(slot) != holder:
            raise ValueError(f"slot {slot} is not held by {holder!r}")
        self._holder[slot] = name
