"""The cache manager: pages of keys and values with a block table per request,
one set of pages per group of layers with the same needs, and slots of
fixed-size state.

Storage of a paged cache (one set of tensors per cache id, that is per writing
call of the run order): whatever the mixer's `CacheNeed` names, each tensor with
the page number in front and the page size where the need says "page". Attention
keeps keys `[pages, kv_heads, page_size, head_size]` and values
`[pages, kv_heads, head_size, page_size]` (values are kept transposed inside a
page: the kernels contract over the tokens of a page). Caches of one group share
page numbers, so one block table serves all of them. The reference's paged
layout is `[num_blocks, block_size, n_kv_heads, d_head]` (decoder.py:1777-1780)
with `slot = block * block_size + offset` (hlo.py:3665-3704); the slot rule is
kept, the order inside a page is ours.

Pages are not cleared when they change hands: every read is bounded by the
reader's own length.
"""
from dataclasses import dataclass, field
from typing import Dict, Hashable, List, Optional

import numpy as np
import torch

from ..parts.base import CacheNeed
from .pages import OutOfPages, OutOfSlots, PagePool, SlotPool


@dataclass
class LayerCache:
    """What one call of the run order is handed."""
    cache_id: int
    group: Optional[str]            # name of the page group (None for state-only caches)
    writes: bool = True
    pages: Dict[str, torch.Tensor] = field(default_factory=dict)   # name -> [pages, *shape with the page size in it]
    state: Dict[str, torch.Tensor] = field(default_factory=dict)   # name -> [slots, *shape]

    @property
    def k_pages(self) -> Optional[torch.Tensor]:
        return self.pages.get("k")

    @property
    def v_pages(self) -> Optional[torch.Tensor]:
        return self.pages.get("v")

    def reader(self) -> "LayerCache":
        return LayerCache(self.cache_id, self.group, False, self.pages, self.state)


@dataclass
class PageGroup:
    name: str
    window: Optional[int]
    page_size: int
    pool: PagePool
    cache_ids: List[int]


@dataclass
class RequestPages:
    slot: int
    num_tokens: int = 0                                  # tokens whose keys/values are stored
    tables: Dict[str, List[int]] = field(default_factory=dict)   # group -> page per position block, -1 once released


class CacheManager:
    """Bookkeeping on the host, tensors on the device.

    needs      {cache id: CacheNeed} of the calls that write a cache
    num_pages  pages per group (an int for all groups, or {group name: int})
    """

    def __init__(self, needs: Dict[int, CacheNeed], page_size: int, num_pages, max_seqs: int,
                 dtype: torch.dtype, device, allocate: bool = True, page_pad_bytes: int = 0, ops=None):
        """`ops`: the kernel backend, which copies pages and state where requests are forked, pages moved.
        `page_pad_bytes`: memory left between one page and the next in every page tensor (a multiple of 32).
        Pages whose size is a power of two lie at distances that are powers of two, and so do the requests
        that fill them side by side: the kernels that read all requests at once then meet the same memory
        channels at the same time. A few hundred bytes between pages take that regularity away."""
        self.page_size, self.max_seqs, self.dtype, self.device = page_size, max_seqs, dtype, device
        if page_pad_bytes < 0 or page_pad_bytes % 32:
            raise ValueError(f"page_pad_bytes must be a multiple of 32 from 0 up, got {page_pad_bytes}")
        self.page_pad_bytes = page_pad_bytes
        self.ops, self.needs, self.allocated = ops, dict(needs), allocate
        self._row_sets: Dict[str, Dict[bool, object]] = {}     # group -> {bounded by tokens: the rows its pages are}
        self._state_rows = None                             # the slots' rows, of every state tensor
        self.slots = SlotPool(max_seqs)
        self.groups: Dict[str, PageGroup] = {}
        self.caches: Dict[int, LayerCache] = {}
        self.requests: Dict[Hashable, RequestPages] = {}
        by_key: Dict[tuple, str] = {}
        for cid in sorted(needs):
            need = needs[cid]
            if need is None:
                self.caches[cid] = LayerCache(cid, None)
                continue
            if need.kind == "paged":
                key = need.group_key()
                if key not in by_key:
                    name = "full" if need.window is None else f"window{need.window}"
                    by_key[key] = name
                    n = num_pages[name] if isinstance(num_pages, dict) else num_pages
                    self.groups[name] = PageGroup(name, need.window, page_size, PagePool(n), [])
                g = self.groups[by_key[key]]
                g.cache_ids.append(cid)
                lc = LayerCache(cid, g.name)
                if allocate:
                    lc.pages.update(self._new_pages(need, g.pool.num_pages))
                    sdt = getattr(torch, need.state_dtype)
                    for name, shape in need.state_shapes:       # a mixer that keeps pages and a fixed state
                        lc.state[name] = torch.zeros(max_seqs, *shape, dtype=sdt, device=device)
                self.caches[cid] = lc
            elif need.kind == "state":
                lc = LayerCache(cid, None)
                if allocate:
                    sdt = getattr(torch, need.state_dtype)
                    for name, shape in need.state_shapes:
                        lc.state[name] = torch.zeros(max_seqs, *shape, dtype=sdt, device=device)
                self.caches[cid] = lc
            else:
                raise ValueError(f"unknown cache kind {need.kind!r}")

    def _new_pages(self, need: CacheNeed, num_pages: int) -> Dict[str, torch.Tensor]:
        item = torch.empty(0, dtype=self.dtype).element_size()
        out = {}
        for name, shape in need.tensors_of_a_page():
            dims = [self.page_size if d == "page" else d for d in shape]
            count = int(np.prod(dims))
            whole = torch.empty(num_pages, count + self.page_pad_bytes // item, dtype=self.dtype, device=self.device)
            out[name] = whole[:, :count].view(num_pages, *dims)
        return out

    # ---------------------------------------------------------------- sizes

    @staticmethod
    def bytes_per_page(needs: Dict[int, CacheNeed], page_size: int, dtype: torch.dtype, page_pad_bytes: int = 0) -> int:
        item = torch.empty(0, dtype=dtype).element_size()
        total = 0
        for n in needs.values():
            if n is None or n.kind != "paged":
                continue
            for _, shape in n.tensors_of_a_page():
                count = 1
                for d in shape:
                    count *= page_size if d == "page" else d
                total += count * item + page_pad_bytes
        return total

    # ---------------------------------------------------------------- requests

    def add_request(self, req: Hashable) -> int:
        if req in self.requests:
            raise ValueError(f"request {req!r} is already live")
        slot = self.slots.allocate(req)
        self.requests[req] = RequestPages(slot, 0, {g: [] for g in self.groups})
        for lc in self.caches.values():
            for t in lc.state.values():
                t[slot].zero_()
        return slot

    def has(self, req: Hashable) -> bool:
        return req in self.requests

    def num_tokens(self, req: Hashable) -> int:
        return self.requests[req].num_tokens

    def _blocks_for(self, length: int) -> int:
        return -(-length // self.page_size)

    def pages_short(self, req: Hashable, new_len: int) -> Dict[str, int]:
        """Pages each group still has to hand out before `req` can hold `new_len` tokens."""
        r = self.requests[req]
        return {g: max(0, self._blocks_for(new_len) - len(r.tables[g])) for g in self.groups}

    def can_grow(self, req: Hashable, new_len: int, reserve: Optional[Dict[str, int]] = None) -> bool:
        short = self.pages_short(req, new_len)
        return all(short[g] + (reserve or {}).get(g, 0) <= self.groups[g].pool.num_free for g in self.groups)

    def grow(self, req: Hashable, new_len: int) -> None:
        """Pages for positions up to `new_len`, in every group or in none."""
        r = self.requests[req]
        short = self.pages_short(req, new_len)
        for g, n in short.items():
            if n > self.groups[g].pool.num_free:
                raise OutOfPages(f"group {g}: {n} pages wanted for request {req!r}, "
                                 f"{self.groups[g].pool.num_free} free")
        for g, n in short.items():
            if n:
                r.tables[g].extend(self.groups[g].pool.allocate(n, req))

    def advance(self, req: Hashable, n_tokens: int) -> None:
        """`n_tokens` more are stored. Pages of a windowed group that no later
        query can reach go back to the pool: a query at position p reads keys
        `j > p - window`, and later queries have `p >= num_tokens`."""
        r = self.requests[req]
        r.num_tokens += n_tokens
        if r.num_tokens > len(next(iter(r.tables.values()), [])) * self.page_size and self.groups:
            raise AssertionError(f"request {req!r} advanced past its pages")
        for g in self.groups.values():
            if g.window is None:
                continue
            first_needed = r.num_tokens - g.window + 1
            table = r.tables[g.name]
            gone = [i for i, p in enumerate(table) if p >= 0 and (i + 1) * self.page_size <= first_needed]
            if gone:
                g.pool.free([table[i] for i in gone], req)
                for i in gone:
                    table[i] = -1

    def free_request(self, req: Hashable) -> None:
        r = self.requests.pop(req)
        for g in self.groups.values():
            g.pool.free([p for p in r.tables[g.name] if p >= 0], req)
        self.slots.free(r.slot, req)

    # ---------------------------------------------------------------- forks

    # Bytes of a run of places of which a part is worth copying alone. Values turned inside a page lie in runs of a line or two of memory:
    # a part of such a line costs more than the whole (8 pages of 40 of 64 tokens' values to 24, all layers of OPT-6.7b: 147 us, whole 77).
    BOUNDED_RUN = 1024

    def _rows(self, group: str, bounded: bool):
        """What the pages of a group are to `copy_rows`, of every layer's tensors; `bounded`: with the axes that tokens are counted on."""
        sets = self._row_sets.setdefault(group, {})
        if bounded not in sets:
            tensors, axes = [], []
            for cid in self.groups[group].cache_ids:
                for name, shape in self.needs[cid].tensors_of_a_page():
                    t = self.caches[cid].pages[name]
                    axis = 1 + tuple(shape).index("page") if "page" in shape else None
                    run = 0 if axis is None else t.stride(axis) * t.shape[axis] * t.element_size()
                    tensors.append(t)
                    axes.append(axis if bounded and run >= self.BOUNDED_RUN else None)
            sets[bounded] = self.ops.row_set(tensors, axes)
        return sets[bounded]

    def _state_tensors(self) -> List[torch.Tensor]:
        return [t for lc in self.caches.values() if lc.writes for t in lc.state.values()]

    def _copier(self):
        if self.ops is None:
            raise RuntimeError("this cache was made without a kernel backend and cannot copy what it holds")
        return self.ops

    @property
    def has_state(self) -> bool:
        return any(n is not None and bool(n.state_shapes) for n in self.needs.values())

    def can_fork(self, parent: Hashable, num_tokens: int) -> bool:
        """Whether the first `num_tokens` tokens of `parent` can be taken over: fixed state is that of the newest token alone, and
        of a windowed group the pages that a later query reads must not have been given back."""
        if parent not in self.requests:
            return False
        r = self.requests[parent]
        if not 0 <= num_tokens <= r.num_tokens or (self.has_state and num_tokens != r.num_tokens):
            return False
        for g in self.groups.values():
            table = r.tables[g.name]
            if any(table[b] < 0 for b in range(self._first_block(g, num_tokens), self._blocks_for(num_tokens))):
                return False
        return True

    def _first_block(self, g: PageGroup, num_tokens: int) -> int:
        """The first block that queries at `num_tokens` and later read (see `advance`)."""
        return 0 if g.window is None else max(0, num_tokens - g.window + 1) // self.page_size

    def fork(self, parent: Hashable, child: Hashable, num_tokens: Optional[int] = None) -> int:
        """`child` becomes a request that holds the first `num_tokens` tokens of `parent` (all it holds, if not given), without computing
        them: full pages are shared, each request keeps them until both have given them back; the page that is not full, which both will
        write to, and the fixed state are copied, by launches on the current stream. All it needs, or nothing, is taken. Returns its slot."""
        r = self.requests[parent]
        n = r.num_tokens if num_tokens is None else int(num_tokens)
        if child in self.requests:
            raise ValueError(f"request {child!r} is already live")
        if not self.can_fork(parent, n):
            raise ValueError(f"request {parent!r} holds {r.num_tokens} tokens, of which the first {n} cannot be taken over")
        full, rest = divmod(n, self.page_size)
        if rest:
            for g in self.groups.values():
                if g.pool.num_free < 1:
                    raise OutOfPages(f"group {g.name}: a page wanted for request {child!r}, none free")
        if self.allocated and (rest and self.groups or self.has_state):
            self._copier()
        slot = self.slots.allocate(child)
        mine = self.requests[child] = RequestPages(slot, n, {name: [] for name in self.groups})
        try:
            for g in self.groups.values():
                theirs, table = r.tables[g.name], mine.tables[g.name]
                table += self._share(g, r, n, child)
                if rest:
                    table += g.pool.allocate(1, child)
                    self._copy_pages(g, [theirs[full]], [table[-1]], [rest])
            self._copy_state([r.slot], [slot])
        except Exception:
            self.free_request(child)
            raise
        return slot

    def _share(self, g: PageGroup, r: RequestPages, num_tokens: int, child: Hashable) -> List[int]:
        """The table of a request that holds the full pages of these tokens too."""
        first, full = self._first_block(g, num_tokens), num_tokens // self.page_size
        shared = r.tables[g.name][first:full]
        g.pool.share(shared, child)
        return [-1] * min(first, full) + shared

    def _copy_pages(self, g: PageGroup, sources: List[int], targets: List[int], tokens: List[int]) -> None:
        if self.allocated and targets:
            rows = self._rows(g.name, True)
            self.ops.copy_rows(rows, sources, targets, tokens if rows.places is not None else None)

    def _copy_state(self, sources: List[int], targets: List[int]) -> None:
        if self.allocated and self.has_state and targets:
            if self._state_rows is None:
                self._state_rows = self.ops.row_set(self._state_tensors())
            self.ops.copy_rows(self._state_rows, sources, targets)

    def reorder(self, names: List[Hashable], parents: List[int]) -> None:
        """Request `names[i]` becomes what `names[parents[i]]` holds now: one that nobody goes on from is over, one that several go on
        from is forked for all but one of them; a name that nobody has yet is that of a new request. All of it or nothing: what is refused is refused first; then pages and slots are set
        aside, free ones before those of requests that are over; then they are copied to, one launch a group; the tables and names
        change last, and nothing of that can fail. (Where a launch fails behind another that has run, pages of requests that would have
        been over may have been written.)"""
        parents = [int(p) for p in parents]
        if len(parents) != len(names) or len(set(names)) != len(names):
            raise ValueError(f"{len(names)} requests, of unlike names, and a parent for each, got {len(parents)}")
        if any(not 0 <= p < len(names) for p in parents):
            raise ValueError(f"parents are 0 to {len(names) - 1}, got {parents}")
        children: Dict[int, List[int]] = {}
        for i, p in enumerate(parents):
            children.setdefault(p, []).append(i)
        for p in children:
            if names[p] not in self.requests:
                raise ValueError(f"request {names[p]!r} is not live")
        over = [name for i, name in enumerate(names) if i not in children and name in self.requests]
        for p, wanted in children.items():           # the first of them takes the parent itself over: it, where it is one of them
            if p in wanted:
                wanted.remove(p)
                wanted.insert(0, p)
        forks = [(self.requests[names[p]], i) for p, wanted in children.items() for i in wanted[1:]]
        copied = [(r, i) for r, i in forks if r.num_tokens % self.page_size]
        if self.allocated and (copied and self.groups or forks and self.has_state):
            self._copier()
        if len(forks) > self.slots.num_free + len(over):
            raise OutOfSlots(f"{len(forks)} request slots wanted, {self.slots.num_free + len(over)} free")
        held = object()                              # who holds what is set aside
        aside: Dict[str, List[int]] = {}
        slots: List[int] = []
        gone = set(over)
        try:
            for g in self.groups.values():
                free = g.pool.allocate(min(len(copied), g.pool.num_free), held)
                aside[g.name] = free
                if len(free) < len(copied):
                    theirs = dict.fromkeys(p for name in over for p in self.requests[name].tables[g.name]
                                           if p >= 0 and gone.issuperset(g.pool.holders_of(p)))
                    more = list(theirs)[:len(copied) - len(free)]
                    if len(free) + len(more) < len(copied):
                        raise OutOfPages(f"group {g.name}: {len(copied)} pages wanted, {len(free) + len(theirs)} free")
                    g.pool.share(more, held)
                    aside[g.name] = free + more
            slots += [self.slots.allocate(held) for _ in range(min(len(forks), self.slots.num_free))]
            taken = over[:len(forks) - len(slots)]
            into = slots + [self.requests[name].slot for name in taken]
            for g in self.groups.values():
                self._copy_pages(g, [r.tables[g.name][r.num_tokens // self.page_size] for r, _ in copied], aside[g.name],
                                 [r.num_tokens % self.page_size for r, _ in copied])
            self._copy_state([r.slot for r, _ in forks], into)
        except Exception:
            for name, pages in aside.items():
                self.groups[name].pool.free(pages, held)
            for s in slots:
                self.slots.free(s, held)
            raise
        marks = [object() for _ in names]            # names of nobody, until all have theirs
        for name in taken:
            self.slots.rename(self.requests[name].slot, name, held)
        for name in over:
            r = self.requests.pop(name)
            for g in self.groups.values():
                g.pool.free([p for p in r.tables[g.name] if p >= 0], name)
            if name not in taken:
                self.slots.free(r.slot, name)
        for slot, (r, i) in zip(into, forks):
            mine = self.requests[marks[i]] = RequestPages(slot, r.num_tokens, {})
            self.slots.rename(slot, held, marks[i])
            for g in self.groups.values():
                table = mine.tables[g.name] = self._share(g, r, r.num_tokens, marks[i])
                if r.num_tokens % self.page_size:
                    page = aside[g.name].pop(0)
                    g.pool.rename([page], held, marks[i])
                    table.append(page)
        for p, wanted in children.items():
            self.rename(names[p], marks[wanted[0]])
        for mark, name in zip(marks, names):
            self.rename(mark, name)

    def rename(self, req: Hashable, name: Hashable) -> None:
        """The request goes by another name from now on."""
        if name in self.requests:
            raise ValueError(f"request {name!r} is already live")
        r = self.requests.pop(req)
        for g in self.groups.values():
            g.pool.rename([p for p in r.tables[g.name] if p >= 0], req, name)
        self.slots.rename(r.slot, req, name)
        self.requests[name] = r

    # ---------------------------------------------------------------- where pages lie

    def _renumber(self, g: PageGroup, where: Dict[int, int]) -> None:
        for r in self.requests.values():
            r.tables[g.name] = [where[p] if p >= 0 else -1 for p in r.tables[g.name]]

    def compact(self) -> int:
        """Held pages move to the lowest numbers of their pools (one launch a group, on the current stream); the number moved. Requests
        keep what they hold; block tables made before are void."""
        moved = 0
        for g in self.groups.values():
            where = g.pool.packed(g.pool.num_pages)
            moves = [(p, q) for p, q in where.items() if p != q]
            if not moves:
                continue
            if self.allocated:
                self._copier().copy_rows(self._rows(g.name, False), [p for p, _ in moves], [q for _, q in moves])
            g.pool.repack(where, g.pool.num_pages)
            self._renumber(g, where)
            moved += len(moves)
        return moved

    def resize(self, num_pages) -> None:
        """Pools of another size (an int for all groups, or {group name: int}), with what is held carried over, layer by layer, so that
        one layer at a time lies in memory twice. `OutOfPages`, and nothing changed, where more pages are held than asked for."""
        sizes = {name: num_pages[name] if isinstance(num_pages, dict) else num_pages for name in self.groups}
        if any(n <= 0 for n in sizes.values()):
            raise ValueError(f"a page pool needs at least one page, got {num_pages}")
        for name, g in self.groups.items():
            g.pool.packed(sizes[name])               # (raises where they do not fit)
        if self.allocated and self.groups:
            self._copier()
        self.compact()
        # From here on a page keeps its number, so a layer that has its new tensors and one that has its old ones go by the same tables:
        # where memory runs out in between, the pools are as large as the smaller of the two, and all is as it was.
        self._row_sets.clear()
        for name, g in self.groups.items():
            held = [p for p in range(g.pool.num_pages) if g.pool.holders_of(p)]
            where = {p: p for p in held}
            try:
                for cid in g.cache_ids if self.allocated else ():
                    lc = self.caches[cid]
                    new = self._new_pages(self.needs[cid], sizes[name])
                    if held:
                        self.ops.copy_rows(self.ops.row_set([lc.pages[k] for k in new], targets=list(new.values())), held, held)
                    lc.pages.update(new)             # (the dictionary is the readers' too)
            except Exception:
                g.pool.repack(where, min(sizes[name], g.pool.num_pages))
                raise
            g.pool.repack(where, sizes[name])

    def reset(self) -> None:
        for req in list(self.requests):
            self.free_request(req)

    # ---------------------------------------------------------------- views

    def slot_of(self, req: Hashable) -> int:
        return self.requests[req].slot

    def block_table(self, reqs: List[Hashable], group: str) -> np.ndarray:
        """int32 `[len(reqs), widest]`, -1 where a request holds no page."""
        tables = [self.requests[r].tables[group] for r in reqs]
        width = max(1, max((len(t) for t in tables), default=1))
        out = np.full((len(reqs), width), -1, dtype=np.int32)
        for i, t in enumerate(tables):
            out[i, :len(t)] = t
        return out

    def check(self) -> None:
        """No page lost, none in a table whose request does not hold it; tables agree with the pools."""
        for g in self.groups.values():
            g.pool.check()
            holders: Dict[int, set] = {}
            for req, r in self.requests.items():
                for p in r.tables[g.name]:
                    if p < 0:
                        continue
                    if req in holders.setdefault(p, set()):
                        raise AssertionError(f"page {p} of group {g.name} is twice in {req!r}'s table")
                    holders[p].add(req)
            for p, reqs in holders.items():
                if set(g.pool.holders_of(p)) != reqs:
                    raise AssertionError(f"page {p} is in the tables of {reqs!r} but held by {g.pool.holders_of(p)!r}")
            if len(holders) + g.pool.num_free != g.pool.num_pages:
                raise AssertionError(f"group {g.name}: {g.pool.num_pages - len(holders) - g.pool.num_free} pages lost")
