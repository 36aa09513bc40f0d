"""The cache manager: pages of keys and values with a block table per request, and slots
for per-request state of fixed size.  Host-side bookkeeping only; the device tensors that
the pages index belong to the engine.

The reference gives every request private pages that it allocates lazily and returns when
the request's buffer is closed (core/src/main/java/io/teknek/deliverance/tensor/
KvBufferCache.java:826-841,851-865); there is no pool with a limit and nothing is shared
between requests.  Here a pool of fixed size serves all requests:

* A *group* is a set of cache slots (one per caching layer call) with the same needs: all
  keys, a window of the last w, or the chunk of c positions that the next one lies in.  Each group has pages of its own; one page id names the
  same page in every slot of the group.
* A request's *block table* for a group lists the page of each run of ``page_size``
  positions; the entry is -1 once a window has passed that run and the page went back
  (pages that hold positions a windowed group keeps for good, ``keep_first``, never do).
* ``extend`` reserves pages for a request's next tokens (all groups or nothing);
  ``commit`` makes them part of the request and returns pages that a window has passed;
  ``close`` returns everything.
* ``fork`` makes a request that continues another one: full pages are held by both (a page goes
  back when nobody holds it any more), the page that is being written is the new request's own.
  ``reorder`` lets requests of one length (the beams of a search) continue one another, in place.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Callable, Dict, Hashable, List, Optional, Sequence, Set, Tuple

import numpy as np


class CacheError(RuntimeError):
    """Misuse of the cache manager (unknown request, double free, ...)."""


class OutOfPages(CacheError):
    """Not enough free pages (or state slots) for what was asked."""


@dataclass(frozen=True)
class KVGroupSpec:
    """Cache slots that share pages.  ``window`` None keeps every key; with a window, the pages that hold
    a request's first ``keep_first`` positions are never given back while it lives.  With ``chunk`` (in place of a
    window) a position sees keys of its own chunk of so many positions only, counted from the sequence's start."""
    slots: Tuple[int, ...]
    n_kv_heads: int
    head_dim: int
    window: Optional[int] = None
    keep_first: int = 0
    chunk: Optional[int] = None


@dataclass(frozen=True)
class StateSpec:
    """Per-request state of fixed size for one cache slot: ``elems`` 32-bit floats."""
    slot: int
    elems: int


class PagePool:
    """Page ids 0..n-1 with an owner each, or several holders; free ids are handed out lowest first
    after reuse in last-freed-first order."""

    def __init__(self, n_pages: int):
        if n_pages < 0:
            raise CacheError("a pool cannot have a negative number of pages")
        self.n_pages = n_pages
        self._free: List[int] = list(range(n_pages - 1, -1, -1))
        self._owner: List[Optional[Hashable]] = [None] * n_pages
        self._holders: Dict[int, Set[Hashable]] = {}      # of the pages that more than one holds

    @property
    def n_free(self) -> int:
        return len(self._free)

    def take(self, n: int, owner: Hashable) -> List[int]:
        if owner is None:
            raise CacheError("pages need an owner")
        if n > len(self._free):
            raise OutOfPages(f"asked for {n} pages, {len(self._free)} free of {self.n_pages}")
        out = [self._free.pop() for _ in range(n)]
        for p in out:
            self._owner[p] = owner
        return out

    def share(self, pages: Sequence[int], owner: Hashable) -> None:
        """``owner`` holds these pages too; they are free again once every holder has given them back."""
        if owner is None:
            raise CacheError("pages need an owner")
        for p in pages:
            if p < 0 or p >= self.n_pages or self._owner[p] is None:
                raise CacheError(f"page {p} is nobody's")
            if self.held_by(p, owner):
                raise CacheError(f"page {p} is held by {owner!r} already")
            self._holders.setdefault(p, {self._owner[p]}).add(owner)

    def held_by(self, page: int, owner: Hashable) -> bool:
        return owner in self._holders[page] if page in self._holders else self._owner[page] == owner

    def give(self, pages: Sequence[int], owner: Hashable) -> List[int]:
        """Returns the pages that are free now (those that somebody else holds are not)."""
        freed = []
        for p in pages:
            if p < 0 or p >= self.n_pages:
                raise CacheError(f"page {p} is not in the pool")
            if self._owner[p] is None:
                raise CacheError(f"page {p} freed twice")
            if not self.held_by(p, owner):
                raise CacheError(f"page {p} belongs to {self._owner[p]!r}, not to {owner!r}")
            holders = self._holders.get(p)
            if holders is not None:
                holders.remove(owner)
                if self._owner[p] == owner:
                    self._owner[p] = next(iter(holders))
                if len(holders) == 1:
                    del self._holders[p]
                continue
            self._owner[p] = None
            self._free.append(p)
            freed.append(p)
        return freed

    def owner_of(self, page: int):
        return self._owner[page]


@dataclass
class _Request:
    length: int = 0                     # positions committed
    pending: int = 0                    # positions reserved by extend, not yet committed
    tables: List[List[int]] = field(default_factory=list)   # per group
    state_slot: int = -1


class CacheManager:
    def __init__(self, groups: Sequence[KVGroupSpec], page_size: int, pages_per_group: Sequence[int],
                 state_specs: Sequence[StateSpec] = (), n_state_slots: int = 0):
        if page_size <= 0:
            raise CacheError("page_size must be positive")
        if len(groups) != len(pages_per_group):
            raise CacheError("one page count per group is needed")
        self.groups = list(groups)
        self.page_size = page_size
        self.pools = [PagePool(n) for n in pages_per_group]
        self.state_specs = list(state_specs)
        self.n_state_slots = n_state_slots
        self._free_slots: List[int] = list(range(n_state_slots - 1, -1, -1))
        self._slot_owner: List[Optional[Hashable]] = [None] * n_state_slots
        self._reqs: Dict[Hashable, _Request] = {}
        # called with (group, pages) whenever pages go back to a pool (a debug run poisons them)
        self.on_release: Optional[Callable[[int, Sequence[int]], None]] = None

    # ---- requests ----------------------------------------------------------------
    def __contains__(self, rid) -> bool:
        return rid in self._reqs

    def live(self):
        return list(self._reqs.keys())

    def open(self, rid: Hashable) -> int:
        """Start a request; returns its state slot (-1 when the model keeps no state)."""
        if rid in self._reqs:
            raise CacheError(f"request {rid!r} is already open")
        slot = -1
        if self.n_state_slots:
            if not self._free_slots:
                raise OutOfPages(f"no state slot free of {self.n_state_slots}")
            slot = self._free_slots.pop()
            self._slot_owner[slot] = rid
        self._reqs[rid] = _Request(tables=[[] for _ in self.groups], state_slot=slot)
        return slot

    def can_open(self) -> bool:
        return self.n_state_slots == 0 or bool(self._free_slots)

    def _req(self, rid) -> _Request:
        try:
            return self._reqs[rid]
        except KeyError:
            raise CacheError(f"request {rid!r} is not open") from None

    def length(self, rid) -> int:
        return self._req(rid).length

    def pending(self, rid) -> int:
        """Positions reserved beyond ``length`` and not yet committed."""
        return self._req(rid).pending

    def state_slot(self, rid) -> int:
        return self._req(rid).state_slot

    def table(self, rid, group: int) -> List[int]:
        return self._req(rid).tables[group]

    # ---- pages -------------------------------------------------------------------
    def _first_live_page(self, group: int, first_query_pos: int) -> int:
        """Index of the first page a query at ``first_query_pos`` or later can still see."""
        w, c = self.groups[group].window, self.groups[group].chunk
        if c is not None:
            return (first_query_pos // c * c) // self.page_size
        if w is None:
            return 0
        lo = max(0, first_query_pos - w + 1)
        return lo // self.page_size

    def pages_needed(self, rid, n_new: int) -> List[int]:
        """New pages per group to hold positions [length, length + pending + n_new)."""
        r = self._req(rid)
        end = r.length + r.pending + n_new
        want = -(-end // self.page_size)
        return [max(0, want - len(t)) for t in r.tables]

    def can_extend(self, rid, n_new: int) -> bool:
        return all(n <= pool.n_free for n, pool in zip(self.pages_needed(rid, n_new), self.pools))

    def extend(self, rid, n_new: int) -> int:
        """Reserve room for ``n_new`` more positions; returns the first new position.
        Either every group gets its pages or nothing changes."""
        if n_new <= 0:
            raise CacheError("extend needs a positive number of positions")
        r = self._req(rid)
        need = self.pages_needed(rid, n_new)
        for n, pool in zip(need, self.pools):
            if n > pool.n_free:
                raise OutOfPages(
                    f"request {rid!r} needs {need} new pages per group, free: {[p.n_free for p in self.pools]}")
        for g, (n, pool) in enumerate(zip(need, self.pools)):
            r.tables[g].extend(pool.take(n, rid))
        start = r.length + r.pending
        r.pending += n_new
        return start

    def _give(self, group: int, pages: Sequence[int], rid) -> List[int]:
        freed = self.pools[group].give(pages, rid)
        if freed and self.on_release is not None:
            self.on_release(group, freed)
        return freed

    def commit(self, rid, n: Optional[int] = None) -> List[Tuple[int, int]]:
        """The reserved positions (the first ``n`` of them, when given: a later step may have
        reserved more already) now belong to the request.  Pages that every later query
        has left behind (window groups) go back; returns them as (group, page)."""
        r = self._req(rid)
        k = r.pending if n is None else n
        if not (0 <= k <= r.pending):
            raise CacheError(f"request {rid!r}: cannot commit {k} of {r.pending} reserved positions")
        r.length += k
        r.pending -= k
        released = []
        for g, pool in enumerate(self.pools):
            first = self._first_live_page(g, r.length)     # the next query sits at r.length
            t = r.tables[g]
            kept = -(-max(0, self.groups[g].keep_first) // self.page_size)   # pages of the first tokens stay
            for j in range(kept, min(first, len(t))):
                if t[j] >= 0:
                    released += [(g, p) for p in self._give(g, [t[j]], rid)]
                    t[j] = -1
        return released

    def rollback(self, rid) -> None:
        """Drop a reservation that was never run (pages beyond the committed length go back)."""
        r = self._req(rid)
        keep = -(-r.length // self.page_size)
        for g, pool in enumerate(self.pools):
            t = r.tables[g]
            extra = [p for p in t[keep:] if p >= 0]
            self._give(g, extra, rid)
            del t[keep:]
        r.pending = 0

    def close(self, rid) -> None:
        """End of a request: every page and the state slot go back."""
        r = self._req(rid)
        for g in range(len(self.pools)):
            self._give(g, [p for p in r.tables[g] if p >= 0], rid)
        if r.state_slot >= 0:
            if self._slot_owner[r.state_slot] != rid:
                raise CacheError(f"state slot {r.state_slot} is not held by {rid!r}")
            self._slot_owner[r.state_slot] = None
            self._free_slots.append(r.state_slot)
        del self._reqs[rid]

    # ---- requests that continue one another ---------------------------------------------------
    def writing(self, rid, group: int) -> int:
        """The page that holds the request's last positions and has room for the next; -1 when the next
        position begins a page."""
        r = self._req(rid)
        return r.tables[group][r.length // self.page_size] if r.length % self.page_size else -1

    def fork(self, rid: Hashable, new: Hashable) -> None:
        """Start a request that continues ``rid`` where it stands.  Full pages are shared; the page that is being written
        (``writing``) and the state slot are the new request's own, and whoever holds the tensors fills them with what ``rid``'s
        hold.  Either everything is there or nothing changes."""
        r = self._req(rid)
        if r.pending:
            raise CacheError(f"request {rid!r} has positions reserved")
        full, part = divmod(r.length, self.page_size)
        if part and any(p.n_free < 1 for p in self.pools):
            raise OutOfPages(f"request {new!r} needs a page per group, free: {[p.n_free for p in self.pools]}")
        self.open(new)
        n = self._reqs[new]
        n.length = r.length
        for g, pool in enumerate(self.pools):
            shared = r.tables[g][:full]
            pool.share([p for p in shared if p >= 0], new)
            n.tables[g] = shared + (pool.take(1, new) if part else [])

    def reorder(self, rids: Sequence[Hashable], parents: Sequence[int]) -> None:
        """Request rids[i] continues what rids[parents[i]] was, for all i at once; they have one length and nothing reserved.  Full
        pages are shared; every request keeps its own page that is being written and its own state slot, and whoever holds
        the tensors reorders what these hold (``kernels.ops.state_reorder``)."""
        reqs = [self._req(rid) for rid in rids]
        if len(set(rids)) != len(reqs) or len(parents) != len(reqs) or any(not 0 <= p < len(reqs) for p in parents):
            raise CacheError(f"parents {list(parents)} of {len(reqs)} requests")
        if any(r.pending or r.length != reqs[0].length for r in reqs):
            raise CacheError("requests that continue one another have one length and nothing reserved")
        full = reqs[0].length // self.page_size if reqs else 0
        for g, pool in enumerate(self.pools):
            old = [r.tables[g] for r in reqs]
            new = [t if p == i else old[p][:full] + t[full:] for i, (t, p) in enumerate(zip(old, parents))]
            for rid, before, after in zip(rids, old, new):        # everybody takes before anybody gives
                if after is not before:
                    have = set(before)
                    pool.share([p for p in after[:full] if p >= 0 and p not in have], rid)
            for rid, r, before, after in zip(rids, reqs, old, new):
                if after is not before:
                    r.tables[g] = after
                    keep = set(after)
                    self._give(g, [p for p in before if p >= 0 and p not in keep], rid)

    # ---- addressing --------------------------------------------------------------
    def slots_for(self, rid, group: int, start: int, n: int) -> List[int]:
        """Cache row (page * page_size + offset) of positions start .. start+n-1."""
        t = self._req(rid).tables[group]
        ps = self.page_size
        if n > 16:                                   # long portions: the same by arrays
            pos = np.arange(start, start + n, dtype=np.int64)
            pages = np.asarray(t, dtype=np.int64)[pos // ps]
            if (pages < 0).any():
                p = int(pos[pages < 0][0])
                raise CacheError(f"position {p} of {rid!r} lies in a page that was given back")
            return (pages * ps + pos % ps).tolist()
        out = []
        for p in range(start, start + n):
            page = t[p // ps]
            if page < 0:
                raise CacheError(f"position {p} of {rid!r} lies in a page that was given back")
            out.append(page * ps + p % ps)
        return out

    # ---- invariants (used by tests and by debug runs) ------------------------------
    def check(self) -> None:
        for g, pool in enumerate(self.pools):
            held = {}
            for rid, r in self._reqs.items():
                for p in r.tables[g]:
                    if p < 0:
                        continue
                    if p in held and p not in pool._holders:
                        raise CacheError(f"group {g}: page {p} held by {held[p][0]!r} and {rid!r}")
                    held.setdefault(p, []).append(rid)
                    if not pool.held_by(p, rid):
                        raise CacheError(f"group {g}: page {p} in the table of {rid!r} but owned by {pool.owner_of(p)!r}")
                want = -(-(r.length + r.pending) // self.page_size)
                if len(r.tables[g]) != want:
                    raise CacheError(f"group {g}: table of {rid!r} has {len(r.tables[g])} entries for "
                                     f"{r.length + r.pending} positions")
            for p, holders in pool._holders.items():
                if len(holders) < 2 or holders != set(held.get(p, [])):
                    raise CacheError(f"group {g}: page {p} counted for {holders!r}, in the tables of {held.get(p)!r}")
            free = pool._free
            if len(set(free)) != len(free):
                raise CacheError(f"group {g}: a page is on the free list twice")
            if set(free) & set(held):
                raise CacheError(f"group {g}: a page is both free and held")
            if len(free) + len(held) != pool.n_pages:
                raise CacheError(f"group {g}: {len(free)} free + {len(held)} held != {pool.n_pages} pages")
        slots = [r.state_slot for r in self._reqs.values() if r.state_slot >= 0]
        if len(set(slots)) != len(slots):
            raise CacheError("a state slot is held twice")
        if self.n_state_slots and len(slots) + len(self._free_slots) != self.n_state_slots:
            raise CacheError("state slots lost")

    def stats(self) -> dict:
        return {"pages_free": [p.n_free for p in self.pools], "pages_total": [p.n_pages for p in self.pools],
                "requests": len(self._reqs), "state_slots_free": len(self._free_slots)}
