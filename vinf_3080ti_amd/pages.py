"""Which pages of the paged caches each sequence slot holds: the host's side of the page table.

The page table that the *_seg ops read is written from here. A page may be held by several slots (a forked prefix); it is given
back when its last holder lets go. Fresh pages are the lowest free ids, so the same calls give the same pages. Every change is
planned on the host, where all of it is known, and handed to the device as one list of page copies and table entries.
"""
from __future__ import annotations

import heapq
from typing import Iterable, Sequence

import numpy as np


class PageBook:
    """Pages 0 .. pages - 1 of `page` positions, slots of up to `per_slot` pages."""

    def __init__(self, pages: int, page: int, per_slot: int, slots: int) -> None:
        self.pages, self.page, self.per_slot, self.slots = pages, page, per_slot, slots
        self.rows: list[list[int]] = [[] for _ in range(slots)]
        self.holders = [0] * pages
        self._free = list(range(pages))  # a heap

    def available(self) -> int:
        return len(self._free)

    def _slot(self, slot: int) -> int:
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} outside [0, {self.slots})")
        return slot

    def _covering(self, length: int) -> int:
        """Pages that hold `length` positions."""
        n = -(-length // self.page)
        if length < 0 or n > self.per_slot:
            raise ValueError(f"{length} positions outside the paged context")
        return n

    def _drop(self, page: int) -> None:
        self.holders[page] -= 1
        if not self.holders[page]:
            heapq.heappush(self._free, page)

    def reserve(self, segments: Iterable[Sequence[int]]) -> tuple[list[tuple[int, int]], list[tuple[int, int]]]:
        """Pages for the rows that each segment (slot, pos0, rows, ...) is about to write, of the slot's own: missing ones are
        taken, shared ones replaced, by a copy unless the segment writes all of the page. Returns (copies, entries); nothing has
        changed when it raises."""
        copies: list[tuple[int, int]] = []
        entries: list[tuple[int, int]] = []
        undo: list[tuple[int, int, int]] = []  # (slot, index, page before; -1: none)
        taken: list[int] = []
        try:
            for slot, pos0, rows in (tuple(int(v) for v in s[:3]) for s in segments):
                row = self.rows[self._slot(slot)]
                if pos0 < 0 or rows < 1:
                    raise ValueError(f"segment ({slot}, {pos0}, {rows}) outside the paged context")
                end = self._covering(pos0 + rows)
                first = pos0 // self.page
                if first > len(row):
                    raise ValueError(f"segment ({slot}, {pos0}, {rows}): slot holds {len(row)} pages, none before position {pos0}")
                for i in range(first, end):
                    old = row[i] if i < len(row) else -1
                    if old >= 0 and self.holders[old] == 1:
                        continue
                    if not self._free:
                        raise ValueError("page pool exhausted")
                    new = heapq.heappop(self._free)
                    taken.append(new)
                    self.holders[new] = 1
                    undo.append((slot, i, old))
                    if old < 0:
                        row.append(new)
                    else:
                        self.holders[old] -= 1  # others hold it still
                        row[i] = new
                        if pos0 > i * self.page or pos0 + rows < (i + 1) * self.page:
                            copies.append((old, new))
                    entries.append((slot * self.per_slot + i, new))
        except Exception:
            for slot, i, old in reversed(undo):
                if old < 0:
                    self.rows[slot].pop()
                else:
                    self.rows[slot][i] = old
                    self.holders[old] += 1
            for page in taken:
                self.holders[page] = 0
                heapq.heappush(self._free, page)
            raise
        return copies, entries

    def _empty(self, slots: Iterable[int]) -> list[int]:
        found = [self._slot(int(s)) for s in slots]
        for s in found:
            if self.rows[s]:
                raise ValueError(f"slot {s} holds {len(self.rows[s])} pages (free them first)")
        if len(set(found)) < len(found):
            raise ValueError("a slot is given twice")
        return found

    def _first(self, slot: int, length: int) -> list[int]:
        n = self._covering(length)
        row = self.rows[self._slot(slot)]
        if n > len(row):
            raise ValueError(f"slot {slot} holds {len(row)} pages, {length} positions need {n}")
        return row[:n]

    def fork(self, src: int, dst: Iterable[int], length: int) -> list[tuple[int, int]]:
        """Empty slots dst hold the pages of src's first `length` positions too. Returns the table's entries."""
        head = self._first(int(src), int(length))
        slots = self._empty(dst)
        for s in slots:
            self.rows[s] = list(head)
        for page in head:
            self.holders[page] += len(slots)
        return [(s * self.per_slot + i, page) for s in slots for i, page in enumerate(head)]

    def copy(self, pairs: Iterable[Sequence[int]]) -> tuple[list[tuple[int, int]], list[tuple[int, int]]]:
        """Empty slots get copies of other slots' first positions, in pages of their own: (src, dst, length) each. Returns
        (copies, entries); nothing has changed when it raises."""
        pairs = [tuple(int(v) for v in p) for p in pairs]
        slots = self._empty(p[1] for p in pairs)
        heads: dict[int, list[int]] = {}  # of slots filled by this call: the pages that their copies are made from
        for src, dst, length in pairs:
            if src in heads:
                n = self._covering(length)
                if n > len(heads[src]):
                    raise ValueError(f"slot {src} holds {len(heads[src])} pages, {length} positions need {n}")
                heads[dst] = heads[src][:n]
            else:
                heads[dst] = self._first(src, length)
        if sum(len(heads[s]) for s in slots) > len(self._free):
            raise ValueError("page pool exhausted")
        copies, entries = [], []
        for s in slots:
            for i, page in enumerate(heads[s]):
                new = heapq.heappop(self._free)
                self.holders[new] = 1
                self.rows[s].append(new)
                copies.append((page, new))
                entries.append((s * self.per_slot + i, new))
        return copies, entries

    def free(self, slots: Iterable[int], length: int = 0) -> None:
        """The slots keep the pages of their first `length` positions."""
        n = self._covering(int(length))
        found = [self._slot(int(s)) for s in slots]
        for s in found:
            row = self.rows[s]
            while len(row) > n:
                self._drop(row.pop())

    def compact(self) -> tuple[list[tuple[int, int]], list[tuple[int, int]]]:
        """The pages in use become 0 .. n - 1: the k-th page at n or above moves to the k-th free one below. No page is both
        read and written, whatever the order of the copies. Returns (copies, entries)."""
        n = self.pages - len(self._free)
        holes = sorted(p for p in self._free if p < n)
        movers = [p for p in range(n, self.pages) if self.holders[p]]
        to = dict(zip(movers, holes))
        entries = []
        if to:
            for s, row in enumerate(self.rows):
                for i, page in enumerate(row):
                    if page in to:
                        row[i] = to[page]
                        entries.append((s * self.per_slot + i, to[page]))
            for old, new in to.items():
                self.holders[new], self.holders[old] = self.holders[old], 0
            self._free = list(range(n, self.pages))
        return list(to.items()), entries


def as_pairs(pairs: Sequence[tuple[int, int]]) -> np.ndarray:
    """int32 [n][2], for the device call."""
    return np.array(pairs, np.int32).reshape(-1, 2)
