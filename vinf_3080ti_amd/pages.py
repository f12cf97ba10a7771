"""Which pages of the paged caches each sequence slot holds: the host's side of the page table (vq_book of include/vq.h).

The page table that the *_seg ops read is written from here. A page may be held by several slots (a forked prefix); it is given
back when its last holder lets go. Fresh pages are the lowest free ids, so the same calls give the same pages. Every change is
planned on the host, where all of it is known, and carried out on the device as one list of page copies and table entries.
"""
from __future__ import annotations

import array
import ctypes
from typing import Iterable, Sequence

from . import _lib


def _ints(values: Iterable[int]) -> array.array:
    try:
        return array.array("i", values)
    except OverflowError:
        raise ValueError("slots, positions and lengths are 32-bit numbers") from None


class PageBook:
    """Pages 0 .. pages - 1 of `page` positions, slots of up to `per_slot` pages. A call that cannot be carried out raises ValueError
    and changes nothing; after any other the plan is there to be read (plan) or carried out (apply), until the next call."""

    def __init__(self, pages: int, page: int, per_slot: int, slots: int) -> None:
        self._lib = _lib.load()
        self.pages, self.page, self.per_slot, self.slots = pages, page, per_slot, slots
        self._book = self._lib.vq_book_create(*_ints((pages, page, per_slot, slots)))
        if not self._book:
            raise ValueError(f"no book for {pages} pages of {page} positions, {slots} slots of {per_slot} pages")

    def __del__(self) -> None:
        if getattr(self, "_book", None):
            self._lib.vq_book_destroy(self._book)

    def _check(self, status: int) -> None:
        if status:
            words = self._lib.vq_book_error(self._book).decode()
            if status < 0 and words:
                raise ValueError(words)
            _lib.check(status, "pages")

    def reserve(self, segments: Iterable[Sequence[int]]) -> None:
        a = _ints(v for s in segments for v in (s[0], s[1], s[2], 0))
        self._check(self._lib.vq_book_reserve(self._book, a.buffer_info()[0], len(a) // 4))

    def fork(self, src: int, dst: Iterable[int], length: int) -> None:
        a = _ints((src, length, *dst))
        self._check(self._lib.vq_book_fork(self._book, a[0], a.buffer_info()[0] + 8, len(a) - 2, a[1]))

    def copy(self, pairs: Iterable[Sequence[int]]) -> None:
        a = _ints(v for p in pairs for v in (p[0], p[1], p[2]))
        self._check(self._lib.vq_book_copy(self._book, a.buffer_info()[0], len(a) // 3))

    def free(self, slots: Iterable[int], length: int = 0) -> None:
        a = _ints((length, *slots))
        self._check(self._lib.vq_book_free(self._book, a.buffer_info()[0] + 4, len(a) - 1, a[0]))

    def compact(self) -> None:
        self._check(self._lib.vq_book_compact(self._book))

    def _lists(self) -> tuple[int, int, int, int]:
        """Addresses and lengths of the plan's copies and entries."""
        c, e, nc, ne = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_int(), ctypes.c_int()
        self._lib.vq_book_plan(self._book, ctypes.byref(c), ctypes.byref(nc), ctypes.byref(e), ctypes.byref(ne))
        return c.value or 0, nc.value, e.value or 0, ne.value

    def copies(self) -> int:
        """Pages that the plan copies."""
        return self._lists()[1]

    def plan(self) -> tuple[list[tuple[int, int]], list[tuple[int, int]]]:
        """(copies, entries) of the last call: (from, to) pages and (index, page) of the table."""
        def pairs(at: int, n: int) -> list[tuple[int, int]]:
            flat = list((ctypes.c_int32 * (2 * n)).from_address(at)) if n else []
            return list(zip(flat[::2], flat[1::2]))

        c, nc, e, ne = self._lists()
        return pairs(c, nc), pairs(e, ne)

    def apply(self, pools: Sequence[int], page_bytes: Sequence[int], table: int, stream: int) -> None:
        """Carry the plan out: pools at these addresses with pages of these sizes, the page table at `table`."""
        at, sizes = array.array("Q", pools), array.array("Q", page_bytes)
        _lib.check(self._lib.vq_book_apply(self._book, at.buffer_info()[0], sizes.buffer_info()[0], len(at), table, stream), "pages")

    def row(self, slot: int) -> list[int]:
        """The pages that a slot holds, in the order of its positions."""
        at = ctypes.c_void_p()
        n = self._lib.vq_book_row(self._book, _ints((slot,))[0], ctypes.byref(at))
        if n < 0:
            raise ValueError(f"slot {slot} outside [0, {self.slots})")
        return list((ctypes.c_int32 * n).from_address(at.value)) if n else []

    def available(self) -> int:
        """Pages that no slot holds."""
        return self._lib.vq_book_available(self._book)

    def holders(self, page: int) -> int:
        """Slots that hold a page."""
        return self._lib.vq_book_holders(self._book, page)
