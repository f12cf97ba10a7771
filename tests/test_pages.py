"""The book of pages on the CPU (pages.py): what each call decides, that a failed call changes nothing, and a random walk of calls
against a model in which every slot has positions of its own; the device entry point's refusals."""
from __future__ import annotations

import ctypes
import random

import pytest

from vinf_3080ti_amd import _lib
from vinf_3080ti_amd.pages import PageBook

FAKE = ctypes.c_void_p(0x10000)


class Book(PageBook):
    """Each call gives its plan."""

    def reserve(self, segments):
        super().reserve(segments)
        return self.plan()

    def fork(self, src, dst, length):
        super().fork(src, dst, length)
        assert self.plan()[0] == []
        return self.plan()[1]

    def copy(self, pairs):
        super().copy(pairs)
        return self.plan()

    def compact(self):
        super().compact()
        assert self.copies() == len(self.plan()[0])
        return self.plan()

    @property
    def rows(self):
        return [self.row(s) for s in range(self.slots)]


def state(book):
    return book.rows, [book.holders(p) for p in range(book.pages)], book.available()


def sound(book):
    count = [0] * book.pages
    for row in book.rows:
        assert len(set(row)) == len(row) <= book.per_slot
        for p in row:
            count[p] += 1
    assert count == [book.holders(p) for p in range(book.pages)]
    assert book.available() == count.count(0)


def test_reserve_takes_the_lowest_pages():
    book = Book(10, 16, 4, 3)
    assert book.reserve([(0, 0, 17), (1, 0, 1)]) == ([], [(0, 0), (1, 1), (4, 2)])
    assert book.reserve([(0, 17, 15)]) == ([], [])  # to the end of a page it holds
    assert book.reserve([(0, 32, 1)]) == ([], [(2, 3)])
    book.free([0])
    assert book.reserve([(2, 0, 40)]) == ([], [(8, 0), (9, 1), (10, 3)])
    sound(book)


def test_fork_shares_until_written():
    book = Book(10, 16, 4, 4)
    book.reserve([(0, 0, 40)])
    assert book.fork(0, [1, 2], 40) == [(4, 0), (5, 1), (6, 2), (8, 0), (9, 1), (10, 2)]
    assert [book.holders(p) for p in range(3)] == [3, 3, 3] and book.available() == 7
    # slots 1 and 2 part from the shared last page, slot 0 is the last to hold it
    assert book.reserve([(1, 40, 1), (2, 40, 8), (0, 40, 1)]) == ([(2, 3), (2, 4)], [(6, 3), (10, 4)])
    # a whole page rewritten needs no copy of what it held
    assert book.reserve([(1, 16, 16)]) == ([], [(5, 5)])
    assert book.reserve([(2, 0, 15)]) == ([(0, 6)], [(8, 6)])
    book.free([0, 1], 16)
    assert [len(r) for r in book.rows] == [1, 1, 3, 0]
    sound(book)


def test_compact_moves_the_highest_into_the_holes():
    book = Book(12, 8, 6, 4)
    book.reserve([(0, 0, 24), (1, 0, 24), (2, 0, 24)])
    book.fork(2, [3], 20)
    book.free([0])
    assert book.compact() == ([(6, 0), (7, 1), (8, 2)], [(12, 0), (13, 1), (14, 2), (18, 0), (19, 1), (20, 2)])
    sound(book)
    assert book.compact() == ([], []) and book.rows[1] == [3, 4, 5]


def test_copy_of_a_copy_reads_the_original():
    book = Book(12, 8, 4, 4)
    book.reserve([(1, 0, 20)])
    copies, entries = book.copy([(1, 0, 20), (0, 2, 9)])
    assert copies == [(0, 3), (1, 4), (2, 5), (0, 6), (1, 7)] and entries[-2:] == [(8, 6), (9, 7)]
    sound(book)


def test_failed_calls_change_nothing():
    book = Book(6, 8, 4, 4)
    book.reserve([(0, 0, 20)])
    book.fork(0, [1], 20)
    before = state(book)
    for call in (lambda: book.reserve([(1, 20, 1), (2, 0, 8), (3, 0, 16)]),  # one page too few, after two were dealt
                 lambda: book.reserve([(2, 0, 8), (2, 24, 1)]), lambda: book.reserve([(4, 0, 1)]), lambda: book.reserve([(-1, 0, 1)]),
                 lambda: book.reserve([(0, 30, 3)]), lambda: book.reserve([(0, 0, 0)]), lambda: book.reserve([(0, -1, 1)]),
                 lambda: book.reserve([(2, 0, 8), (2 ** 32, 0, 1)]), lambda: book.reserve([(0, 2 ** 31 - 1, 1)]), lambda: book.fork(0, [1], 8), lambda: book.fork(0, [2, 2], 8),
                 lambda: book.fork(0, [2], 25), lambda: book.fork(0, [0], 0), lambda: book.fork(2, [3], 1), lambda: book.fork(9, [3], 0),
                 lambda: book.copy([(0, 2, 20), (0, 3, 8)]), lambda: book.copy([(0, 2, 8), (2, 3, 9)]), lambda: book.copy([(0, 0, 8)]),
                 lambda: book.copy([(2, 2, 8)]), lambda: book.copy([(0, 2, 8), (0, 2, 8)]), lambda: book.free([0, 7]),
                 lambda: book.free([0], -1), lambda: book.free([0], 33)):
        with pytest.raises(ValueError):
            call()
        assert state(book) == before


def test_book_shapes():
    lib = _lib.load()
    for bad in ((0, 8, 4, 4), (4, 0, 4, 4), (4, 8, 0, 4), (4, 8, 4, 0), (4, 8, 2 ** 16, 2 ** 15), (-1, 8, 4, 4), (2 ** 31, 8, 4, 4)):
        with pytest.raises(ValueError):
            PageBook(*bad)
    assert lib.vq_book_reserve(None, None, 0) == lib.vq_book_compact(None) == lib.vq_book_available(None) == _lib.VQ_ERR_ARG
    assert lib.vq_book_apply(None, None, None, 0, FAKE, None) == _lib.VQ_ERR_ARG
    book = Book(130, 8, 40, 4)  # more than two words of pages, the last one partly used
    book.reserve([(i, 0, 320) for i in range(3)])
    assert book.rows[2] == list(range(80, 120)) and book.available() == 10
    book.reserve([(3, 0, 80)])
    with pytest.raises(ValueError, match="exhausted"):
        book.reserve([(3, 80, 1)])
    book.free([1], 8)
    assert book.compact()[0] == [(p, p - 50) for p in range(91, 130)]
    sound(book)
    with pytest.raises(TypeError):
        book.free([0.5])
    with pytest.raises(TypeError):
        book.fork(0, 3, 8)


@pytest.mark.parametrize("seed", range(12))
def test_random_calls_against_a_model(seed):
    """Every position of every slot has a value; page contents follow the copies that the calls return, written only where a slot
    reserved: what a slot reads through its row is what the model says, whatever the others did."""
    rng = random.Random(seed)
    page, per, slots, pages = rng.choice([1, 4, 8]), 5, 6, rng.choice([9, 20, 30])
    book = Book(pages, page, per, slots)
    memory = [[None] * page for _ in range(pages)]
    model: list[list[int]] = [[] for _ in range(slots)]
    table = [None] * (slots * per)

    def apply(copies, entries=()):
        assert len({b for _, b in copies}) == len(copies) and not {a for a, _ in copies} & {b for _, b in copies}
        for a, b in copies:
            memory[b] = list(memory[a])
        for i, p in entries:
            table[i] = p

    for step in range(300):
        op, s = rng.randrange(6), rng.randrange(slots)
        try:
            if op <= 1:
                pos0 = rng.randint(0, len(model[s]))
                rows = rng.randint(1, 2 * page)
                apply(*book.reserve([(s, pos0, rows)]))
                for i in range(pos0, pos0 + rows):
                    model[s][i:i + 1] = [step * 1000 + i]
                    assert book.holders(book.rows[s][i // page]) == 1
                    memory[book.rows[s][i // page]][i % page] = step * 1000 + i
            elif op == 2:
                n, to = rng.randint(0, len(model[s])), [t for t in range(slots) if t != s and rng.random() < 0.3]
                apply([], book.fork(s, to, n))
                for t in to:
                    model[t] = model[s][:n]
            elif op == 3:
                t, n = rng.randrange(slots), rng.randint(0, len(model[s]))
                apply(*book.copy([(s, t, n)]))
                model[t] = model[s][:n]
            elif op == 4:
                n = rng.randint(0, len(model[s]))
                book.free([s], n)
                model[s] = model[s][:n]
            else:
                apply(*book.compact())
                assert all(p < pages - book.available() for row in book.rows for p in row)
        except ValueError:
            pass
        sound(book)
        for t in range(slots):
            assert [memory[table[t * per + i // page]][i % page] for i in range(len(model[t]))] == model[t]
            assert len(book.rows[t]) == -(-len(model[t]) // page)


def test_move_pages_refusals():
    lib = _lib.load()
    pools, size = (ctypes.c_void_p * 2)(0x10000, 0x20000), (ctypes.c_size_t * 2)(64, 32)

    def pairs(*p):
        return (ctypes.c_int32 * (2 * len(p)))(*[v for x in p for v in x])

    def call(copies=pairs((0, 1)), n=1, entries=None, m=0, pools=pools, size=size, count=2, pages=4, table=FAKE, length=8):
        return lib.vq_move_pages(pools, size, count, pages, copies, n, table, length, entries, m, None)

    assert call(n=0) == 0  # nothing to do, nothing launched
    for bad in (dict(copies=None), dict(pools=None), dict(size=None), dict(n=0, m=1), dict(n=0, m=1, entries=pairs((0, 0)), table=None),
                dict(pools=(ctypes.c_void_p * 2)(0x10000, None)), dict(copies=pairs((0, 1), (2, 1)), n=2),
                dict(copies=pairs((0, 1), (1, 2)), n=2), dict(copies=pairs((1, 2), (0, 1)), n=2), dict(copies=pairs((3, 3)))):
        assert call(**bad) == _lib.VQ_ERR_ARG, bad
    for bad in (dict(n=-1), dict(m=-1), dict(count=-1), dict(pages=0), dict(copies=pairs((0, 4))), dict(copies=pairs((-1, 0))),
                dict(size=(ctypes.c_size_t * 2)(64, 0)), dict(entries=pairs((8, 0)), m=1), dict(entries=pairs((-1, 0)), m=1)):
        assert call(**bad) == _lib.VQ_ERR_SHAPE, bad
