"""The runtime's page queries beside another thread's page calls, on the CPU (a Runtime without its device, its book alone)."""
from __future__ import annotations

import threading

import pytest

from vinf_3080ti_amd.pages import PageBook
from vinf_3080ti_amd.runtime import Runtime


class Watched:
    """The runtime's kind of lock, which knows whether it is held."""

    def __init__(self):
        self.lock, self.held = threading.RLock(), 0

    def __enter__(self):
        self.lock.acquire()
        self.held += 1

    def __exit__(self, *_):
        self.held -= 1
        self.lock.release()


@pytest.fixture
def rt():
    r = Runtime.__new__(Runtime)
    r._pages_lock = Watched()
    r._paging = None
    r._pages = (PageBook(280, 1, 300, 4), {}, [])
    return r


def test_queries_wait_for_a_change(rt):
    """The book is never read outside of the lock that its changes hold."""
    class Held(PageBook):
        def row(self, slot):
            assert rt._pages_lock.held
            return super().row(slot)

        def available(self):
            assert rt._pages_lock.held
            return super().available()

    rt._pages = (Held(280, 1, 300, 4), {}, [])
    assert rt.pages_of(0) == [] and rt.pages_available() == 280
    seen = []
    with rt._pages_lock:
        asks = [threading.Thread(target=lambda f=f: seen.append(f())) for f in (lambda: rt.pages_of(1), rt.pages_available)]
        for t in asks:
            t.start()
        asks[0].join(0.2)
        assert not seen
        rt._pages[0].reserve([(1, 0, 3)])
    for t in asks:
        t.join()
    assert sorted(seen, key=str) == [277, [0, 1, 2]]


def test_refused_calls_are_not_seen(rt):
    """While one thread's reserve is refused again and again, which changes nothing, another one sees the same pages."""
    book, stop = rt._pages[0], threading.Event()
    book.reserve([(0, 0, 20)])

    def refused():
        while not stop.is_set():
            with rt._pages_lock, pytest.raises(ValueError):
                book.reserve([(0, 0, 300)])

    t = threading.Thread(target=refused)
    t.start()
    try:
        for _ in range(2000):
            assert rt.pages_of(0) == list(range(20)) and rt.pages_available() == 260
    finally:
        stop.set()
        t.join()


def test_arguments_that_ask_for_pages(rt, monkeypatch):
    """A call's slots may come from an iterator that asks which slots are empty."""
    monkeypatch.setattr(rt, "_page_work", lambda what, plan, *args: plan(rt._pages[0], *args), raising=False)
    rt._pages[0].reserve([(0, 0, 20), (2, 0, 1)])
    done = threading.Thread(target=lambda: rt.pages_fork(0, (s for s in range(4) if not rt.pages_of(s)), 20), daemon=True)
    done.start()
    done.join(20)
    assert not done.is_alive() and [len(rt.pages_of(s)) for s in range(4)] == [20, 20, 1, 20]
