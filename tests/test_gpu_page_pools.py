"""What the runtime's page calls are given: pools and tables that changed since they were named."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    t = pytest.importorskip("torch")
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


@pytest.fixture
def rt(torch):
    from vinf_3080ti_amd.runtime import HipWeightRuntime

    rt = HipWeightRuntime()
    rt.alloc("table", 8)
    rt.set_paging("table", 8, 4, 2)
    rt.alloc("h", 4 * 2 * 8 * 32, 2)
    rt.alloc_kv4("q", 4 * 2, 8, 32)
    rt.set_page_pools(["h", "q"], 4)
    rt.pages_reserve([(0, 0, 20)])
    return rt


@pytest.mark.parametrize("change", [lambda r: r.alloc("h", 4 * 2 * 8 * 32), lambda r: r.alloc("h", 4 * 4 * 8 * 32, 2),
                                    lambda r: r.alloc("h", 4 * 2 * 8 * 32 - 4, 2), lambda r: r.alloc("h", 2 * 2 * 8 * 32),
                                    lambda r: r.alloc_kv4("q", 4 * 4, 8, 32), lambda r: r.alloc_kv4("q", 4 * 2, 8, 64),
                                    lambda r: r.alloc_kv4("q", 4, 16, 32), lambda r: r.alloc("q", 4 * 2 * 8 * 32, 2),
                                    lambda r: r.alloc_kv4("h", 4 * 2, 8, 32)])
def test_a_pool_of_another_layout_is_refused(rt, change):
    """Grown, shrunk, in another precision or of another shape, also of the same bytes: its pages are elsewhere."""
    change(rt)
    for call in (lambda: rt.pages_reserve([(1, 0, 1)]), lambda: rt.pages_fork(0, [1], 20), lambda: rt.pages_copy([(0, 1, 8)]),
                 lambda: rt.pages_free([0]), lambda: rt.pages_compact()):
        with pytest.raises(ValueError):
            call()
    assert rt.pages_of(0) == [0, 1, 2] and rt.pages_of(1) == []
    rt.alloc("h", 4 * 2 * 8 * 32, 2)
    rt.alloc_kv4("q", 4 * 2, 8, 32)
    rt.pages_fork(0, [1], 20)
    assert rt.pages_of(1) == [0, 1, 2]


def test_a_pool_in_another_storage_is_followed(rt, torch):
    """A lent pool whose storage is exchanged for one of the same size: the copies go there; of another size: refused."""
    for name in ("h", "q"):
        t = rt.buffer_tensor(name)
        t.data = torch.arange(t.numel(), device="cuda").remainder(113).to(t.dtype)
    rt.pages_fork(0, [1], 20)
    rt.pages_reserve([(1, 17, 1)])  # page 2 goes to page 3
    assert rt.pages_of(1) == [0, 1, 3]
    for name in ("h", "q"):
        t = rt.buffer_tensor(name).view(4, -1)
        assert torch.equal(t[3], t[2]) and bool((t[2] != 0).any())
    t = rt.buffer_tensor("h")
    t.data = torch.zeros(2 * t.numel(), dtype=t.dtype, device="cuda")
    with pytest.raises(ValueError):
        rt.pages_free([0])
    t = rt.buffer_tensor("h")
    t.data = torch.zeros(4 * 2 * 8 * 32, dtype=t.dtype, device="cuda")
    t = rt.buffer_tensor("q")
    t.data = torch.zeros(t.numel() - 16, dtype=t.dtype, device="cuda")
    with pytest.raises(ValueError):
        rt.pages_free([0])
    assert rt.pages_of(0) == [0, 1, 2]


def test_a_table_in_a_smaller_storage_is_refused(rt, torch):
    """A lent page table whose storage is exchanged for a smaller one: no entry is written or read behind it."""
    for name in ("k", "v", "x", "o"):
        rt.alloc(name, 2 * 2 * 32)
    rt.set_segments([(0, 18, 2)])
    t = rt.buffer_tensor("table")
    held = t.data
    t.data = torch.zeros(7, device="cuda")
    for call in (lambda: rt.pages_fork(0, [1], 20), lambda: rt.pages_free([0]), lambda: rt.kv_append_seg("k", "v", "q", "q", 2, 32),
                 lambda: rt.kv4_read_seg("q", "q", "k", "v", 2, 32), lambda: rt.attention_seg("x", "q", "q", "o", 2, 2, 32),
                 lambda: rt.attention_seg("x", "h", "h", "o", 2, 2, 32)):
        for _ in range(2):
            with pytest.raises(ValueError):
                call()
    assert rt.pages_of(0) == [0, 1, 2] and rt.pages_of(1) == []
    rt.buffer_tensor("table").data = held
    rt.pages_fork(0, [1], 20)
    assert rt.pages_of(1) == [0, 1, 2]


@pytest.mark.parametrize("blocks,positions,pages", [(10, 8, 4), (9, 8, 2), (4, 16, 4), (2, 8, 4)])
def test_a_4_bit_pool_that_is_not_whole_pages_is_refused(rt, blocks, positions, pages):
    """Its bytes may divide by the pages all the same: 10 blocks of 144 bytes make 4 times 360."""
    rt.alloc_kv4("p", blocks, positions, 32)
    with pytest.raises(ValueError):
        rt.set_page_pools(["p"], pages)
