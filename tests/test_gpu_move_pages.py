"""vq_move_pages: every entry of the page table, and pages whose bytes lie past 32 bits."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from vinf_3080ti_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    t = pytest.importorskip("torch")
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


def move(torch, pools, sizes, pages, copies, table, entries):
    n = len(pools)
    c, e = (np.ascontiguousarray(a, np.int32).reshape(-1, 2) for a in (copies, entries))
    st = _lib.load().vq_move_pages((ctypes.c_void_p * n)(*[p.data_ptr() for p in pools]), (ctypes.c_size_t * n)(*sizes), n, pages,
                                   c.ctypes.data, len(c), table.data_ptr() if len(e) else None, table.numel() if len(e) else 0,
                                   e.ctypes.data, len(e), torch.cuda.current_stream().cuda_stream)
    assert st == 0


@pytest.mark.parametrize("npools", [0, 1, 33])
@pytest.mark.parametrize("ncopies,nentries", [(0, 1), (0, 192), (0, 193), (0, 600), (5, 600), (192, 385), (400, 200)])
def test_every_entry_is_written(torch, npools, ncopies, nentries):
    """As many as one launch takes, one more, several launches' worth, beside more and fewer copies and pools than one takes."""
    rng = np.random.default_rng(nentries + ncopies)
    pages, size = 900, 64
    pools = [torch.randint(0, 256, (pages * size,), dtype=torch.uint8, device="cuda") for _ in range(npools)]
    ids = rng.permutation(pages)
    copies = np.stack([ids[400:400 + ncopies], ids[:ncopies]], 1)
    entries = np.stack([rng.permutation(700)[:nentries], rng.integers(-5, 2 ** 31 - 1, nentries)], 1)
    table = torch.full((700,), -3, dtype=torch.int32, device="cuda")
    want = np.full(700, -3)
    want[entries[:, 0]] = entries[:, 1]
    held = [p.cpu().numpy().reshape(pages, size).copy() for p in pools]
    move(torch, pools, [size] * npools, pages, copies, table, entries)
    assert np.array_equal(table.cpu().numpy(), want)
    for p, h in zip(pools, held):
        h[copies[:, 1]] = h[copies[:, 0]]
        assert np.array_equal(p.cpu().numpy().reshape(pages, size), h)


@pytest.mark.parametrize("size", [1 << 20, (1 << 20) + 2, (1 << 19) + 1])
def test_pages_past_4_gib(torch, size):
    """A page moved from the low end to the far one and another back, in pieces of 16 bytes, of two and of one."""
    pages = (1 << 32) // size + 40
    pool = torch.zeros(pages * size, dtype=torch.uint8, device="cuda")
    view = pool.view(pages, size)
    low, high, mid = 1, pages - 1, pages - 20  # high and mid begin past 2^32
    assert mid * size > 1 << 32
    view[low] = torch.randint(0, 256, (size,), dtype=torch.uint8, device="cuda")
    view[mid] = torch.randint(0, 256, (size,), dtype=torch.uint8, device="cuda")
    a, b = view[low].clone(), view[mid].clone()
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    move(torch, [pool], [size], pages, [(low, high), (mid, 3)], none, np.zeros((0, 2)))
    assert torch.equal(view[high], a) and torch.equal(view[3], b) and torch.equal(view[low], a) and torch.equal(view[mid], b)
    move(torch, [pool], [size], pages, [(high, 0), (3, high - 1)], none, np.zeros((0, 2)))
    assert torch.equal(view[0], a) and torch.equal(view[high - 1], b)
    written = {0, low, 3, mid, high - 1, high}
    assert all(p in written or not bool(view[p].any()) for p in (2, 4, mid - 1, mid + 1, high - 2, (pages - 1) % ((1 << 32) // size)))
