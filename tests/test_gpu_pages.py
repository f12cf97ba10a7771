"""Page work on the GPU: the runtime's pages_* calls over fp32, fp16 and 4-bit pools against a model that keeps every sequence apart,
and the device entry point over odd page sizes, many pools and many pages."""
from __future__ import annotations

import ctypes
import random

import numpy as np
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

    return HipWeightRuntime()


@pytest.mark.parametrize("sizes,offset", [((4096,), 0), ((48, 16 * 1025, 65536 * 3 + 16), 0), ((6, 34), 0), ((7, 1), 0), ((64,), 2),
                                          ((64, 5), 1), (tuple([160] * 37), 0)])
@pytest.mark.parametrize("ncopies,nentries", [(1, 0), (0, 5), (3, 200), (200, 3), (450, 600)])
def test_move_pages(torch, sizes, offset, ncopies, nentries):
    """Pages of any size, aligned or not, more pools, copies and entries than one launch takes; everything else untouched."""
    from vinf_3080ti_amd import _lib

    lib, rng = _lib.load(), np.random.default_rng(ncopies + nentries)
    pages = 1000 if max(sizes) < 100000 else 460 if ncopies < 400 else 910
    ids = rng.permutation(pages)
    dst = ids[:ncopies]
    src = rng.choice(ids[ncopies:], ncopies)  # a page may be read more than once
    copies = np.stack([src, dst], 1).astype(np.int32).copy()
    entries = np.stack([rng.permutation(700)[:nentries], rng.integers(0, pages, nentries)], 1).astype(np.int32).copy()
    pools = [torch.randint(0, 256, (offset + pages * s + 9,), dtype=torch.uint8, device="cuda") for s in sizes]
    table = torch.full((705,), -3, dtype=torch.int32, device="cuda")
    want = [p.clone() for p in pools]
    for w, s in zip(want, sizes):
        v = w[offset:offset + pages * s].view(pages, s)
        v[torch.from_numpy(dst).cuda()] = v[torch.from_numpy(src).cuda()]
    n = len(sizes)
    st = lib.vq_move_pages((ctypes.c_void_p * n)(*[p.data_ptr() + offset for p in pools]), (ctypes.c_size_t * n)(*sizes), n, pages,
                           copies.ctypes.data, ncopies, table.data_ptr(), 700, entries.ctypes.data, nentries,
                           torch.cuda.current_stream().cuda_stream)
    assert st == 0
    copies[:], entries[:] = -9, -9  # read before the call returned
    for p, w in zip(pools, want):
        assert torch.equal(p, w)
    t = torch.full((705,), -3, dtype=torch.int32)
    st = lib.vq_move_pages(None, None, 0, 0, None, 0, None, 0, None, 0, None)
    assert st == 0 and (table.cpu()[700:] == t[700:]).all()


@pytest.mark.parametrize("seed", range(4))
def test_pages_follow_their_sequences(rt, torch, seed):
    """A random walk of reserve and append, fork, copy, free and compact over an fp32, an fp16 and a pair of 4-bit pools: what a slot
    reads back through the page table is what it was given, whatever the other slots did."""
    rng, npr = random.Random(seed), np.random.default_rng(seed)
    page, per, slots, pages, kvh, hd = 8, 5, 6, 24, 2, 32
    rt.alloc("table", slots * per)
    rt.set_paging("table", page, per, slots)
    rt.alloc("k32", pages * kvh * page * hd)
    rt.alloc("v32", pages * kvh * page * hd)
    rt.alloc("k16", pages * kvh * page * hd, 2)
    rt.alloc("v16", pages * kvh * page * hd, 2)
    rt.alloc_kv4("k4", pages * kvh, page, hd)
    rt.alloc_kv4("v4", pages * kvh, page, hd)
    rt.set_page_pools(["k32", "v32", "k16", "v16", "k4", "v4"], pages)
    for name in ("k", "v", "rk", "rv"):
        rt.alloc(name, per * page * kvh * hd)
    # Values that all three precisions hold exactly: groups whose span is 15 steps.
    model = [np.zeros((0, kvh, hd), np.float32) for _ in range(slots)]

    def fresh(n):
        x = npr.integers(-7, 9, (n, kvh, hd)).astype(np.float32)
        x[..., 0], x[..., 1] = -7, 8
        return x

    for step in range(120):
        op, s = rng.randrange(6), rng.randrange(slots)
        try:
            if op <= 1:
                pos0 = rng.randint(0, len(model[s]))
                n = rng.randint(1, 2 * page)
                rt.pages_reserve([(s, pos0, n)])
                x = fresh(n)
                rt.write("k", x.tobytes())
                rt.write("v", x.tobytes())
                rt.set_segments([(s, pos0, n)])
                for b in ("32", "16", "4"):
                    rt.kv_append_seg("k", "v", "k" + b, "v" + b, kvh, hd)
                model[s] = np.concatenate([model[s][:pos0], x, model[s][pos0 + n:]])
            elif op == 2:
                n, to = rng.randint(0, len(model[s])), [t for t in range(slots) if t != s and rng.random() < 0.3]
                rt.pages_fork(s, to, n)
                for t in to:
                    model[t] = model[s][:n]
            elif op == 3:
                t, n = rng.randrange(slots), rng.randint(0, len(model[s]))
                rt.pages_copy([(s, t, n)])
                model[t] = model[s][:n]
            elif op == 4:
                n = rng.randint(0, len(model[s]))
                rt.pages_free([s], n)
                model[s] = model[s][:n]
            else:
                rt.pages_compact()
        except ValueError:
            pass
        table = np.frombuffer(rt.read("table"), np.int32).reshape(slots, per)
        pools = {b: np.frombuffer(rt.read("k" + b), np.float32 if b == "32" else np.float16).reshape(pages, kvh, page, hd)
                 for b in ("32", "16")}
        for t in range(slots):
            n = len(model[t])
            held = rt.pages_of(t)
            assert len(held) == -(-n // page) and table[t, :len(held)].tolist() == held
            if not n:
                continue
            for b, pool in pools.items():
                got = pool[held].transpose(0, 2, 1, 3).reshape(-1, kvh, hd)[:n]
                assert np.array_equal(got, model[t]), (step, t, b)
            rt.set_segments([(t, 0, n)])
            rt.kv4_read_seg("k4", "v4", "rk", "rv", kvh, hd)
            for name in ("rk", "rv"):
                assert np.array_equal(np.frombuffer(rt.read(name, n * kvh * hd), np.float32).reshape(n, kvh, hd), model[t]), (step, t)


def test_runtime_contract(rt, torch):
    with pytest.raises(RuntimeError):
        rt.set_page_pools(["a"], 4)
    rt.alloc("table", 8)
    rt.set_paging("table", 8, 4, 2)
    for call in (lambda: rt.pages_reserve([(0, 0, 1)]), lambda: rt.pages_free([0]), lambda: rt.pages_compact(), lambda: rt.pages_of(0),
                 lambda: rt.pages_available()):
        with pytest.raises(RuntimeError):
            call()
    rt.alloc("a", 100)
    rt.alloc("b", 64, 2)
    for bad in ((["a"], 3), (["a"], 0), (["a"], -1), (["a", "a"], 4), ("a", 4), (["b"], 2 ** 31)):
        with pytest.raises(ValueError):
            rt.set_page_pools(*bad)
    with pytest.raises(KeyError):
        rt.set_page_pools(["none"], 4)
    rt.set_page_pools(["a", "b"], 4)
    rt.pages_reserve([(0, 0, 20)])
    assert rt.pages_of(0) == [0, 1, 2] and rt.pages_available() == 1
    rt.pages_fork(0, [1], 20)
    with pytest.raises(ValueError):
        rt.pages_reserve([(1, 0, 20)])  # three copies, one page
    with pytest.raises(ValueError):
        rt.pages_of(2)
    rt.set_paging("table", 8, 4, 2)  # the same again: the book stays
    assert rt.pages_of(1) == [0, 1, 2]
    rt.alloc("b", 30, 2)
    with pytest.raises(ValueError):  # a pool that has shrunk
        rt.pages_reserve([(1, 20, 1)])
    assert rt.pages_of(1) == [0, 1, 2]
    rt.alloc("b", 64, 2)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError):
            rt.pages_reserve([(1, 20, 1)])
        rt.zero("a")
    assert rt.pages_of(1) == [0, 1, 2]
    rt.set_paging("table", 4, 4, 2)
    with pytest.raises(RuntimeError):
        rt.pages_free([0])
