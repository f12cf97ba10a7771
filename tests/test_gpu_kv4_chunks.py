"""Attention over the 4-bit cache in contexts that are cut into many chunks: both ways of merging them, against the float64 oracle.
How many chunks a pass has is read off its workspace, so that a change of the rule cannot leave a way untested."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
from test_gpu_kv4 import caches, get, put, put_ints

from vinf_3080ti_amd import _lib

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


def rows_of(rng, n, kvh, hd):
    """K whose every 97th position points where the queries do (a score of 6, the others' are near 0), V of one size: a chunk that is
    lost or counted twice moves the result by its share of those keys."""
    along = np.where(np.arange(hd) % 3 == 0, -1.0, 1.0)
    k = rng.standard_normal((n, kvh, hd)) * 0.3
    k[rng.integers(97)::97] += 2 * along
    return k.astype(np.float32), rng.uniform(-1, 1, (n, kvh, hd)).astype(np.float32)


def queries(rng, rows, heads, hd):
    along = np.where(np.arange(hd) % 3 == 0, -1.0, 1.0)
    return (rng.standard_normal((rows, heads, hd)) * 0.3 + along * 3 / np.sqrt(hd)).astype(np.float32)


def check(got, q, k, v, heads, kvh, seq_len, oracle_mod, window=0):
    """Of a result of values up to max |v|: twice a score's error e, in numerator and denominator, the weights' 2^-23, and one
    rounding for each of a wave's terms (n / 4 keys in two halves at most) and of 64 + 160 joins of waves and chunks."""
    n = k.shape[1]
    want = oracle_mod.attention(q, k, v, heads, kvh, seq_len, False, window)
    for h in range(heads):
        size = (np.abs(q[:, h].astype(np.float64)) @ np.abs(k[h * kvh // heads]).T).max(1) / np.sqrt(q.shape[2])
        e = (q.shape[2] + 8) * 2.0 ** -24 * size
        off = np.abs(got[:, h] - want[:, h]).max(1)
        assert (off <= 2 * np.abs(v).max() * (2 * e + 2.0 ** -23 + (n / 2 + 224) * 2.0 ** -24)).all(), (h, off.max())


def chunks(heads, kvh, hd, seq_len, ntok, window=0):
    return (_lib.load().vq_attention4_workspace_bytes(heads, kvh, hd, seq_len, ntok, window) - 16) / ((hd + 2) * 4 * ntok * heads)


def one_pass(rt, oracle_mod, heads, kvh, hd, n, ntok, window):
    rng = np.random.default_rng(n + hd + ntok)
    k, v = rows_of(rng, n, kvh, hd)
    caches(rt, kvh, n, hd)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append("k", "v", "kc", "vc", kvh, n, hd, 0, n)
    wk, wv = (x.transpose(1, 0, 2) for x in oracle_mod.kv4_values(k, v))
    q = queries(rng, ntok, heads, hd)
    put(rt, "q", q)
    put(rt, "o", np.full(q.size + 4, 3.0))
    rt.attention("q", "kc", "vc", "o", heads, kvh, hd, n, n - ntok + 1, ntok, 0, window)
    got = get(rt, "o", -1)
    assert (got[q.size:] == 3.0).all()
    check(got[: q.size].reshape(q.shape), q, wk, wv, heads, kvh, n - ntok + 1, oracle_mod, window)


SHAPES = [(24, 4, 256), (32, 8, 128), (6, 2, 96), (5, 5, 32), (64, 8, 64), (8, 1, 160), (3, 1, 224), (40, 2, 192)]


@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
@pytest.mark.parametrize("n,ntok,window", [(1200, 1, 0), (6000, 1, 0), (3000, 4, 0), (6000, 17, 0), (9001, 2, 4000), (6000, 19, 3001),
                                           (20000, 1, 0)])
def test_many_chunks(rt, oracle_mod, heads, kvh, hd, n, ntok, window):
    """Chunks merged by (row, head): from 10 to 157 of them, decode, verified rows, prompts and windows."""
    most = chunks(heads, kvh, hd, n - ntok + 1, ntok, window)
    assert most > 8 and (most > 32 or ntok * heads * hd < 1 << 18)
    one_pass(rt, oracle_mod, heads, kvh, hd, n, ntok, window)


@pytest.mark.parametrize("heads,kvh,hd,n,ntok,window", [(24, 4, 256, 1200, 64, 0), (24, 4, 256, 6000, 50, 0), (16, 2, 256, 6000, 70, 0),
                                                        (24, 4, 256, 5000, 64, 3001), (14, 2, 224, 3000, 90, 0)])
def test_up_to_32_chunks_of_many_rows(rt, oracle_mod, heads, kvh, hd, n, ntok, window):
    """Chunks merged by rows."""
    assert 8 < chunks(heads, kvh, hd, n - ntok + 1, ntok, window) <= 32 and ntok * heads * hd >= 1 << 18
    one_pass(rt, oracle_mod, heads, kvh, hd, n, ntok, window)


@pytest.mark.parametrize("heads,kvh,hd,page", [(24, 4, 256, 64), (32, 8, 128, 16), (64, 8, 64, 8), (6, 2, 96, 24), (32, 8, 128, 24)])
@pytest.mark.parametrize("segments", [[(0, 7999, 1), (1, 0, 1), (2, 2990, 2), (3, 700, 1)], [(2, 5000, 2), (0, 7980, 20), (1, 3, 1), (3, 6400, 3)]])
def test_segments_of_mixed_length(rt, oracle_mod, heads, kvh, hd, page, segments):
    """One key to 8000 in one pass over pages: every segment has its own number of chunks."""
    rng = np.random.default_rng(page * hd)
    per, slots = -(-8000 // page), 4
    put_ints(rt, "pt", rng.permutation(per * slots).reshape(slots, per))
    rt.set_paging("pt", page, per, slots)
    caches(rt, per * slots * kvh, page, hd)
    held = {}
    for slot, pos0, rows in segments:
        k, v = rows_of(rng, pos0 + rows, kvh, hd)
        rt.set_segments([(slot, 0, pos0 + rows)])
        put(rt, "k", k)
        put(rt, "v", v)
        rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
        held[slot] = [w.transpose(1, 0, 2) for w in oracle_mod.kv4_values(k, v)]
    n = rt.set_segments(segments)
    flat = (ctypes.c_int32 * (4 * len(segments)))(*[x for s in segments for x in (*s, 0)])
    parts = (_lib.load().vq_attention4_seg_workspace_bytes(flat, len(segments), heads, kvh, hd) - 16) / ((hd + 2) * 4 * heads)
    assert parts > 8 * n  # the mean over the rows: the longest segment has more than that
    q = queries(rng, n, heads, hd)
    put(rt, "q", q)
    put(rt, "o", np.zeros(q.size))
    rt.attention_seg("q", "kc", "vc", "o", heads, kvh, hd)
    got, row = get(rt, "o", q.shape), 0
    for slot, pos0, rows in segments:
        check(got[row:row + rows], q[row:row + rows], *held[slot], heads, kvh, pos0 + 1, oracle_mod)
        row += rows
