"""The 4-bit KV cache on the GPU, through the runtime: what append writes bit for bit, what comes back, and attention over it against
the float64 oracle on the values that the cache holds."""
from __future__ import annotations

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


def put(rt, name: str, a) -> None:
    a = np.ascontiguousarray(a, np.float32).reshape(-1)
    rt.alloc(name, a.size)
    rt.write(name, a.tobytes())


def get(rt, name: str, shape) -> np.ndarray:
    return np.frombuffer(rt.read(name), np.float32).reshape(shape)


def put_ints(rt, name: str, a) -> None:
    a = np.ascontiguousarray(a, np.int32).reshape(-1)
    rt.alloc(name, a.size)
    rt.write(name, a.tobytes())


def keys(rng, *shape):
    """K with a few dims many times larger than the others."""
    return (rng.standard_normal(shape) * np.where(rng.random(shape[-1]) < 0.05, 7.0, 0.8)).astype(np.float32)


def caches(rt, kv_blocks, positions, hd):
    for name in ("kc", "vc"):
        rt.alloc_kv4(name, kv_blocks, positions, hd)


def blocks(rt, name):
    b = rt.buffers[name].kv4
    return np.frombuffer(rt.read(name), np.uint8).reshape(b[0], -1)


# ---- append and read-back -------------------------------------------------------------------------------------


@pytest.mark.parametrize("hd,kvh,max_seq,cuts", [(256, 4, 64, (0, 1, 2, 9, 40, 64)), (128, 1, 40, (0, 8, 16, 40)), (64, 3, 21, (0, 21)),
                                                 (96, 2, 30, (0, 3, 4, 29, 30)), (32, 5, 17, (0, 7, 17)), (224, 1, 9, (0, 5, 9)),
                                                 (160, 2, 16, (0, 15, 16)), (192, 2, 12, (0, 4, 12))])
def test_append_writes_the_documented_bytes(rt, oracle_mod, hd, kvh, max_seq, cuts):
    """A contiguous cache filled pass by pass (cuts inside and at the ends of slabs): the bytes of the layout, zeros past the last
    position; what is read back is what the bytes stand for."""
    rng = np.random.default_rng(hd + max_seq)
    k, v = keys(rng, max_seq, kvh, hd), rng.standard_normal((max_seq, kvh, hd)).astype(np.float32)
    caches(rt, kvh, max_seq, hd)
    for a, b in zip(cuts, cuts[1:]):
        put(rt, "k", k[a:b])
        put(rt, "v", v[a:b])
        rt.kv_append("k", "v", "kc", "vc", kvh, max_seq, hd, a, b - a)
    full = -(-max_seq // 8) * 8
    for name, x, values in (("kc", k, False), ("vc", v, True)):
        got = blocks(rt, name)
        for h in range(kvh):
            row = np.zeros((full, hd), np.float32)
            row[:max_seq] = x[:, h]
            assert np.array_equal(got[h], oracle_mod.kv4_block(row, values)), (name, h)
    a, n = max_seq // 3, max_seq - max_seq // 3
    for name in ("rk", "rv"):
        put(rt, name, np.full((n + 1, kvh, hd), 9.0))
    rt.kv4_read("kc", "vc", "rk", "rv", kvh, max_seq, hd, a, n)
    want = oracle_mod.kv4_values(k[a:], v[a:])
    for name, w in zip(("rk", "rv"), want):
        got = get(rt, name, (n + 1, kvh, hd))
        assert np.array_equal(got[:n], w.astype(np.float32)) and (got[n] == 9.0).all()


def test_append_values_at_the_edges(rt, oracle_mod):
    """Exact ties, groups of one sign, zeros, the smallest and largest magnitudes, values past the largest scale, values that are
    not finite; a rewritten position."""
    hd, rng = 64, np.random.default_rng(3)
    rows = []
    rows.append(np.tile(np.arange(16) / 2 - 3.5, 4) * 0.75)  # halves of a step: ties
    rows.append(np.abs(rng.standard_normal(hd)) + 4)
    rows.append(-np.abs(rng.standard_normal(hd)) - 4)
    rows.append(np.zeros(hd))
    rows.append(np.r_[rng.standard_normal(32) * 1e-6, rng.standard_normal(32) * 1e-42])
    rows.append(np.r_[rng.standard_normal(32) * 30000, rng.standard_normal(32) * 1e30])
    rows.append(np.r_[np.full(32, 3.0e38), np.full(32, -3.0e38)])
    rows.append(np.r_[np.linspace(-65280, 65280, 32), np.linspace(0, 65280, 32)])
    rows.append(np.r_[np.full(31, 1e-45), 0, np.full(32, 2.0 ** -20 * 7.5)])
    rows += [x for x in rng.standard_normal((64, hd)) * np.exp2(rng.integers(-30, 14, (64, 1)))]
    grid = rng.integers(-7, 9, (200, hd)) + rng.choice([0, 0.5], (200, hd))  # more ties, on many scales
    rows += [x for x in grid * np.exp2(rng.integers(-18, 8, (200, 1))) * rng.integers(64, 128, (200, 1))]
    x = np.array(rows, np.float32)
    n = len(x)
    k, v = x[:, None].repeat(2, 1), x[::-1, None].repeat(2, 1).copy()
    k[20, 0, 5], v[21, 1, 63], k[22, 1, 0], v[23, 0, 8] = np.inf, np.nan, np.nan, -np.inf
    caches(rt, 2, n, hd)
    put(rt, "k", k[::-1])
    put(rt, "v", v)
    rt.kv_append("k", "v", "kc", "vc", 2, n, hd, 0, n)  # overwritten by the next call
    put(rt, "k", k)
    rt.kv_append("k", "v", "kc", "vc", 2, n, hd, 0, n)
    put(rt, "rk", np.zeros(n * 2 * hd))
    put(rt, "rv", np.zeros(n * 2 * hd))
    rt.kv4_read("kc", "vc", "rk", "rv", 2, n, hd, 0, n)
    for name, w in zip(("rk", "rv"), oracle_mod.kv4_values(k, v)):
        got = get(rt, name, k.shape)
        bad = ~((got == w.astype(np.float32)) | (np.isnan(got) & np.isnan(w)))
        assert not bad.any(), np.argwhere(bad)[:5]


@pytest.mark.parametrize("page,kvh,hd", [(8, 2, 64), (16, 4, 256), (24, 1, 96), (64, 2, 128)])
def test_append_seg_into_pages(rt, oracle_mod, page, kvh, hd):
    """Segments of several slots, two of them one after the other in one slot and meeting inside a slab, one placed behind a gap:
    their positions are written, every other byte of the pool stays."""
    rng = np.random.default_rng(page * hd)
    pps, slots = 6, 4
    table = rng.permutation(pps * slots + 3)[: pps * slots].reshape(slots, pps).astype(np.int32)
    put_ints(rt, "pt", table)
    rt.set_paging("pt", page, pps, slots)
    caches(rt, (pps * slots + 3) * kvh, page, hd)
    held = {}
    for name, values in (("kc", False), ("vc", True)):  # something valid everywhere
        x = rng.standard_normal(((pps * slots + 3) * kvh, page, hd)).astype(np.float32)
        raw = np.stack([oracle_mod.kv4_block(b, values) for b in x])
        rt.write(name, raw.tobytes())
        held[name] = np.stack([oracle_mod.kv4_values(b, b)[0] for b in x])
    segments = [(2, 3, 10), (0, page - 1, page + 3), (2, 13, 4), (3, 5, 1, 2 * page + 40), (1, 0, 9)]
    n = rt.set_segments(segments)
    k, v = keys(rng, n, kvh, hd), rng.standard_normal((n, kvh, hd)).astype(np.float32)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
    wk, wv = oracle_mod.kv4_values(k, v)
    row, want = 0, {name: held[name].copy() for name in held}
    for slot, pos0, rows, *at in segments:
        row = at[0] if at else row
        for t in range(rows):
            pg = table[slot, (pos0 + t) // page]
            for h in range(kvh):
                want["kc"][pg * kvh + h, (pos0 + t) % page] = wk[row + t, h]
                want["vc"][pg * kvh + h, (pos0 + t) % page] = wv[row + t, h]
        row += rows
    # The bytes, by what they stand for: values on a scale's grid are their own rounding.
    for name, values in (("kc", False), ("vc", True)):
        got = blocks(rt, name)
        for b in range(got.shape[0]):
            assert np.array_equal(values_of(got[b], page, hd, values), want[name][b]), (name, b)
    put(rt, "rk", np.full(k.size, 5.0))
    put(rt, "rv", np.full(k.size, 5.0))
    rt.kv4_read_seg("kc", "vc", "rk", "rv", kvh, hd)
    used = np.zeros(n, bool)
    row = 0
    for slot, pos0, rows, *at in segments:
        row = at[0] if at else row
        used[row:row + rows] = True
        row += rows
    for name, w in (("rk", wk), ("rv", wv)):
        got = get(rt, name, k.shape)
        assert np.array_equal(got[used], w[used].astype(np.float32)) and (got[~used] == 5.0).all()


def values_of(raw, page, hd, values):
    """float64 [page][hd] of a block's bytes."""
    words, heads = raw[: page * hd // 2].view(np.uint32), raw[page * hd // 2:].view(np.uint16)
    pos, dim = np.arange(page)[:, None], np.arange(hd)
    w = 4 if hd % 64 == 0 else 2
    if values:
        at, e = (pos // 8) * hd + (dim // (16 * w) * 16 + dim % 16) * w + dim // 16 % w, pos % 8 + 0 * dim
        head = heads[((pos // 8) * (hd // 32) + dim // 32) * 8 + pos % 8]
    else:
        at, e = pos * hd // 8 + (dim % 32 // 8) * (hd // 32) + dim // 32, dim % 8 + 0 * pos
        head = heads[pos * (hd // 32) + dim // 32]
    code = (words[at] >> (4 * (e // 2) + 16 * (e % 2)).astype(np.uint32)) & 15
    return (head & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64) * (code.astype(float) - (head & 15))


def test_wrong_pages_are_not_followed(rt):
    """Entries of the page table that are no pages: nothing is written through them, their positions read as NaN, attention over
    them gives NaN and over the others what it gives without them."""
    page, kvh, hd, heads = 16, 2, 64, 4
    put_ints(rt, "pt", [1, -1, 0, 7, 2, 3])
    rt.set_paging("pt", page, 3, 2)
    caches(rt, 4 * kvh, page, hd)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((64, kvh, hd)).astype(np.float32)
    put(rt, "k", x)
    put(rt, "v", x)
    rt.set_segments([(0, 0, 16), (1, 16, 32)])
    rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
    before = blocks(rt, "kc").copy(), blocks(rt, "vc").copy()
    rt.set_segments([(0, 16, 16), (1, 0, 16)])
    rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
    assert np.array_equal(before[0], blocks(rt, "kc")) and np.array_equal(before[1], blocks(rt, "vc"))
    for name in ("rk", "rv"):
        put(rt, name, np.zeros(x.size))
    rt.kv4_read_seg("kc", "vc", "rk", "rv", kvh, hd)
    assert np.isnan(get(rt, "rk", x.shape)[:32]).all()
    q = rng.standard_normal((20, heads, hd)).astype(np.float32)
    put(rt, "q", q)
    for rows in (2, 18):
        put(rt, "o", np.zeros(q.size))
        rt.set_segments([(0, 16 - rows // 2, rows), (0, 10, 2, 18)])
        rt.attention_seg("q", "kc", "vc", "o", heads, kvh, hd)
        o = get(rt, "o", q.shape)
        assert np.isfinite(o[:rows // 2]).all() and np.isnan(o[rows // 2:rows]).all() and np.isfinite(o[18:20]).all()


# ---- attention ------------------------------------------------------------------------------------------------


def bound(q, k, v, heads, kvh, seq_len, bidirectional, window):
    """How far fp32 sums of products with 22-bit query and weight pairs may be from the exact result, per (row, head): a score's
    error is at most e = (hd + 8) 2^-24 sum |q k| / sqrt(hd), a weight's relative one 2 e more than the sums' own (n + 64) 2^-24,
    of values up to max |v|; both numerator and denominator have it."""
    ntok, _, hd = q.shape
    out = np.zeros((ntok, heads, 1))
    for t in range(ntok):
        end = seq_len + (ntok - 1 if bidirectional else t)
        start = max(0, seq_len + t - window) if window else 0
        for h in range(heads):
            kk, vv = np.abs(k[h * kvh // heads, start:end]), np.abs(v[h * kvh // heads, start:end])
            e = (hd + 8) * 2.0 ** -24 * (kk @ np.abs(q[t, h].astype(np.float64))).max() / np.sqrt(hd)
            out[t, h] = 2 * vv.max() * (2 * e + (end - start + 64) * 2.0 ** -24)
    return out


def check(got, q, k, v, heads, kvh, seq_len, oracle_mod, bidirectional=0, window=0):
    want = oracle_mod.attention(q, k, v, heads, kvh, seq_len, bool(bidirectional), window)
    off = np.abs(got - want)
    assert (off <= bound(q, k, v, heads, kvh, seq_len, bidirectional, window)).all(), off.max()


def fill(rt, oracle_mod, rng, kvh, max_seq, hd):
    """Contiguous 4-bit caches of random rows; returns what they hold, [kvh][max_seq][hd]."""
    k, v = keys(rng, max_seq, kvh, hd), rng.standard_normal((max_seq, kvh, hd)).astype(np.float32)
    caches(rt, kvh, max_seq, hd)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append("k", "v", "kc", "vc", kvh, max_seq, hd, 0, max_seq)
    wk, wv = oracle_mod.kv4_values(k, v)
    return wk.transpose(1, 0, 2), wv.transpose(1, 0, 2)


SHAPES = [(24, 4, 256), (32, 8, 128), (5, 5, 32), (6, 2, 96), (64, 8, 64), (8, 1, 160), (40, 2, 192), (3, 1, 224)]


@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
@pytest.mark.parametrize("ntok,seq_len,bidirectional,window", [(1, 1, 0, 0), (1, 33, 0, 0), (2, 300, 0, 0), (8, 130, 0, 0), (3, 90, 1, 0),
                                                               (1, 500, 0, 100), (7, 200, 0, 5), (40, 1, 0, 0), (19, 71, 0, 30),
                                                               (33, 100, 1, 0), (17, 17, 1, 9)])
def test_attention(rt, oracle_mod, heads, kvh, hd, ntok, seq_len, bidirectional, window):
    """Decode, verify and prompt passes over a contiguous cache, causal, windowed and bidirectional, one key to several hundred,
    with and without a workspace (batch-invariant mode)."""
    rng = np.random.default_rng(heads * hd + 7 * ntok + seq_len)
    max_seq = seq_len + ntok + 3
    k, v = fill(rt, oracle_mod, rng, kvh, max_seq, hd)
    q = rng.standard_normal((ntok, heads, hd)).astype(np.float32)
    put(rt, "q", q)
    for invariant in (False, True):
        rt.set_batch_invariant(invariant)
        put(rt, "o", np.full(q.size + 4, 3.0))
        rt.attention("q", "kc", "vc", "o", heads, kvh, hd, max_seq, seq_len, ntok, bidirectional, window)
        got = get(rt, "o", -1)
        assert (got[q.size:] == 3.0).all()
        check(got[: q.size].reshape(q.shape), q, k, v, heads, kvh, seq_len, oracle_mod, bidirectional, window)


@pytest.mark.parametrize("heads,kvh,hd,page", [(24, 4, 256, 64), (32, 8, 128, 16), (64, 8, 64, 8), (6, 2, 96, 24), (5, 5, 32, 40), (24, 4, 256, 24),
                                                (32, 8, 128, 8), (16, 16, 128, 40), (12, 2, 256, 16), (8, 1, 160, 32), (14, 2, 224, 8)])
def test_attention_seg(rt, oracle_mod, heads, kvh, hd, page):
    """A pass of decode, verify and prompt segments over pages in random order, one segment behind a gap whose rows stay as they
    are; each segment is also checked in passes of its own kind."""
    rng = np.random.default_rng(page + hd)
    pps, slots = -(-700 // page), 5
    table = rng.permutation(pps * slots).reshape(slots, pps).astype(np.int32)
    put_ints(rt, "pt", table)
    rt.set_paging("pt", page, pps, slots)
    caches(rt, pps * slots * kvh, page, hd)
    have = [600, 1, 77, 256, 310]
    n = rt.set_segments([(i, 0, c) for i, c in enumerate(have)])
    k, v = keys(rng, n, kvh, hd), rng.standard_normal((n, kvh, hd)).astype(np.float32)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
    wk, wv = oracle_mod.kv4_values(k, v)
    first = np.cumsum([0] + have)
    held = [tuple(w[first[i]:first[i + 1]].transpose(1, 0, 2) for w in (wk, wv)) for i in range(slots)]
    for segments in ([(0, 599, 1), (1, 0, 1), (3, 255, 1), (2, 76, 1), (4, 309, 1)],
                     [(0, 593, 7), (2, 70, 5, 20), (4, 302, 8)],
                     [(0, 555, 45), (1, 0, 1, 50), (2, 60, 17), (3, 250, 6), (4, 0, 11)]):
        n = rt.set_segments(segments)
        q = rng.standard_normal((n, heads, hd)).astype(np.float32)
        put(rt, "q", q)
        put(rt, "o", np.full(q.size, 7.0))
        rt.attention_seg("q", "kc", "vc", "o", heads, kvh, hd)
        got, row, used = get(rt, "o", q.shape), 0, np.zeros(n, bool)
        for slot, pos0, rows, *at in segments:
            row = at[0] if at else row
            check(got[row:row + rows], q[row:row + rows], *held[slot], heads, kvh, pos0 + 1, oracle_mod)
            used[row:row + rows] = True
            row += rows
        assert (got[~used] == 7.0).all()


def test_attention_is_told_what_it_is_given(rt, torch):
    """Refusals that only the runtime can give: caches of other shapes or precisions than the call's."""
    caches(rt, 2, 40, 64)
    rt.alloc("h", 2 * 40 * 64, 2)
    for name in ("q", "o", "k", "v"):
        rt.alloc(name, 4 * 4 * 64)
    call = dict(heads=4, kv_heads=2, hd=64, max_seq=40, seq_len=10, ntok=4)

    def attention(kc="kc", vc="vc", **kw):
        rt.attention("q", kc, vc, "o", **{**call, **kw})

    attention()
    for kw in (dict(max_seq=48), dict(max_seq=32), dict(hd=32), dict(kv_heads=4), dict(seq_len=38), dict(ntok=0)):
        with pytest.raises(ValueError):
            attention(**kw)
    attention(max_seq=36, seq_len=33)  # rounds up to the same blocks
    for pair in (("kc", "h"), ("h", "vc")):
        with pytest.raises(TypeError):
            attention(*pair)
        with pytest.raises(TypeError):
            rt.kv_append("k", "v", *pair, 2, 40, 64, 0, 4)
    with pytest.raises(TypeError):
        rt.rmsnorm("kc", "w", "o", 64)
    with pytest.raises(TypeError):
        rt.read_floats("kc")
    with pytest.raises(TypeError):
        rt.write_floats("kc", [1.0])
    for bad in ((0, 8, 64), (1, 8, 48), (1, 0, 64), (1, 8, 512), (1, 2 ** 32 + 8, 64), (1, 8, 2 ** 32 + 64)):
        with pytest.raises(ValueError):
            rt.alloc_kv4("bad", *bad)
    assert "bad" not in rt.buffers
    put_ints(rt, "pt", [0, 1])
    rt.set_paging("pt", 32, 1, 2)
    rt.set_segments([(0, 3, 2)])
    with pytest.raises(ValueError):  # blocks of 40 positions, pages of 32
        rt.attention_seg("q", "kc", "vc", "o", 4, 2, 64)
    assert rt.buffer_elem("kc") == 1 and rt.buffer_bytes() >= 2 * 2 * 40 * 64 * 9 // 16
    rt.zero("kc")
    assert not blocks(rt, "kc").any()
