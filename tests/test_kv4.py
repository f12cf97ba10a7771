"""The 4-bit KV cache on the CPU: the oracle's rounding rule and layout by closed forms, and the entry points' refusals (checked on
the host before anything is launched; the pointers below are never followed)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from vinf_3080ti_amd import _lib

FAKE = ctypes.c_void_p(0x10000)
ODD = ctypes.c_void_p(0x10008)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def segs(*rows):
    return (ctypes.c_int32 * (4 * len(rows)))(*[v for r in rows for v in r]), len(rows)


def test_rounding_rule(oracle_mod):
    """Every value within half a step, whole steps kept, the scale on its grid and no larger than it has to be."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 64)) * np.exp(rng.uniform(-14, 8, (200, 1)))
    x[:50] = np.abs(x[:50])
    x[50:90] += 3 * np.abs(x[50:90]).max(-1, keepdims=True)
    c, d, z = oracle_mod.kv4_quantize(x)
    step, zero = np.repeat(d, 32, -1), np.repeat(z, 32, -1).astype(float)
    assert (np.abs(step * (c - zero) - x) <= step / 2 + 1e-300).all()
    assert (c <= 15).all() and (z <= 15).all()
    bits = d.astype(np.float16)
    assert (bits.astype(np.float64) == d).all() and not (bits.view(np.uint16) & 15).any()
    smaller = np.where(d > 2.0 ** -20, (bits.view(np.uint16) - 16).view(np.float16).astype(float), 0)
    g = x.reshape(200, 2, 32)
    span = np.maximum(g.max(-1), 0) - np.minimum(g.min(-1), 0)
    assert (15 * d >= span).all() and (15 * smaller < span).all()
    k = np.arange(32.0)[None] % 16 - 5
    c, d, z = oracle_mod.kv4_quantize(0.75 * k)
    assert d == 0.75 and z == 5 and (c == k + 5).all()
    c, d, z = oracle_mod.kv4_quantize(np.zeros((1, 32)))
    assert d == 0 and z == 0 and not c.any()


@pytest.mark.parametrize("hd", [32, 64, 96, 256])
def test_layout_places_each_value_once(oracle_mod, hd):
    """One value set at a time moves one nibble, at the documented place, and its group's header."""
    p = 16
    size = p * hd * 9 // 16
    assert _lib.load().vq_kv4_bytes(3, p, hd) == 3 * size
    for values in (False, True):
        for pos, dim in ((0, 0), (3, 17), (7, hd - 1), (8, 9), (15, hd // 2 + 5)):
            x = np.zeros((p, hd), np.float32)
            x[pos, dim] = 15.0
            b = oracle_mod.kv4_block(x, values)
            assert b.size == size
            words, heads = b[: p * hd // 2].view(np.uint32), b[p * hd // 2:].view(np.uint16)
            w = 4 if hd % 64 == 0 else 2
            at = (pos // 8) * hd + (dim // (16 * w) * 16 + dim % 16) * w + dim // 16 % w if values else \
                pos * hd // 8 + (dim % 32 // 8) * (hd // 32) + dim // 32
            e = pos % 8 if values else dim % 8
            assert np.flatnonzero(words).tolist() == [at] and words[at] == 15 << (4 * (e // 2) + 16 * (e % 2))
            h = ((pos // 8) * (hd // 32) + dim // 32) * 8 + pos % 8 if values else pos * (hd // 32) + dim // 32
            assert np.flatnonzero(heads).tolist() == [h] and heads[h] == np.float16(1.0).view(np.uint16)


def test_broken_rows(oracle_mod):
    k, v = np.ones((3, 32)), np.ones((3, 32))
    k[0, 3], v[1, 31] = np.inf, np.nan
    gk, gv = oracle_mod.kv4_values(k, v)
    assert np.isnan(gk[:2]).all() and not gv[:2].any()
    # All ones: the code 15 of a scale that is 1 / 15 rounded up to 7 significant bits.
    assert (gk[2] >= 1).all() and (gk[2] <= 1 + 2.0 ** -6).all() and (gv[2] == gk[2]).all()


def test_sizes(lib):
    assert lib.vq_kv4_bytes(4, 64, 256) == 4 * 64 * 144
    assert lib.vq_kv4_bytes(1, 1, 32) == lib.vq_kv4_bytes(1, 8, 32) == 8 * 18
    for bad in ((0, 8, 32), (1, 0, 32), (1, 8, 0), (1, 8, 48), (1, 8, 288), (1, 8, -32), (-1, 8, 32), (2 ** 62, 8, 32),
                (1, 2 ** 31 - 1, 32)):
        assert lib.vq_kv4_bytes(*bad) == 0


def test_append_and_read_refusals(lib):
    seg, n = segs((0, 5, 3, 0))
    for name in ("vq_kv4_append", "vq_kv4_read"):
        fn, fs = getattr(lib, name), getattr(lib, name + "_seg")
        ok = dict(ntok=3, kvh=2, max_seq=100, hd=64, pos0=5)

        def call(a=FAKE, b=FAKE, c=FAKE, d=FAKE, **kw):
            s = {**ok, **kw}
            return fn(a, b, c, d, s["ntok"], s["kvh"], s["max_seq"], s["hd"], s["pos0"], None)

        for i in range(4):
            assert call(*[None if i == j else FAKE for j in range(4)]) == _lib.VQ_ERR_ARG
        assert call(*([FAKE, FAKE, ODD, FAKE] if "append" in name else [ODD, FAKE, FAKE, FAKE])) == _lib.VQ_ERR_ARG
        for bad in (dict(ntok=0), dict(kvh=0), dict(hd=48), dict(hd=0), dict(hd=288), dict(pos0=-1), dict(pos0=98), dict(max_seq=0),
                    dict(ntok=101), dict(pos0=2 ** 31 - 2), dict(max_seq=2 ** 31 - 1, pos0=2 ** 31 - 4)):
            assert call(**bad) == _lib.VQ_ERR_SHAPE, bad

        def seg_call(table=seg, nseg=n, pt=FAKE, page=16, pps=4, pages=9, hd=64, kvh=2):
            return fs(FAKE, FAKE, FAKE, FAKE, table, nseg, kvh, hd, pt, page, pps, pages, None)

        assert seg_call(table=None) == seg_call(nseg=0) == seg_call(nseg=65) == seg_call(pt=None) == _lib.VQ_ERR_ARG
        for bad in (dict(page=12), dict(page=0), dict(page=-8), dict(pps=0), dict(pages=0), dict(pages=-1), dict(hd=40), dict(kvh=0),
                    dict(page=8, pps=0), dict(table=segs((0, 60, 5, 0))[0]), dict(table=segs((-1, 0, 5, 0))[0]),
                    dict(table=segs((0, 0, 0, 0))[0]), dict(table=segs((0, -1, 1, 0))[0])):
            assert seg_call(**bad) == _lib.VQ_ERR_SHAPE, bad


def test_attention_refusals(lib):
    ok = dict(heads=4, kvh=2, hd=64, max_seq=100, seq_len=50, ntok=3, bi=0, window=0)

    def call(a=FAKE, b=FAKE, c=FAKE, d=FAKE, ws=None, nws=0, **kw):
        s = {**ok, **kw}
        return lib.vq_attention4_ws(a, b, c, d, s["heads"], s["kvh"], s["hd"], s["max_seq"], s["seq_len"], s["ntok"], s["bi"],
                                    s["window"], ws, nws, None)

    for i in range(4):
        assert call(*[None if i == j else FAKE for j in range(4)]) == _lib.VQ_ERR_ARG
    assert call(FAKE, ODD) == call(FAKE, FAKE, ODD) == _lib.VQ_ERR_ARG
    for bad in (dict(heads=3), dict(heads=0), dict(heads=1), dict(kvh=0), dict(hd=80), dict(seq_len=0), dict(seq_len=99),
                dict(ntok=0), dict(ntok=101), dict(window=-1), dict(seq_len=2 ** 31 - 1), dict(max_seq=0)):
        assert call(**bad) == _lib.VQ_ERR_SHAPE, bad
    seg, n = segs((0, 5, 3, 0), (1, 0, 1, 3))

    def seg_call(table=seg, nseg=n, heads=4, kvh=2, hd=64, pt=FAKE, page=16, pps=4, pages=9, ws=None, nws=0):
        return lib.vq_attention4_seg_ws(FAKE, FAKE, FAKE, FAKE, table, nseg, heads, kvh, hd, pt, page, pps, pages, ws, nws, None)

    assert seg_call(table=None) == seg_call(pt=None) == _lib.VQ_ERR_ARG
    for bad in (dict(heads=5), dict(kvh=0), dict(hd=31), dict(page=20), dict(pps=0), dict(pages=0),
                dict(table=segs((0, 63, 2, 0), (1, 0, 1, 3))[0])):
        assert seg_call(**bad) == _lib.VQ_ERR_SHAPE, bad
    # Invalid shapes need no workspace; a workspace that is too small or misaligned is refused.
    for bad in ((3, 2, 64, 50, 1, 0), (4, 2, 48, 50, 1, 0), (4, 2, 64, 0, 1, 0), (4, 2, 64, 50, 0, 0), (4, 2, 64, 50, 1, -1)):
        assert lib.vq_attention4_workspace_bytes(*bad) == 0
    assert lib.vq_attention4_seg_workspace_bytes(None, 1, 4, 2, 64) == 0
    need = lib.vq_attention4_workspace_bytes(24, 4, 256, 100000, 1, 0)
    if need:
        big = dict(heads=24, kvh=4, hd=256, max_seq=100000, seq_len=100000, ntok=1)
        assert call(**big, ws=FAKE, nws=need - 1) == call(**big, ws=ODD, nws=need) == _lib.VQ_ERR_WORKSPACE


def test_attention_ends_inside_32_bits(lib):
    """Contexts so near the end of 32 bits that a wave's step past the last key would leave them, and passes with more query vectors
    than that: no workspace size, and a refusal."""
    end = 2 ** 31 - 1
    assert lib.vq_attention4_workspace_bytes(8, 2, 64, end - 1024, 1, 0) > 0
    assert lib.vq_attention4_workspace_bytes(8, 2, 64, end - 1022, 1, 0) == 0
    assert lib.vq_attention4_ws(FAKE, FAKE, FAKE, FAKE, 8, 2, 64, end - 8, end - 1022, 1, 0, 0, None, 0, None) == _lib.VQ_ERR_SHAPE
    assert lib.vq_attention4_workspace_bytes(8, 2, 64, 5, 2 ** 27 + 1, 0) == 0
    assert lib.vq_attention4_seg_workspace_bytes(segs((0, 0, 2 ** 26, 0), (1, 0, 2 ** 26 + 1, 0))[0], 2, 8, 2, 64) == 0
    assert lib.vq_attention4_ws(FAKE, FAKE, FAKE, FAKE, 8, 2, 64, end - 8, 5, 2 ** 27 + 1, 0, 0, None, 0, None) == _lib.VQ_ERR_SHAPE
