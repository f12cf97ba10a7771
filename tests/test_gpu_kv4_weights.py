"""Attention over the 4-bit cache where one key takes nearly all of the softmax: what the others' small weights give to the output."""
from __future__ import annotations

import numpy as np
import pytest
from test_gpu_kv4 import caches, get, put

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


@pytest.mark.parametrize("heads,kvh,hd", [(24, 4, 256), (32, 8, 128), (8, 2, 64), (6, 2, 96)])
@pytest.mark.parametrize("ntok", [1, 4, 40])
@pytest.mark.parametrize("sink", [0.0, 1.5])
@pytest.mark.parametrize("gap", [8, 12, 14])
def test_one_dominant_key(rt, oracle_mod, heads, kvh, hd, ntok, sink, gap):
    """The first key lies `gap` nats above the other 2999, its V is `sink`, theirs lie around 1. All terms are positive, so each error is
    relative to the output's part that it belongs to:
     - a score's error e (query pairs of 22 bits, fp32 sums and scalings, for the first key, whose products but one are zero, without
       the sums) changes a weight by its share e, and so do exp2 and the pair's 2^-23;
     - a weight's second half ends at 2^-36 of the row's largest weight: the first key's, 1;
     - a sum's terms go through at most a wave's n / 4 keys, in both halves, and 64 joins: (n / 2 + 64) 2^-24."""
    n = 3000
    rng = np.random.default_rng(hd + ntok + gap)
    k = np.zeros((n, kvh, hd), np.float32)
    k[0, :, 0] = 8.0
    k[1:, :, 32:] = rng.standard_normal((n - 1, kvh, hd - 32))
    v = np.maximum(rng.normal(1.0, 0.25, (n, kvh, hd)), 0.3).astype(np.float32)
    v[0] = sink
    caches(rt, kvh, n, hd)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append("k", "v", "kc", "vc", kvh, n, hd, 0, n)
    wk, wv = (x.transpose(1, 0, 2) for x in oracle_mod.kv4_values(k, v))
    q = (rng.standard_normal((ntok, heads, hd)) * 0.4).astype(np.float32)
    q[..., 0] = gap * np.sqrt(hd) / 8
    put(rt, "q", q)
    want = oracle_mod.attention(q, wk, wv, heads, kvh, n - ntok + 1, False, 0)
    kv = np.arange(heads) * kvh // heads
    score = np.einsum("thd,hnd->thn", q.astype(np.float64), wk[kv]) / np.sqrt(hd)
    size = np.einsum("thd,hnd->thn", np.abs(q[..., 1:].astype(np.float64)), np.abs(wk[kv][..., 1:])) / np.sqrt(hd)
    w = np.exp(score[..., 1:] - score[..., :1])
    e = 2.0 ** -24 * ((hd + 8) * size.max(-1) + 8 * score[..., 0]) + 2.0 ** -22
    rel = 2 * (2 * e + 2.0 ** -23 + (n / 2 + 64) * 2.0 ** -24)
    floor = n * 2.0 ** -36 * wv[kv].max(1) / (1 + w.sum(-1))[..., None]
    for invariant in (False, True):
        rt.set_batch_invariant(invariant)
        put(rt, "o", np.zeros(q.size))
        rt.attention("q", "kc", "vc", "o", heads, kvh, hd, n, n - ntok + 1, ntok)
        off = np.abs(get(rt, "o", q.shape) - want)
        assert (off <= rel[..., None] * want + floor).all(), (off / want).max()


@pytest.mark.parametrize("heads,kvh,hd", [(24, 4, 256), (32, 8, 128), (8, 2, 64), (6, 2, 96)])
@pytest.mark.parametrize("ntok", [1, 40])
@pytest.mark.parametrize("power", [20, 22, 24, 26, 28, 40, 80])
def test_scores_whose_roundings_are_large(rt, oracle_mod, heads, kvh, hd, ntok, power):
    """Scores near 2^power, whose differences are far beyond their fp32 roundings and beyond what exp holds: the keys of the largest one
    share all of the softmax. Off by a rounding for each of them, in numerator and denominator, and for 16 joins and the pairs."""
    n = 700
    rng = np.random.default_rng(power + ntok)
    k = np.zeros((n, kvh, hd), np.float32)
    k[:, :, 0] = rng.permuted(np.repeat(np.arange(1.0, n + 1)[:, None], kvh, 1), axis=0)
    v = rng.standard_normal((n, kvh, hd)).astype(np.float32)
    caches(rt, kvh, n, hd)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append("k", "v", "kc", "vc", kvh, n, hd, 0, n)
    wk, wv = (x.transpose(1, 0, 2) for x in oracle_mod.kv4_values(k, v))
    q = np.zeros((ntok, heads, hd), np.float32)
    q[..., 0] = 2.0 ** power * np.sqrt(hd) / n * rng.uniform(0.7, 1, (ntok, heads))
    put(rt, "q", q)
    kv = np.arange(heads) * kvh // heads
    for invariant in (False, True):
        rt.set_batch_invariant(invariant)
        put(rt, "o", np.zeros(q.size))
        rt.attention("q", "kc", "vc", "o", heads, kvh, hd, n, n - ntok + 1, ntok)
        got = get(rt, "o", q.shape)
        for t in range(ntok):
            sees = wk[kv, : n - ntok + 1 + t, 0]
            best = sees.max(1, keepdims=True)
            top = [np.flatnonzero(row == b[0]) for row, b in zip(sees, best)]
            want = np.stack([wv[h, i].mean(0) for h, i in zip(kv, top)])
            most = np.stack([np.abs(wv[h, i]).max(0) for h, i in zip(kv, top)])
            assert (np.abs(got[t] - want) <= most * (len(max(top, key=len)) + 16) * 2.0 ** -23).all(), (t, np.abs(got[t] - want).max())
