"""Verification of drafted tokens on the CPU: the oracle's rule by closed forms and frequencies, and the entry point's refusals (the
pointers below are never followed)."""
from __future__ import annotations

import ctypes

import numpy as np

from vinf_3080ti_amd import _lib

FAKE = ctypes.c_void_p(0x10000)


def test_rule_by_hand(oracle_mod):
    """p = (1/2, 1/4, 1/8, 1/8): acceptance at the border of u q < p, what a refusal draws from, the token after all drafts."""
    l = np.log([[4.0, 2, 1, 1]] * 2)
    q = np.array([[0.25, 0.5, 0.25, 0.0]])

    def go(x, u0, u1, v1=0.0, probs=q):
        return [a.tolist() for a in oracle_mod.verify_draft(l, [x], probs, [[u0, u1], [0, v1]], [1], [1.0])]

    assert go(1, 0.49, 0)[:2] == [[1, 0], [1]] and go(1, 0.51, 0)[:2] == [[0, -1], [0]]
    # left over: (1/4, 0, 0, 1/8) -> 2/3, 1/3
    assert go(1, 0.9, 0.66)[0] == [0, -1] and go(1, 0.9, 0.67)[0] == [3, -1]
    # a draft chosen without chance: accepted with p(x), else any other token
    assert go(1, 0.24, 0, 0.51, None)[0] == [1, 1] and go(1, 0.26, 0.66, 0, None)[0] == [0, -1]
    assert go(1, 0.26, 0.7, 0, None)[0] == [2, -1] and go(1, 0.26, 0.9, 0, None)[0] == [3, -1]
    assert go(0, 0.0, 0, 0.99)[0] == [0, 3]
    assert np.allclose(go(1, 0.1, 0, 0.6)[2], np.log([0.25, 0.25]))


def test_emitted_tokens_follow_the_target(oracle_mod):
    """The first token's distribution is the target's whatever the draft's is: 40000 passes, each frequency within five standard
    deviations."""
    rng = np.random.default_rng(0)
    l = rng.standard_normal(6) * 1.5
    p = np.exp(l / 0.8) / np.exp(l / 0.8).sum()
    q = rng.dirichlet(np.ones(6))
    n, seen = 40000, np.zeros(6)
    for _ in range(n):
        x = rng.choice(6, p=q)
        tokens, _, _ = oracle_mod.verify_draft([l, l], [x], [q], rng.random((2, 2)), [1], [0.8])
        seen[tokens[0]] += 1
    assert (np.abs(seen / n - p) < 5 * np.sqrt(p * (1 - p) / n)).all()


def test_refusals():
    lib = _lib.load()
    ks, ts = (ctypes.c_int32 * 3)(2, 0, 4), (ctypes.c_double * 3)(1.0, 0.0, 0.5)
    need = lib.vq_verify_draft_workspace_bytes(5000, ks, 3)
    assert need >= 9 * 3 * 16

    def call(logits=FAKE, draft=FAKE, probs=None, u=FAKE, tokens=FAKE, counts=FAKE, lp=None, vocab=5000, ks=ks, ts=ts, n=3, ws=FAKE,
             nws=need):
        return lib.vq_verify_draft(logits, draft, probs, u, tokens, counts, lp, vocab, ks, ts, n, ws, nws, None)

    for bad in (dict(logits=None), dict(draft=None), dict(u=None), dict(tokens=None), dict(counts=None), dict(ks=None), dict(ts=None),
                dict(n=0), dict(n=65), dict(n=-1)):
        assert call(**bad) == _lib.VQ_ERR_ARG, bad
    for bad in (dict(vocab=0), dict(vocab=-3), dict(vocab=2 ** 31 - 1), dict(ks=(ctypes.c_int32 * 3)(2, -1, 4)),
                dict(ks=(ctypes.c_int32 * 3)(2, 129, 4)), dict(ts=(ctypes.c_double * 3)(1, -0.5, 1)),
                dict(ts=(ctypes.c_double * 3)(1, float("nan"), 1)), dict(ts=(ctypes.c_double * 3)(float("inf"), 1, 1))):
        assert call(**bad) == _lib.VQ_ERR_SHAPE, bad
    for bad in (dict(ws=None), dict(nws=need - 1), dict(ws=ctypes.c_void_p(0x10008))):
        assert call(**bad) == _lib.VQ_ERR_WORKSPACE, bad
    for bad in ((0, ks, 3), (5000, None, 3), (5000, ks, 0), (5000, ks, 65), (5000, (ctypes.c_int32 * 1)(200), 1)):
        assert lib.vq_verify_draft_workspace_bytes(*bad) == 0
