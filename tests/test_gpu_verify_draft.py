"""Verification of drafted tokens on the GPU, through the runtime, against the float64 oracle."""
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


def put(rt, name, a):
    a = np.ascontiguousarray(a).reshape(-1)
    rt.alloc(name, max(a.size, 1))
    if a.size:
        rt.write(name, a.tobytes())


def case(rng, vocab, drafted, temps, with_probs):
    """Peaked logits as a model has them, drafts near the target so that some are accepted."""
    rows, d = sum(drafted) + len(drafted), sum(drafted)
    l = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    for r in range(rows):
        top = rng.integers(0, vocab, min(12, vocab))
        l[r, top] += 9 + 2 * rng.standard_normal(top.size).astype(np.float32)
    at = [r for r, last in zip(range(rows), [j == k for k in drafted for j in range(k + 1)]) if not last]
    ts = [t for k, t in zip(drafted, temps) for _ in range(k)]
    guess = l[at] + 0.5 * rng.standard_normal((d, vocab)).astype(np.float32)
    draft, probs = guess.argmax(1).astype(np.int32) if d else np.zeros(0, np.int32), None
    if with_probs:
        e = np.exp((guess - guess.max(1, keepdims=True)) / np.maximum(np.array(ts), 0.3)[:, None]) if d else guess
        probs = (e / e.sum(1, keepdims=True)).astype(np.float32) if d else guess
        draft = np.array([rng.choice(vocab, p=p.astype(np.float64) / p.sum(dtype=np.float64)) for p in probs], np.int32)
    return l, draft, probs, rng.random((rows, 2)).astype(np.float32)


def run(rt, l, draft, probs, u, drafted, temps, logprobs=True):
    rows, vocab = l.shape
    put(rt, "l", l)
    put(rt, "u", u)
    put(rt, "d", draft)
    if probs is not None:
        put(rt, "p", probs)
    for name, n in (("t", rows + 3), ("c", len(drafted) + 3), ("lp", rows + 3)):
        put(rt, name, np.full(n, -77, np.int32))
    rt.verify_draft("l", "d" if len(draft) else None, "u", "t", "c", vocab, drafted, temperature=temps,
                    probs="p" if probs is not None else None, logprobs="lp" if logprobs else None)
    out = [np.frombuffer(rt.read(name), t) for name, t in (("t", np.int32), ("c", np.int32), ("lp", np.float32))]
    assert (out[0][rows:] == -77).all() and (out[1][len(drafted):] == -77).all()
    assert (out[2].view(np.int32)[rows if logprobs else 0:] == -77).all()
    return out[0][:rows], out[1][:len(drafted)], out[2][:rows]


def check(oracle_mod, got, args):
    """Whole numbers equal; log-probabilities (64 bits, rounded once) within one rounding to fp32 and 1e-9."""
    tokens, counts, lp = oracle_mod.verify_draft(*args)
    assert np.array_equal(got[1], counts) and np.array_equal(got[0], tokens)
    fin = np.isfinite(lp)
    assert np.array_equal(got[2][~fin], lp[~fin].astype(np.float32))
    assert (np.abs(got[2][fin] - lp[fin]) <= np.abs(lp[fin]) * 2.0 ** -24 + 1e-9).all()


@pytest.mark.parametrize("vocab", [1, 7, 2047, 2048, 2049, 32001, 248320])
@pytest.mark.parametrize("with_probs", [False, True])
def test_against_the_oracle(rt, oracle_mod, vocab, with_probs):
    rng = np.random.default_rng(vocab + with_probs)
    drafted = [3, 0, 1, 4, 2] if vocab < 100000 else [3, 0, 2]
    temps = [0.7, 1.0, 0.0, 1.6, 0.05][:len(drafted)]
    l, draft, probs, u = case(rng, vocab, drafted, temps, with_probs)
    check(oracle_mod, run(rt, l, draft, probs, u, drafted, temps), (l, draft, probs, u, drafted, temps))


@pytest.mark.parametrize("seed", range(6))
def test_ragged_batches(rt, oracle_mod, seed):
    """More sequences than one launch takes, drafts up to the limit, every kind of temperature; logprobs left out."""
    rng = np.random.default_rng(seed)
    n = [1, 2, 64, 65, 130, 9][seed]
    drafted = [int(k) for k in rng.integers(0, 6, n)]
    drafted[rng.integers(n)] = 128 if n < 10 else 17
    temps = [float(t) for t in rng.choice([0.0, 0.2, 1.0, 3.0], n)]
    l, draft, probs, u = case(rng, int(rng.integers(50, 4000)), drafted, temps, seed % 2 == 1)
    got = run(rt, l, draft, probs, u, drafted, temps, logprobs=seed != 2)
    want = oracle_mod.verify_draft(l, draft, probs, u, drafted, temps)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_values_at_the_edges(rt, oracle_mod):
    """Rows with NaN, infinities and nothing above -inf; drafts outside the vocabulary; random numbers 0 and 1; probabilities that
    are NaN, negative, all zero, or the target's own; ties at temperature 0."""
    rng = np.random.default_rng(5)
    vocab, inf, nan = 5000, np.inf, np.nan
    drafted = [1] * 14
    temps = [1.0] * 10 + [0.0] * 4
    l, draft, _, u = case(rng, vocab, drafted, temps, True)
    probs = np.exp(l[::2].astype(np.float64) - l[::2].max(1, keepdims=True))
    probs = (probs / probs.sum(1, keepdims=True) * 0.999).astype(np.float32)
    draft = np.array([int(p.argmax()) for p in probs], np.int32)
    l[0, ::3] = nan
    l[2, [17, 4000]] = inf
    l[4] = -inf
    l[6] = nan
    l[8, 10:] = -inf
    draft[5], draft[6], draft[7] = -1, vocab, 2 ** 31 - 1
    u[0] = 0
    u[3], u[10], u[13], u[15] = 0, 1, [0.5, 1.0], [0.5, 0.0]
    u[18] = [1.0, 0.3]
    probs[9] = 2.0  # takes everything off
    probs[8, ::2], probs[8, 1::4] = nan, -1.0
    probs[5] = 0
    l[20], l[22, [9, 3]] = 1.0, inf  # greedy: ties everywhere, ties at +inf
    l[24] = -inf
    l[26, 0] = nan
    draft[10], draft[11], draft[12], draft[13] = 0, 3, 0, int(np.nanargmax(l[26]))
    args = (l, draft, probs, u, drafted, temps)
    check(oracle_mod, run(rt, *args), args)
    args = (l, draft, None, u, drafted, temps)
    check(oracle_mod, run(rt, *args), args)


def test_temperatures_at_the_ends(rt, oracle_mod):
    """The smallest positive temperatures leave the largest logit (ties share), the largest one makes all tokens alike."""
    rng = np.random.default_rng(6)
    drafted, temps = [2, 0, 1, 2, 0], [5e-324, 1e-310, 1e-300, 1.7e308, 1e-308]
    l, draft, probs, u = case(rng, 3000, drafted, temps, True)
    l[3, [5, 90]] = 50.0
    l[0, draft[0]] = 60.0
    for p in (probs, None):
        args = (l, draft, p, u, drafted, temps)
        check(oracle_mod, run(rt, *args), args)


def test_a_sequence_does_not_depend_on_the_others(rt):
    """The bits of a sequence's results alone, in a batch, and behind a capture that is replayed."""
    import torch

    rng = np.random.default_rng(8)
    vocab, drafted, temps = 30000, [2, 4, 0, 3], [0.9, 0.6, 1.0, 1.3]
    l, draft, probs, u = case(rng, vocab, drafted, temps, True)
    whole = run(rt, l, draft, probs, u, drafted, temps)
    row = d = 0
    for i, k in enumerate(drafted):
        got = run(rt, l[row:row + k + 1], draft[d:d + k], probs[d:d + k] if k else None, u[row:row + k + 1], [k], [temps[i]])
        assert got[1][0] == whole[1][i]
        for a, b in ((0, 0), (2, 2)):
            assert np.array_equal(got[a].view(np.int32), whole[b][row:row + k + 1].view(np.int32))
        row, d = row + k + 1, d + k
    put(rt, "l", l)
    put(rt, "u", u)
    put(rt, "d", draft)
    put(rt, "p", probs)
    for name, n in (("t", len(l)), ("c", 4), ("lp", len(l))):
        rt.alloc(name, n)
    call = lambda: rt.verify_draft("l", "d", "u", "t", "c", vocab, drafted, temperature=temps, probs="p", logprobs="lp")  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    for rep in range(4):
        lt, u2 = rt.buffer_tensor("l").view(l.shape), rng.random(u.shape).astype(np.float32)
        lt.copy_(torch.from_numpy(l).flip(1) if rep % 2 else torch.from_numpy(l))
        rt.write("u", u2.tobytes())
        torch.cuda.synchronize()
        for name in ("t", "c", "lp"):
            rt.buffer_tensor(name).fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        got = [rt.read(name) for name in ("t", "c", "lp")]
        call()
        torch.cuda.synchronize()
        assert got == [rt.read(name) for name in ("t", "c", "lp")]


def test_runtime_refusals(rt):
    for name, n in (("l", 300), ("u", 6), ("t", 3), ("c", 1), ("d", 2), ("p", 200)):
        rt.alloc(name, n)
    ok = dict(logits="l", draft="d", uniforms="u", tokens="t", counts="c", vocab=100, drafted=[2])
    rt.verify_draft(**ok, temperature=0.5, probs="p")
    for bad in (dict(drafted=[]), dict(drafted=[129]), dict(drafted=[-1]), dict(vocab=0), dict(vocab=101), dict(draft=None),
                dict(drafted=[3]), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=[1.0, 1.0]),
                dict(temperature=float("inf")), dict(drafted=[1, 0], temperature=[1.0]), dict(tokens="c"),
                dict(probs="u")):
        with pytest.raises(ValueError):
            rt.verify_draft(**{**ok, **bad})
    with pytest.raises(KeyError):
        rt.verify_draft(**{**ok, "logits": "none"})
