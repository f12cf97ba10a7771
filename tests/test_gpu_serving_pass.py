"""The 4-bit cache, the pages and the verification of drafts used together as a serving loop uses them, and the 4-bit attention where
other rows, other passes, graphs, unwritten memory or large pools could reach into it."""
from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest
from test_gpu_kv4 import blocks, bound, caches, check, get, keys, put, put_ints

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


# ---- one serving loop -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("heads,kvh,hd,page,seed", [(24, 4, 256, 16, 0), (8, 2, 128, 16, 1), (6, 2, 96, 24, 2), (8, 8, 64, 8, 3)])
def test_speculative_serving(rt, oracle_mod, heads, kvh, hd, page, seed):
    """A prompt in one slot, forked into three, then rounds of: reserve, append and attend the last token and its drafts, verify, give
    back the pages of what was refused. Attention against the oracle over each sequence's own history, the tokens and counts against
    the oracle's, the pages against the lengths; one sequence ends and its slot takes a copy of another on the way."""
    rng, pick = np.random.default_rng(seed), random.Random(seed)
    per, slots, vocab = -(-120 // page), 4, 300
    pages = per * slots
    put_ints(rt, "table", np.full((slots, per), -1))
    rt.set_paging("table", page, per, slots)
    caches(rt, pages * kvh, page, hd)
    rt.set_page_pools(["kc", "vc"], pages)
    hist: dict[int, list[np.ndarray]] = {}

    def attend(segments):
        rt.pages_reserve(segments)
        n = rt.set_segments(segments)
        k, v = keys(rng, n, kvh, hd), rng.standard_normal((n, kvh, hd)).astype(np.float32)
        q = rng.standard_normal((n, heads, hd)).astype(np.float32)
        for name, x in (("k", k), ("v", v), ("q", q), ("o", np.full(q.size, 9.0))):
            put(rt, name, x)
        rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
        rt.attention_seg("q", "kc", "vc", "o", heads, kvh, hd)
        got, row = get(rt, "o", q.shape), 0
        wk, wv = oracle_mod.kv4_values(k, v)
        for slot, pos0, rows in segments:
            old = hist.get(slot, [np.zeros((0, kvh, hd))] * 2)
            hist[slot] = [np.concatenate([o[:pos0], w[row:row + rows]]) for o, w in zip(old, (wk, wv))]
            check(got[row:row + rows], q[row:row + rows], *(x.transpose(1, 0, 2) for x in hist[slot]), heads, kvh, pos0 + 1, oracle_mod)
            row += rows

    attend([(0, 0, 37)])
    rt.pages_fork(0, [1, 2], 37)
    hist[1], hist[2] = hist[0], hist[0]
    assert rt.pages_available() == pages - -(-37 // page)
    length = {0: 37, 1: 37, 2: 37}
    for step in range(7):
        if step == 3:
            rt.pages_free([1])
            rt.pages_copy([(2, 3, length[2] - 5)])
            hist[3], length[3] = [x[:length[2] - 5] for x in hist[2]], length[2] - 5
            del hist[1], length[1]
            rt.pages_compact()
        live = sorted(length)
        drafted = [pick.randint(0, 4) for _ in live]
        attend([(s, length[s], k + 1) for s, k in zip(live, drafted)])
        rows, drafts = sum(drafted) + len(live), sum(drafted)
        logits = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
        probs = rng.dirichlet(np.ones(vocab), drafts).astype(np.float32) if drafts else np.zeros((0, vocab), np.float32)
        draft = np.array([rng.choice(vocab, p=p.astype(np.float64) / p.sum(dtype=np.float64)) for p in probs], np.int32)
        at = 0
        for i, k in enumerate(drafted):  # (drafts that the target often agrees with)
            for j in range(k):
                if pick.random() < 0.7:
                    logits[at + i + j, draft[at + j]] += 8
            at += k
        u = rng.random((rows, 2)).astype(np.float32)
        put(rt, "logits", logits)
        put(rt, "u", u)
        for name, n in (("tokens", rows), ("counts", len(live))):
            put_ints(rt, name, np.full(n, 77))
        if drafts:
            put(rt, "probs", probs)
            put_ints(rt, "draft", draft)
        rt.verify_draft("logits", "draft" if drafts else None, "u", "tokens", "counts", vocab, drafted, temperature=0.8,
                        probs="probs" if drafts else None)
        tokens, counts = (np.frombuffer(rt.read(x), np.int32) for x in ("tokens", "counts"))
        want = oracle_mod.verify_draft(logits, draft, probs if drafts else None, u, drafted, [0.8] * len(live))
        assert tokens.tolist() == list(want[0]) and counts.tolist() == list(want[1]), step
        for s, accepted in zip(live, counts.tolist()):
            length[s] += accepted + 1
            rt.pages_free([s], length[s])
            hist[s] = [x[:length[s]] for x in hist[s]]
            assert len(rt.pages_of(s)) == -(-length[s] // page)
    for s in list(length):
        rt.pages_free([s])
    assert rt.pages_available() == pages


# ---- attention: what must not reach a row -------------------------------------------------------------------------


@pytest.mark.parametrize("heads,kvh,hd", [(24, 4, 256), (32, 8, 128), (64, 8, 64), (6, 2, 96)])
@pytest.mark.parametrize("ntok,seq_len", [(1, 13), (1, 700), (5, 600), (40, 3), (33, 481)])
def test_memory_behind_the_last_key(rt, oracle_mod, heads, kvh, hd, ntok, seq_len):
    """Blocks whose unwritten positions hold any bytes (all ones: scales that are no numbers)."""
    rng = np.random.default_rng(ntok + seq_len)
    n, max_seq = seq_len + ntok - 1, seq_len + ntok + 70
    caches(rt, kvh, max_seq, hd)
    for name in ("kc", "vc"):
        rt.write(name, b"\xff" * blocks(rt, name).size)
    k, v = keys(rng, n, kvh, hd), rng.standard_normal((n, kvh, hd)).astype(np.float32)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append("k", "v", "kc", "vc", kvh, max_seq, hd, 0, n)
    wk, wv = (x.transpose(1, 0, 2) for x in oracle_mod.kv4_values(k, v))
    q = rng.standard_normal((ntok, heads, hd)).astype(np.float32)
    put(rt, "q", q)
    for invariant in (False, True):
        rt.set_batch_invariant(invariant)
        put(rt, "o", np.zeros(q.size))
        rt.attention("q", "kc", "vc", "o", heads, kvh, hd, max_seq, seq_len, ntok)
        check(get(rt, "o", q.shape), q, wk, wv, heads, kvh, seq_len, oracle_mod)


@pytest.mark.parametrize("heads,kvh,hd", [(8, 4, 256), (8, 2, 128), (12, 3, 64)])
@pytest.mark.parametrize("ntok", [1, 30])
@pytest.mark.parametrize("step", [0.03, -0.03, 1.0])
def test_scores_that_climb(rt, oracle_mod, heads, kvh, hd, ntok, step):
    """Scores that rise (or fall) steadily along the keys, by less and by more than a softmax's sums are rescaled for."""
    rng = np.random.default_rng(hd)
    n = 400 + ntok
    k = np.zeros((n, kvh, hd), np.float32)
    k[..., : hd // 2] = (np.arange(n)[:, None, None] * (step * 2 / np.sqrt(hd)))
    k += rng.standard_normal(k.shape).astype(np.float32) * 0.01
    v = rng.standard_normal((n, kvh, hd)).astype(np.float32)
    caches(rt, kvh, n, hd)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append("k", "v", "kc", "vc", kvh, n, hd, 0, n)
    wk, wv = (x.transpose(1, 0, 2) for x in oracle_mod.kv4_values(k, v))
    q = np.ones((ntok, heads, hd), np.float32) + rng.standard_normal((ntok, heads, hd)).astype(np.float32) * 0.1
    put(rt, "q", q)
    put(rt, "o", np.zeros(q.size))
    rt.attention("q", "kc", "vc", "o", heads, kvh, hd, n, 400, ntok)
    check(get(rt, "o", q.shape), q, wk, wv, heads, kvh, 400, oracle_mod)


@pytest.mark.parametrize("heads,kvh,hd", [(24, 4, 256), (32, 8, 128), (8, 2, 64)])
def test_broken_queries_and_keys_stay_by_themselves(rt, oracle_mod, heads, kvh, hd):
    """A query with a value that is no number, an infinite one, one of zeros: other rows and heads do not see them. A key that was not
    finite makes the rows that see it NaN, and only those of its kv head."""
    rng = np.random.default_rng(hd)
    ntok, seq_len = 20, 90
    n = seq_len + ntok - 1
    k, v = keys(rng, n, kvh, hd), rng.standard_normal((n, kvh, hd)).astype(np.float32)
    k[100, 0, 3] = np.inf
    caches(rt, kvh, n, hd)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append("k", "v", "kc", "vc", kvh, n, hd, 0, n)
    wk, wv = (x.transpose(1, 0, 2) for x in oracle_mod.kv4_values(k, v))
    q = rng.standard_normal((ntok, heads, hd)).astype(np.float32)
    q[2, 1, 5], q[3, heads - 1, 0], q[4] = np.nan, np.inf, 0
    put(rt, "q", q)
    for invariant in (False, True):
        rt.set_batch_invariant(invariant)
        put(rt, "o", np.zeros(q.size))
        rt.attention("q", "kc", "vc", "o", heads, kvh, hd, n, seq_len, ntok)
        got = get(rt, "o", q.shape)
        sees = np.zeros((ntok, heads), bool)
        sees[100 - seq_len + 1:, : heads // kvh] = True  # row t's last key is seq_len - 1 + t
        sees[2, 1] = sees[3, heads - 1] = True
        assert np.isnan(got[sees]).all() and np.isfinite(got[~sees]).all()
        qq, kk = q.copy(), np.nan_to_num(wk)
        qq[2, 1], qq[3, heads - 1] = 0, 0
        want = oracle_mod.attention(qq, kk, wv, heads, kvh, seq_len, False, 0)
        off = bound(qq, kk, wv, heads, kvh, seq_len, 0, 0)
        assert (np.abs(got - want) <= off)[~sees].all()


@pytest.mark.parametrize("heads,kvh,hd,page", [(24, 4, 256, 64), (32, 8, 128, 16), (8, 2, 64, 8), (6, 2, 96, 24)])
def test_rows_of_a_batch_invariant_pass(rt, heads, kvh, hd, page):
    """A row's bits are the same alone, among other sequences' and in passes cut elsewhere."""
    rng = np.random.default_rng(page)
    per, slots = -(-400 // page), 3
    put_ints(rt, "pt", rng.permutation(per * slots).reshape(slots, per))
    rt.set_paging("pt", page, per, slots)
    caches(rt, per * slots * kvh, page, hd)
    n = rt.set_segments([(0, 0, 390), (1, 0, 77), (2, 0, 260)])
    put(rt, "k", keys(rng, n, kvh, hd))
    put(rt, "v", rng.standard_normal((n, kvh, hd)))
    rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
    rt.set_batch_invariant(True)

    def run(segments, q):
        rt.set_segments(segments)
        put(rt, "q", q)
        put(rt, "o", np.zeros(q.size))
        rt.attention_seg("q", "kc", "vc", "o", heads, kvh, hd)
        return get(rt, "o", q.shape).copy()

    q = rng.standard_normal((60, heads, hd)).astype(np.float32)
    whole = run([(0, 330, 60)], q)
    others = rng.standard_normal((90, heads, hd)).astype(np.float32)
    mixed = run([(1, 0, 77), (0, 330, 60), (2, 247, 13)], np.concatenate([others[:77], q, others[77:]]))
    assert np.array_equal(whole, mixed[77:137])
    cut = np.concatenate([run([(0, 330, 7)], q[:7]), run([(0, 337, 1)], q[7:8]), run([(2, 259, 1), (0, 338, 52)], np.concatenate([others[:1], q[8:]]))[1:]])
    assert np.array_equal(whole, cut)


def test_more_segments_than_a_table_holds(rt, oracle_mod):
    """70 sequences of one to 200 keys in one pass."""
    rng = np.random.default_rng(70)
    heads, kvh, hd, page, slots = 8, 2, 64, 16, 70
    per = -(-200 // page)
    put_ints(rt, "pt", rng.permutation(per * slots).reshape(slots, per))
    rt.set_paging("pt", page, per, slots)
    caches(rt, per * slots * kvh, page, hd)
    have = [1 + int(x) for x in rng.integers(0, 199, slots)]
    n = rt.set_segments([(i, 0, c) for i, c in enumerate(have)])
    k, v = keys(rng, n, kvh, hd), rng.standard_normal((n, kvh, hd)).astype(np.float32)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
    wk, wv = oracle_mod.kv4_values(k, v)
    rt.set_segments([(i, c - 1, 1) for i, c in enumerate(have)])
    q = rng.standard_normal((slots, heads, hd)).astype(np.float32)
    put(rt, "q", q)
    put(rt, "o", np.zeros(q.size))
    rt.attention_seg("q", "kc", "vc", "o", heads, kvh, hd)
    got, first = get(rt, "o", q.shape), np.cumsum([0] + have)
    for i, c in enumerate(have):
        held = (w[first[i]:first[i + 1]].transpose(1, 0, 2) for w in (wk, wv))
        check(got[i:i + 1], q[i:i + 1], *held, heads, kvh, c, oracle_mod)


def test_pools_past_4_gib(rt, oracle_mod):
    """Pages at byte offsets past 32 bits: append, read-back, attention, and a page moved there and back."""
    rng = np.random.default_rng(4)
    heads, kvh, hd, page = 8, 4, 256, 64
    pages = (1 << 32) // (kvh * page * hd * 9 // 16) + 300
    high = [pages - 1, pages - 300, pages - 7, 3]
    put_ints(rt, "pt", [high])
    rt.set_paging("pt", page, 4, 1)
    caches(rt, pages * kvh, page, hd)
    n = rt.set_segments([(0, 0, 250)])
    k, v = keys(rng, n, kvh, hd), rng.standard_normal((n, kvh, hd)).astype(np.float32)
    put(rt, "k", k)
    put(rt, "v", v)
    rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
    for name in ("rk", "rv"):
        put(rt, name, np.zeros(k.size))
    rt.kv4_read_seg("kc", "vc", "rk", "rv", kvh, hd)
    wk, wv = oracle_mod.kv4_values(k, v)
    assert np.array_equal(get(rt, "rk", k.shape), wk.astype(np.float32)) and np.array_equal(get(rt, "rv", k.shape), wv.astype(np.float32))
    for segments in ([(0, 249, 1)], [(0, 230, 20)]):
        n = rt.set_segments(segments)
        q = rng.standard_normal((n, heads, hd)).astype(np.float32)
        put(rt, "q", q)
        put(rt, "o", np.zeros(q.size))
        rt.attention_seg("q", "kc", "vc", "o", heads, kvh, hd)
        check(get(rt, "o", q.shape), q, wk.transpose(1, 0, 2), wv.transpose(1, 0, 2), heads, kvh, segments[0][1] + 1, oracle_mod)


@pytest.mark.parametrize("heads,kvh,hd", [(24, 4, 256), (8, 2, 128), (6, 2, 96)])
@pytest.mark.parametrize("ntok", [1, 9])
def test_queries_and_results_at_any_float(torch, rt, heads, kvh, hd, ntok):
    """Queries and results that begin 4 bytes past an allocation give what aligned ones give, and nothing beside them is written."""
    rng = np.random.default_rng(heads)
    n = 600
    from vinf_3080ti_amd import _lib

    fill_rows = rng.standard_normal((n, kvh, hd)).astype(np.float32)
    caches(rt, kvh, n, hd)
    put(rt, "k", fill_rows)
    put(rt, "v", fill_rows[::-1])
    rt.kv_append("k", "v", "kc", "vc", kvh, n, hd, 0, n)
    lib = _lib.load()
    q = torch.from_numpy(rng.standard_normal((ntok * heads * hd,)).astype(np.float32)).cuda()
    nws = lib.vq_attention4_workspace_bytes(heads, kvh, hd, n - ntok + 1, ntok, 0)
    ws = torch.empty(nws, dtype=torch.uint8, device="cuda")
    results = []
    for off in (0, 1, 3):
        qq, o = torch.zeros(q.numel() + 8, device="cuda"), torch.full((q.numel() + 8,), 5.0, device="cuda")
        qq[off:off + q.numel()] = q
        for work, size in ((ws.data_ptr(), nws), (None, 0)):
            st = lib.vq_attention4_ws(qq.data_ptr() + 4 * off, rt.buffers["kc"].ptr, rt.buffers["vc"].ptr, o.data_ptr() + 4 * off, heads,
                                      kvh, hd, n, n - ntok + 1, ntok, 0, 0, work, size, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
            assert st == 0
            results.append(o[off:off + q.numel()].cpu().numpy().copy())
            rest = torch.cat([o[:off], o[off + q.numel():]])
            assert bool((rest == 5.0).all())
    for r in results[2:]:
        assert any(np.array_equal(r, x) for x in results[:2])


# ---- graphs -------------------------------------------------------------------------------------------------------


def test_two_graphs_and_eager_calls_in_turn(torch, rt):
    """Two captured passes (decode over four sequences; a prompt with verification behind it) that share the stream's workspace, replayed
    in turn with eager passes between: every replay gives the eager results bit for bit, from the inputs of its time."""
    rng = np.random.default_rng(9)
    heads, kvh, hd, page, slots, vocab = 8, 2, 128, 16, 5, 5000
    per = -(-600 // page)
    put_ints(rt, "pt", rng.permutation(per * slots).reshape(slots, per))
    rt.set_paging("pt", page, per, slots)
    caches(rt, per * slots * kvh, page, hd)
    n = rt.set_segments([(i, 0, 500 + i) for i in range(slots)])
    put(rt, "k", keys(rng, n, kvh, hd))
    put(rt, "v", rng.standard_normal((n, kvh, hd)))
    rt.kv_append_seg("k", "v", "kc", "vc", kvh, hd)
    rows = 40
    for name in ("q", "o"):
        put(rt, name, np.zeros(rows * heads * hd))
    for name in ("nk", "nv"):
        put(rt, name, np.zeros(rows * kvh * hd))
    put(rt, "logits", np.zeros((4, vocab)))
    put(rt, "u", np.zeros((4, 2)))
    put_ints(rt, "draft", [3, 4, 5])
    put_ints(rt, "tokens", [0] * 4)
    put_ints(rt, "counts", [0])

    def decode():
        rt.set_segments([(i, 500 + i, 1) for i in range(4)])
        rt.kv_append_seg("nk", "nv", "kc", "vc", kvh, hd)
        rt.attention_seg("q", "kc", "vc", "o", heads, kvh, hd)

    def prompt():
        rt.set_segments([(4, 490, rows)])
        rt.kv_append_seg("nk", "nv", "kc", "vc", kvh, hd)
        rt.attention_seg("q", "kc", "vc", "o", heads, kvh, hd)
        rt.verify_draft("logits", "draft", "u", "tokens", "counts", vocab, [3])

    def inputs(seed):
        r = np.random.default_rng(seed)
        for name, size in (("q", rows * heads * hd), ("nk", rows * kvh * hd), ("nv", rows * kvh * hd), ("logits", 4 * vocab)):
            rt.write(name, r.standard_normal(size).astype(np.float32).tobytes())
        rt.write("u", r.random(8).astype(np.float32).tobytes())
        rt.write("draft", r.integers(0, vocab, 3).astype(np.int32).tobytes())
        rt.write("o", np.full(rows * heads * hd, np.nan, np.float32).tobytes())
        rt.write("tokens", np.full(4, 88, np.int32).tobytes())

    def results():
        torch.cuda.synchronize()
        return [rt.read(x) for x in ("o", "tokens", "counts")]

    stream = torch.cuda.Stream()
    graphs = {}
    with torch.cuda.stream(stream):
        for f in (decode, prompt):
            f()  # (workspaces grow outside of a capture)
        torch.cuda.synchronize()
        for f in (decode, prompt):
            graphs[f] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graphs[f], stream=stream):
                f()
        for i, f in enumerate((decode, prompt, prompt, decode, decode, prompt)):
            inputs(i)
            f()
            want = results()
            inputs(i + 100)
            (prompt if f is decode else decode)()
            torch.cuda.synchronize()
            inputs(i)
            graphs[f].replay()
            got = results()
            for a, b, name in zip(got, want, ("o", "tokens", "counts")):
                if f is decode and name != "o":
                    continue
                assert a == b, (i, f.__name__, name)
