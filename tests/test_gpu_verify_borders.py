"""Random numbers that fall on a border of the cumulative sum: a token without weight is not drawn there."""
from __future__ import annotations

import numpy as np
import pytest
from test_gpu_verify_draft import run

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


# Half of the tokens that have weight, all the same, lie before a gap and half behind it, and the random number is 1/2: the border
# at the gap is the target, so that the sums' roundings take either the last token before the gap or the first one behind it.


def rows(spans, vocab):
    """Logits 0 in each row's spans, -inf elsewhere."""
    l = np.full((len(spans), vocab), -np.inf, np.float32)
    for row, ss in zip(l, spans):
        for a, b in ss:
            row[a:b] = 0
    return l


def halves(rt, l, ends):
    u = np.full((len(l), 2), 0.5, np.float32)
    tokens, counts, _ = run(rt, l, np.zeros(0, np.int32), None, u, [0] * len(l), [1.0] * len(l))
    assert not counts.any()
    wrong = [(t, e) for t, e in zip(tokens.tolist(), ends) if t not in e]
    assert not wrong, wrong[:5]


def test_gaps_inside_a_chunk(rt):
    sizes = range(8, 1900)
    behind = [-(-n // 8) * 8 + 16 for n in sizes]
    halves(rt, rows([[(0, n), (b, b + n)] for n, b in zip(sizes, behind)], 4096), [(n - 1, b) for n, b in zip(sizes, behind)])


@pytest.mark.parametrize("m", [1, 3, 5])
def test_gaps_of_whole_chunks(rt, m):
    rng, spans, ends = np.random.default_rng(m), [], []
    for _ in range(200):
        n = [int(x) for x in rng.integers(1, 2000, m)]
        at = [2048 * i for i in range(2 * m + 1) if i != m]
        spans.append([(a, a + k) for a, k in zip(at, n + n[::-1])])
        ends.append((2048 * (m - 1) + n[-1] - 1, 2048 * (m + 1)))
    halves(rt, rows(spans, 2048 * (2 * m + 1)), ends)


def test_a_refused_draft_is_not_drawn(rt):
    """A draft chosen without chance, refused: as many tokens before it as behind it."""
    sizes = list(range(8, 1900, 8))
    l = np.repeat(rows([[(0, 2 * n + 1)] for n in sizes], 4096), 2, 0)
    u = np.tile(np.array([[0.999, 0.5], [0.5, 0.5]], np.float32), (len(sizes), 1))
    tokens, counts, _ = run(rt, l, np.array(sizes, np.int32), None, u, [1] * len(sizes), [1.0] * len(sizes))
    assert not counts.any()
    wrong = [(t, n) for t, n in zip(tokens[::2].tolist(), sizes) if t not in (n - 1, n + 1)]
    assert not wrong, wrong[:5]
