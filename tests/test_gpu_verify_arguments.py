"""The kinds of numbers that verify_draft's temperature may be."""
from __future__ import annotations

import numpy as np
import pytest
from test_gpu_verify_draft import case, run

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


@pytest.mark.parametrize("kind", [np.float32, np.float16, np.float64, np.int64, int, lambda t: [np.float32(t)] * 3, lambda t: np.full(3, t)])
def test_temperatures_of_any_kind(rt, kind):
    rng = np.random.default_rng(2)
    l, draft, _, u = case(rng, 500, [2, 0, 1], [2.0] * 3, False)
    want = run(rt, l, draft, None, u, [2, 0, 1], [2.0] * 3)
    got = run(rt, l, draft, None, u, [2, 0, 1], kind(2))
    for a, b in zip(got, want):
        assert np.array_equal(a.view(np.int32), b.view(np.int32))
    with pytest.raises(ValueError):
        run(rt, l, draft, None, u, [2, 0, 1], np.float32(-1))
