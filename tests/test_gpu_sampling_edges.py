"""Row sampling where its weights end: temperatures so small, or logits so large,
that the steps between neighbouring values are tens to hundreds of nats.

The reference is the definition in 64 bits with weights below e^-700 of the largest
taken as 0 (include/tinybrain_cuda.h).  Tokens are equal; probability and entropy
within 2^-23 of max(1, value), as in test_gpu_serving.py.
"""
import numpy as np
import pytest

from tests.test_gpu_serving import STAT_TOL, dev, sample_numpy, serving  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def check(serving, x, u, t, k=None, p=None, m=None):  # noqa: F811
    rows, V = x.shape
    full = lambda v, ty: None if v is None else dev(np.full(rows, v, ty))  # noqa: E731
    token, prob, ent = (o.cpu().numpy() for o in serving.sample_rows(
        dev(x), dev(u), temperature=full(t, np.float32), top_k=full(k, np.int32), top_p=full(p, np.float32),
        min_p=full(m, np.float32)))
    for i in range(rows):
        y = (x[i].astype(np.float64) - x[i].max().astype(np.float64)) / np.float64(np.float32(t))
        assert not ((y > -700.01) & (y < -699.99)).any()  # no value at the very end
        want = sample_numpy(np.where(y < -700, -np.inf, x[i]).astype(np.float32), u[i], np.float32(t), k or 0,
                            np.float32(1.0 if p is None else p), np.float32(m or 0.0))
        assert token[i] == want[0], (i, token[i], want)
        assert abs(prob[i] - want[1]) <= STAT_TOL and abs(ent[i] - want[2]) <= STAT_TOL * max(1.0, want[2]), (i, want)


# one step of the maximum is 47, 191, 950, 1900, 14 nats; then 2, 40, 80, 800 nats
@pytest.mark.parametrize("top,t", [(20.0, 4e-8), (20.0, 1e-8), (20.0, 2e-9), (20.0, 1e-9), (1e5, 5.5e-4), (1.1e7, 0.5),
                                   (3.3e7, 0.05), (1e8, 0.1), (1e8, 0.01)])
@pytest.mark.parametrize("V", [300, 40001, 400000])
@pytest.mark.parametrize("s", [dict(), dict(p=0.9), dict(k=40), dict(k=700, p=0.5, m=0.01), dict(p=0.9999999)])
def test_values_a_few_steps_below_the_maximum(serving, top, t, V, s):  # noqa: F811
    g = np.random.default_rng(V)
    top = np.float32(top)
    step = top - np.nextafter(top, np.float32(0))
    x = (top - step * g.integers(0, 60, (4, V)).astype(np.float32)).astype(np.float32)
    x[1] = top - step * np.maximum(1, g.integers(-200, 40, V)).astype(np.float32)  # one maximum, many just below
    x[1, V // 2] = top
    x[2, ::3] = -np.inf
    check(serving, x, np.array([0.0, 0.3, 0.7, 0.9999], np.float32), t, **s)
