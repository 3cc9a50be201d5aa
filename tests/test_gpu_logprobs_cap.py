"""Log probabilities under a cap: they are those of the probabilities that softmax_rows
gives, at every cap.

Tolerances.  As in test_gpu_logprobs, but of a capped logit f(x) = cap tanh(x / cap) each
is off by at most 2^-21 |f(x)| whatever the cap is: an exponent by 2^-20 max|f| / T more
(its own logit and the largest), a log probability by twice that (its exponent and ln L),
the entropy by (2 + sum p |z|) times that.
"""
import numpy as np
import pytest

from test_gpu_logprobs import _near, _run, _want
from test_gpu_logprobs_greedy import FORMS, _probabilities

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _capped(hip, x, temp, cap, tokens, top, slab):
    f = x.astype(np.float64)
    ok = np.isfinite(f)
    f[ok] = cap * np.tanh(f[ok] / cap)
    (lp, tol), (ent, etol), ids, (alt, atol) = _want(f, temp, 0.0, tokens, top)
    for r, t in enumerate(temp.astype(np.float64)):
        y = np.where(np.isfinite(f[r]), f[r], 0)
        d = 2.0 ** -20 * np.abs(y).max() / t
        z = np.where(np.isfinite(f[r]), (y - f[r].max()) / t, 0)
        q = np.where(np.isfinite(f[r]), np.exp(z), 0)
        q /= q.sum()
        tol[r] += 2 * d if np.isfinite(lp[r]) else 0
        atol[r] += 2 * d
        etol[r] += (2 + (q * np.abs(z)).sum()) * d
    got = _run(hip, x, temp, cap, tokens, top, slab)
    if top:
        assert np.array_equal(got[2], ids)
    _near(got[0], lp, tol)
    _near(got[1], ent, etol)
    _near(got[3], alt, atol)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [5.0, 30.0, 1e3, 1e4, 1e6, 2e38])
@pytest.mark.parametrize("rows,n", FORMS)
def test_every_cap(hip, dtype, cap, rows, n):
    """Logits of a hundredth, of a few and, at the cap's border, of all sizes; low temperatures."""
    r = np.random.default_rng(n)
    x = r.standard_normal((rows, n))
    size = np.array([0.01, 4.0, min(0.6 * cap, 20.0), min(cap, 40.0)])[np.arange(rows) % 4]
    x = (x * size[:, None]).astype(dtype)
    x[:, ::50] = -np.inf
    temp = np.array([0.01, 0.3, 1.0, 1.0], np.float32)[np.arange(rows) % 4]
    _capped(hip, x, temp, cap, r.integers(0, n, rows), 0, 4 << 20)
    _capped(hip, x, temp, cap, x.argmax(1), 1, 4 << 20)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [1e-30, 1e-39, 1e-44])
@pytest.mark.parametrize("rows,n", FORMS)
def test_caps_next_to_nothing(hip, dtype, cap, rows, n):
    """All that may be taken is as likely as any other."""
    r = np.random.default_rng(n)
    x = (r.standard_normal((rows, n)) * 4).astype(dtype)
    x[:, ::7], x[:, 1::7] = 0, -np.inf
    left = n - len(range(1, n, 7))
    tokens = np.where(np.arange(rows) % 2, 0, 2)
    lp, ent, _, _ = _run(hip, x, np.ones(rows, np.float32), cap, tokens, 0, 4 << 20)
    # 2^-24 for each of 40 additions, the logarithm's and the result's roundings
    bound = 2.0 ** -18 + 2.0 ** -23 * np.log(left)
    assert (np.abs(lp + np.log(left)) <= bound).all() and (np.abs(ent - np.log(left)) <= bound).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [5.0, 30.0, 1e3, 1e6])
@pytest.mark.parametrize("rows,n", FORMS)
def test_agrees_with_the_probabilities_under_a_cap(hip, dtype, cap, rows, n):
    r = np.random.default_rng(n + 1)
    x = (r.standard_normal((rows, n)) * 4).astype(dtype)
    temp = np.array([0.3, 1.0, 1.5, 7.0], np.float32)[np.arange(rows) % 4]
    p = _probabilities(hip, x, temp, cap).astype(np.float64)
    tokens = r.integers(0, n, rows)
    lp, _, ids, alt = _run(hip, x, temp, cap, tokens, 32, 4 << 20)
    size = np.minimum(np.abs(x.astype(np.float64)).max(1), cap)
    # both sides: 2^-20 (1 + |z|) of itself and the capped logits' part
    for got, want in ((alt, np.take_along_axis(p, ids.astype(np.int64), 1)), (lp[:, None], p[np.arange(rows), tokens][:, None])):
        got = got.astype(np.float64)
        rel = 2.0 ** -18 * (1 + np.minimum(np.abs(got), 100)) + 2 * 2.0 ** -19 * (size / temp)[:, None]
        assert (np.abs(np.exp(got) - want) <= want * rel + 2.0 ** -140).all()
