"""Log probabilities at the largest and the smallest temperatures that fp32 has, of logits as
large and as small.  Tolerances as in test_gpu_logprobs; log2(e) / T of the largest
temperatures is held to 2^-21 of itself, which 2^-22 |z| of an exponent covers with its
other roundings up to |z| 8 and 2^-20 (1 + sum p |z|) of ln L always."""
import numpy as np
import pytest

from test_gpu_logprobs import _check, _near, _run
from test_gpu_logprobs_cap import _capped
from test_gpu_logprobs_greedy import FORMS

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n", FORMS)
def test_logits_as_large_as_the_largest_caps(hip, rows, n):
    r = np.random.default_rng(n)
    x = (r.standard_normal((rows, n)) * 4e37).astype(np.float32)
    _capped(hip, x, np.full(rows, 2e37, np.float32), 2e38, x.argmax(1), 1, 4 << 20)


@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("t", [1e-38, 2e-38, 1e-30, 1e30, 1e37, 2e37, 1e38, 3e38])
def test_logits_of_the_temperature_s_size(hip, rows, n, t):
    """Of 0.7 temperatures, some of them tokens that may not be taken."""
    r = np.random.default_rng(n)
    x = (r.standard_normal((rows, n)).clip(-4, 4) * (0.7 * t if t < 1e38 else 5e37)).astype(np.float32)
    x[:, ::9] = -np.inf
    temp = np.full(rows, t, np.float32)
    for tokens, top in ((r.integers(0, n, rows), 0), (x.argmax(1), 1)):
        _check(hip, x, temp, 0.0, tokens, top)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("t", [1e30, 2e37, 3e38, np.inf])
def test_all_are_as_likely(hip, dtype, cap, rows, n, t):
    r = np.random.default_rng(n)
    x = (r.standard_normal((rows, n)) * 4).astype(dtype)
    x[:, 1::7] = -np.inf
    left = n - len(range(1, n, 7))
    tokens = np.where(np.arange(rows) % 2, 0, 1)                # of which one may not be taken
    lp, ent, _, _ = _run(hip, x, np.full(rows, t, np.float32), cap, tokens, 0, 4 << 20)
    # 2^-24 for each of 40 additions, the logarithm's and the result's roundings
    bound = 2.0 ** -18 + 2.0 ** -23 * np.log(left)
    _near(lp, np.where(tokens == 0, -np.log(left), -np.inf), np.full(rows, bound))
    _near(ent, np.full(rows, np.log(left)), np.full(rows, bound))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("rows,n", FORMS)
@pytest.mark.parametrize("t", [1e-45, 1e-40, 5e-39, 1e-37])
def test_the_largest_alone_next_to_no_temperature(hip, dtype, cap, rows, n, t):
    """Of two equal ones each has a half."""
    r = np.random.default_rng(n)
    x = (r.standard_normal((rows, n)) * 2).clip(-9, 9).astype(dtype)
    x[:, 1::7] = -np.inf
    x[:, n // 2], x[1::2, n - 3] = 10, 10
    two = np.arange(rows) % 2
    lp, ent, _, alt = _run(hip, x, np.full(rows, t, np.float32), cap, np.full(rows, n // 2), 1, 4 << 20)
    for got in (lp, alt[:, 0], -ent):
        _near(got, -np.log(1.0 + two), np.full(rows, 2.0 ** -20))
