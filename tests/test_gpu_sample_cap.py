"""Capped softmax of rows that hold infinite logits and NaN: the cap is taken of
finite logits, a logit of -inf (a token that may not be taken) keeps no
probability at any temperature.

Tolerances as in test_gpu_sample: a finite logit of size x becomes cap * tanh(x
/ cap), off by cap * (2^-22 + 2^-23) (tanh, the quotient and the product), the
exponent by that and the largest logit's over T; 2^-20 (1 + |z|) covers the
difference, the exponential, the sum and the division.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _want(x, temp, cap):
    """Rows in 64 bits and the bound on their error."""
    z = x.astype(np.float64)
    finite = np.isfinite(z)
    z[finite] = cap * np.tanh(z[finite] / cap)
    want, tol = np.zeros_like(z), np.zeros_like(z)
    for r, t in enumerate(temp.astype(np.float64)):
        m = z[r].max()
        if m == -np.inf:
            continue
        if t <= 0:
            want[r, np.flatnonzero(z[r] == m)[0]] = 1.0
            continue
        e = np.where(z[r] == -np.inf, -np.inf, (np.where(z[r] == -np.inf, m, z[r]) - m) / t)
        p = np.exp(e)
        want[r] = p / p.sum()
        tol[r] = want[r] * (2.0 ** -20 * (1 + np.abs(np.where(p > 0, e, 0))) + cap * 2.0 ** -20 / t) + 2.0 ** -140 * (p > 0)
    return want, tol


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [1, 7, 255, 2049, 8192, 8193, 32003, 40000, 65537, 151936])
@pytest.mark.parametrize("cap", [30.0, 2.0])
def test_masked_tokens_of_a_capped_row_have_no_probability(hip, dtype, n, cap):
    """Whole rows and rows in parts of both sizes; warm, hot and infinite
    temperatures, at which -cap would weigh most."""
    r = np.random.default_rng(n)
    temp = np.array([0.7, 1.0, 5.0, np.inf, 0.0, 1.0, 1e-3], np.float32)
    x = (r.standard_normal((len(temp), n)) * 4).astype(dtype)
    x[:, ::3] = -np.inf
    x[0] = (r.standard_normal(n) * 4).astype(dtype)             # nothing masked
    x[5] = -np.inf                                              # nothing left
    for slab in (16 * 7 * -(-n // 8192), 1 << 16):
        y = torch.full((len(temp), n), 7.0, device="cuda")
        hip.softmax_rows(torch.from_numpy(x).cuda(), y, len(temp), n, torch.from_numpy(temp).cuda(), 1, cap,
                         torch.empty(slab, dtype=torch.uint8, device="cuda"))
        torch.cuda.synchronize()
        got = y.cpu().numpy()
        want, tol = _want(x, temp, cap)
        assert (got[np.isneginf(x)] == 0).all()
        assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [5, 9000, 40000])
def test_nan_and_infinity_of_a_capped_row(hip, dtype, n):
    """NaN and +inf make a row NaN; at temperature 0 +inf is the largest, NaN the
    lowest, and the first of equal capped logits is taken."""
    r = np.random.default_rng(n)
    x = r.standard_normal((6, n)).astype(dtype)
    x[0, n - 2] = np.nan
    x[1, 2] = np.inf
    x[2, [1, n - 1]] = 60000                                    # both cap to the same number
    x[3, 0], x[3, n - 1], x[3, 1] = np.nan, np.inf, 60000
    x[4, 0] = np.nan
    x[5] = -np.inf
    temp = np.array([1, 1, 0, 0, -1, 0], np.float32)
    y = torch.empty((6, n), device="cuda")
    hip.softmax_rows(torch.from_numpy(x).cuda(), y, 6, n, torch.from_numpy(temp).cuda(), 1, 30.0,
                     torch.empty(1 << 16, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    got = y.cpu().numpy()
    assert np.isnan(got[0]).all() and np.isnan(got[1]).all()
    for row, at in ((2, 1), (3, n - 1), (4, np.nanargmax(x[4].astype(np.float32)))):
        assert got[row, at] == 1 and got[row].sum() == 1
    assert not got[5].any()


def test_masked_tokens_are_not_drawn(hip):
    """A capped row at an infinite temperature is even over the tokens that are
    left; drawing from it by numbers over all of [0, 1) takes no other."""
    S, V, cap = 512, 900, 30.0
    x = np.random.default_rng(4).standard_normal((S, V)).astype(np.float16)
    left = np.arange(V) % 7 == 3
    x[:, ~left] = -np.inf
    p = torch.empty((S, 1, V), device="cuda")
    slab = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    temp = torch.full((1,), float("inf"), device="cuda")
    hip.softmax_rows(torch.from_numpy(x).cuda(), p, S, V, temp, S, cap, slab)
    u = ((torch.arange(S, device="cuda") + 0.5) / S)[:, None]
    accepted, tokens = (torch.zeros(S, dtype=torch.int32, device="cuda") for _ in range(2))
    hip.verify_drafts(p, None, None, None, u, accepted, tokens, None, S, 0, V, slab)
    torch.cuda.synchronize()
    got = tokens.cpu().numpy()
    assert left[got].all() and len(np.unique(got)) == left.sum()


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("n", [5, 9000, 40000])
def test_a_temperature_that_is_no_number_takes_the_largest(hip, n, cap):
    x = np.random.default_rng(n).standard_normal((3, n)).astype(np.float16)
    x[:, :2] = -np.inf
    temp = np.array([np.nan, -0.0, -np.inf], np.float32)
    y = torch.empty((3, n), device="cuda")
    hip.softmax_rows(torch.from_numpy(x).cuda(), y, 3, n, torch.from_numpy(temp).cuda(), 1, cap,
                     torch.empty(1 << 16, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    want = np.zeros((3, n))
    want[np.arange(3), x.argmax(1)] = 1
    assert np.array_equal(y.cpu().numpy(), want)
