"""Log probabilities under a cap where one token is left (a temperature of 0 or below, or NaN): the
one that softmax_rows gives 1."""
import numpy as np
import pytest

from test_gpu_logprobs import _run

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# rows of one workgroup in its three forms, rows in parts of 2048 and of 8192
FORMS = [(4, 700), (4, 5000), (4, 20011), (4, 50001), (150, 40000)]


def _probabilities(hip, x, temp, cap):
    rows, n = x.shape
    y = torch.empty((rows, n), device="cuda")
    hip.softmax_rows(torch.from_numpy(x).cuda(), y, rows, n, torch.from_numpy(temp).cuda(), 1, cap,
                     torch.empty(8 << 20, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    return y.cpu().numpy()


def _capped_rows(rows, n, dtype, cap, seed):
    """Rows whose largest logits are the same under the cap, the first of them not the
    largest: pairs, many, fp32 neighbours, beside others that may not be taken."""
    r = np.random.default_rng(seed)
    x = (r.standard_normal((rows, n)) * 4).astype(dtype)
    for i in range(rows):
        kind = i % 10
        if kind == 0:
            x[i, n // 3], x[i, n - 2] = 280, 300
        elif kind == 1:                                  # rising: the first is the least of them
            x[i] = np.linspace(250, 900, n)
        elif kind == 2:
            x[i, 5:45] = np.arange(400, 440)             # more than are listed
        elif kind == 3 and dtype == np.float32:          # neighbours: the cap makes many equal
            m = min(n, 600) - 3
            x[i, 2:2 + m] = np.float32(2 * cap) + np.arange(m) * np.spacing(np.float32(2 * cap))
        elif kind == 4:
            x[i, ::2], x[i, 1::2] = -np.inf, -5
            x[i, 3], x[i, n - 1 - (n - 1) % 2 - 1] = 270, 290
        elif kind == 5:
            x[i] = -np.inf
        elif kind == 6:
            x[i, 1], x[i, n // 2], x[i, 7] = np.nan, 300, 280
        elif kind == 7:
            x[i, 9], x[i, 4] = np.inf, 300
        elif kind == 8:
            x[i] = np.linspace(-250, -900, n)
            x[i, 0] = -np.inf
    return x


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [5.0, 30.0])
@pytest.mark.parametrize("rows,n", FORMS)
def test_the_token_that_is_left(hip, dtype, cap, rows, n):
    """At temperatures of 0 and below, or NaN: the token that softmax_rows gives 1 has 0 and comes
    first, the others follow by their logits."""
    rows = max(rows, 10)
    x = _capped_rows(rows, n, dtype, cap, n)
    temp = np.array([0.0, -1.0, np.nan], np.float32)[np.arange(rows) % 3]
    p = _probabilities(hip, x, temp, cap)
    best = np.where(p.max(1) == 1, p.argmax(1), -1)
    assert ((p != 0).sum(1) == (best >= 0)).all()
    largest = np.nanargmax(np.where(np.isnan(x), -np.inf, x), 1)
    assert (largest != best).sum() >= rows // 3          # as the rows are meant
    for tokens, top in ((best, 0), (largest, 1), (best, 5), (largest, 32)):
        for slab in ((16 + 256 * x.itemsize) * rows * -(-n // 8192) if n > 32768 else 0, 4 << 20):
            lp, ent, ids, alt = _run(hip, x, temp, cap, tokens, top, slab)
            assert np.array_equal(lp, np.where((tokens == best) & (best >= 0), 0, -np.inf))
            assert not ent.any()
            for i in range(rows):
                may = np.flatnonzero(x[i].astype(np.float64) > -np.inf)
                order = may[np.argsort(-x[i][may].astype(np.float64), kind="stable")]
                order = np.concatenate([[best[i]], order[order != best[i]]])[:top] if len(may) else order
                assert np.array_equal(ids[i, :len(order)], order), (i, ids[i], order)
                assert (ids[i, len(order):] == -1).all()
                want = np.full(top, -np.inf)
                want[:1] = 0 if len(order) else -np.inf
                assert np.array_equal(alt[i], want)


@pytest.mark.parametrize("cap", [2e38, 3e37, 1.0, 1e-37])
@pytest.mark.parametrize("size", [0.01, 1e-5, 1e-30, 1e-38, 1e-41])
@pytest.mark.parametrize("rows,n", FORMS)
def test_quotients_next_to_nothing(hip, cap, size, rows, n):
    """x / cap among the numbers below 2^-126, which are far apart: logits whose capped values are
    the same though they differ by more than roundings do elsewhere."""
    r = np.random.default_rng(n)
    x = (size * (1 - 1e-3 * r.random((rows, n)) ** 8)).astype(np.float32)
    x[1::2] = np.sort(x[1::2], 1)
    temp = np.zeros(rows, np.float32)
    p = _probabilities(hip, x, temp, cap)
    best = np.where(p.max(1) == 1, p.argmax(1), -1)
    lp, _, ids, alt = _run(hip, x, temp, cap, best, 3, 4 << 20)
    assert np.array_equal(lp, np.where(best >= 0, 0, -np.inf))
    assert np.array_equal(ids[:, 0], best) and (alt[:, 0] == 0).all()
