"""Log probabilities of tokens, entropies and likeliest alternatives of rows of
logits, against 64 bits on the host.

Tolerances.  An exponent z = (f(x) - m) / T is formed in fp32, off by 2^-22 |z| (its
difference, the scale and the product), under a cap by cap * 2^-20 / T more (tanh,
the quotient and the product, of the logit and of the largest); the exponential adds
2^-22, the fp32 sums of a part 2^-24 for each of at most 40 additions in a row.  ln L
is then off by at most 2^-20 (1 + sum p |z|) and a log probability by that, 2^-22 |z|
and its rounding; the entropy by 2^-20 (1 + sum p |z| (1 + |z|)).  Ids are equal.
"""
import numpy as np
import pytest

from cima_amd.hip import E_INVALID, EngineError

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SIZES = [1, 7, 255, 2049, 8192, 8193, 32003, 40000, 65537, 151936]


def _want(x, temp, cap, tokens, top):
    """(logprob, entropy, ids, logprobs of them), the first three's bounds as (value, bound)."""
    rows, n = x.shape
    z = x.astype(np.float64)
    if cap:
        ok = np.isfinite(z)
        z[ok] = cap * np.tanh(z[ok] / cap)
    lp, ent = np.full(rows, -np.inf), np.zeros(rows)
    ids, alt = np.full((rows, top), -1), np.full((rows, top), -np.inf)
    tol, etol, atol = np.zeros(rows), np.zeros(rows), np.zeros((rows, top))
    for r in range(rows):
        t, y = float(temp[r]), z[r]
        # by the logits, the lower id first; what may not be taken and NaN is not listed
        may = np.flatnonzero(x[r].astype(np.float64) > -np.inf)
        order = may[np.argsort(-x[r][may].astype(np.float64), kind="stable")][:top]
        ids[r, :len(order)] = order
        known = 0 <= tokens[r] < n
        if not t > 0:
            best = may[np.argmax(x[r][may].astype(np.float64))] if len(may) else -1
            lp[r] = 0 if known and tokens[r] == best else -np.inf
            alt[r, :min(1, len(order))] = 0
            continue
        bad = np.isnan(y).any() or np.isposinf(y).any()
        if bad or not len(may):
            ent[r] = np.nan if bad else 0
            if bad:
                alt[r, :len(order)] = np.nan
                lp[r] = np.nan if known and y[tokens[r]] != -np.inf else -np.inf
            continue
        e = np.where(y == -np.inf, -np.inf, (np.where(y == -np.inf, 0, y) - y.max()) / t)
        p = np.exp(e)
        L = np.log(p.sum())
        q = p / p.sum()
        a = np.where(p > 0, np.abs(np.where(p > 0, e, 0)), 0)
        each = 2.0 ** -22 * (1 + np.abs(e)) + cap * 2.0 ** -20 / t
        base = 2.0 ** -20 * (1 + (q * a).sum()) + cap * 2.0 ** -20 / t
        ent[r] = L - (q * np.where(p > 0, e, 0)).sum()
        etol[r] = 2.0 ** -20 * (1 + (q * a * (1 + a)).sum()) + cap * 2.0 ** -20 / t * (2 + (q * a).sum())
        alt[r, :len(order)], atol[r, :len(order)] = (e - L)[order], (base + each)[order]
        if known:
            lp[r] = (e - L)[tokens[r]]
            tol[r] = base + each[tokens[r]] if np.isfinite(lp[r]) else 0
    return (lp, tol), (ent, etol), ids, (alt, atol)


def _near(got, want, tol):
    got = got.astype(np.float64)
    odd = ~np.isfinite(want)
    assert np.array_equal(got[odd], want[odd], equal_nan=True), (got[odd], want[odd])
    assert (np.abs(got - want)[~odd] <= tol[~odd]).all(), np.max(np.abs(got - want)[~odd] / np.maximum(tol[~odd], 1e-12))


def _run(hip, x, temp, cap, tokens, top, slab, rows_per_temp=1):
    rows, n = x.shape
    lp, ent = (torch.full((rows + 1,), 7.0, device="cuda") for _ in range(2))
    ids = torch.full((rows + 1, top), 7, dtype=torch.int32, device="cuda")
    alt = torch.full((rows + 1, top), 7.0, device="cuda")
    hip.logprobs_rows(torch.from_numpy(x).cuda(), rows, n, torch.tensor(tokens, dtype=torch.int32, device="cuda"), lp, ent,
                      top, ids if top else None, alt if top else None,
                      None if temp is None else torch.from_numpy(temp).cuda(), rows_per_temp, cap,
                      torch.full((slab,), 255, dtype=torch.uint8, device="cuda") if slab else None)
    torch.cuda.synchronize()
    assert lp[-1] == 7 and ent[-1] == 7 and (ids[-1] == 7).all() and (alt[-1] == 7).all()
    return [v[:-1].cpu().numpy() for v in (lp, ent, ids, alt)]


def _check(hip, x, temp, cap, tokens, top, slabs=None):
    want = _want(x, temp, cap, tokens, top)
    rows, n = x.shape
    least = (16 + 256 * x.itemsize) * rows * -(-n // 8192) if n > 32768 else 0
    for slab in slabs or (least, 1 << 20):
        got = _run(hip, x, temp, cap, tokens, top, slab)
        assert np.array_equal(got[2], want[2])
        _near(got[0], *want[0])
        _near(got[1], *want[1])
        _near(got[3], *want[3])


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("n", SIZES)
def test_logprobs(hip, dtype, cap, n):
    """Rows whole and in parts of both sizes, masked tokens, every temperature."""
    r = np.random.default_rng(n)
    temp = np.array([0.7, 1.0, 5.0, np.inf, 0.0, 1.0, 1e-3, np.nan, -1.0, 1e-30], np.float32)
    x = (r.standard_normal((len(temp), n)) * 4).astype(dtype)
    x[1:4, ::3] = -np.inf
    x[5] = -np.inf                                              # nothing left
    x[6, n // 2:] = -np.inf
    tokens = r.integers(0, n, len(temp))
    tokens[0], tokens[4] = x[0].argmax(), x[4].argmax()
    for top in (0, 1, 5, 32):
        _check(hip, x, temp, cap, tokens, top)


@pytest.mark.parametrize("n", [40, 5000, 20000, 70000])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_equal_logits_go_by_their_ids(hip, dtype, n):
    """Rows of one value, of two, of few, of zeros of both signs, rising and falling:
    more equal ones than are looked at one by one among them."""
    r = np.random.default_rng(n)
    x = np.stack([np.full(n, 1.5), np.full(n, -np.inf), r.integers(0, 2, n) * 3.0, r.integers(-3, 4, n) * 1.0,
                  np.where(r.random(n) < 0.5, 0.0, -0.0), np.linspace(-8, 8, n), np.linspace(8, -8, n),
                  np.where(np.arange(n) % 97 == 5, 4.0, -np.inf), np.where(np.arange(n) == n - 1, 9.0, 1.0)]).astype(dtype)
    tokens = r.integers(0, n, len(x))
    for top in (1, 20, 32):
        _check(hip, x, np.full(len(x), 0.9, np.float32), 0.0, tokens, top)
    _check(hip, x, np.zeros(len(x), np.float32), 0.0, np.argmax(x, 1), 0)


@pytest.mark.parametrize("n", [30, 9000, 50000])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_rows_that_are_not_finite(hip, n, cap):
    r = np.random.default_rng(n)
    x = (r.standard_normal((7, n)) * 2).astype(np.float32)
    x[0, n // 3], x[1, n // 2], x[2] = np.nan, np.inf, np.nan
    x[3, :2], x[4, 5] = np.inf, np.nan
    x[4, ::2] = -np.inf
    x[5, 7], x[6, n - 1] = np.nan, np.inf
    temp = np.array([1, 1, 1, 1, 1, 0, 0], np.float32)
    _check(hip, x, temp, cap, np.array([3, n // 2, 0, 1, 4, 7, n - 1]), 8)


def test_tokens_that_do_not_exist_and_outputs_not_wanted(hip):
    r = np.random.default_rng(1)
    for n in (300, 45000):
        x = r.standard_normal((4, n)).astype(np.float16)
        tokens = np.array([-1, n, 5, 2 ** 31 - 1])
        _check(hip, x, np.ones(4, np.float32), 0.0, tokens, 3)
        xd, slab = torch.from_numpy(x).cuda(), torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
        full = _run(hip, x, None, 0.0, tokens, 3, 1 << 16)
        ent = torch.zeros(4, device="cuda")
        hip.logprobs_rows(xd, 4, n, entropy=ent, slab=slab)
        lp = torch.zeros(4, device="cuda")
        hip.logprobs_rows(xd, 4, n, torch.tensor(tokens, dtype=torch.int32, device="cuda"), lp, slab=slab)
        ids, alt = torch.zeros((4, 3), dtype=torch.int32, device="cuda"), torch.zeros((4, 3), device="cuda")
        hip.logprobs_rows(xd, 4, n, n_top=3, top_ids=ids, top_logprobs=alt, slab=slab)
        torch.cuda.synchronize()
        for a, b in zip((lp, ent, ids, alt), full):
            assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("n", [2000, 60000])
def test_rows_share_temperatures(hip, n):
    r = np.random.default_rng(n)
    x = (r.standard_normal((7, n)) * 3).astype(np.float32)
    temp = np.array([0.5, 0.0, 2.0], np.float32)
    tokens = r.integers(0, n, 7)
    want = _want(x, temp.repeat(3)[:7], 0.0, tokens, 4)
    got = _run(hip, x, temp, 0.0, tokens, 4, 1 << 20, rows_per_temp=3)
    assert np.array_equal(got[2], want[2])
    for g, w in ((got[0], want[0]), (got[1], want[1]), (got[3], want[3])):
        _near(g, *w)


def test_rows_at_odd_addresses(hip):
    """Rows that begin at any element, as slices of a larger tensor."""
    r = np.random.default_rng(3)
    for dtype in (np.float16, np.float32):
        flat = (r.standard_normal(3 * 8191 + 7) * 3).astype(dtype)
        base = torch.from_numpy(flat).cuda()
        for off in (1, 3, 7):
            x = flat[off:off + 3 * 8191].reshape(3, 8191)
            lp, ent = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
            hip.logprobs_rows(base[off:off + 3 * 8191], 3, 8191, torch.tensor([1, 2, 8190], dtype=torch.int32, device="cuda"),
                              lp, ent)
            torch.cuda.synchronize()
            want = _want(x, np.ones(3), 0.0, [1, 2, 8190], 0)
            _near(lp.cpu().numpy(), *want[0])
            _near(ent.cpu().numpy(), *want[1])


def test_agrees_with_the_probabilities(hip):
    """exp of the log probabilities is what softmax_rows writes."""
    r = np.random.default_rng(4)
    x = torch.from_numpy((r.standard_normal((5, 50000)) * 4).astype(np.float16)).cuda()
    temp = torch.tensor([0.3, 1.0, 1.5, 0.0, 7.0], device="cuda")
    slab = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    y = torch.empty((5, 50000), device="cuda")
    ids, alt = torch.zeros((5, 32), dtype=torch.int32, device="cuda"), torch.zeros((5, 32), device="cuda")
    hip.softmax_rows(x, y, 5, 50000, temp, 1, 0.0, slab)
    hip.logprobs_rows(x, 5, 50000, n_top=32, top_ids=ids, top_logprobs=alt, temp=temp, slab=slab)
    torch.cuda.synchronize()
    p = y.gather(1, ids.long()).double()
    # each is off by 2^-20 (1 + |z|) of itself
    assert ((alt.double().exp() - p).abs() <= p * 2.0 ** -18 * (1 + alt.abs().clamp(max=100)) + 2.0 ** -140).all()


def test_many_rows_and_a_replayed_graph(hip):
    """A captured call gives the same on every replay, with other logits too."""
    r = np.random.default_rng(5)
    rows, n, top = 300, 33000, 20
    xs = [(r.standard_normal((rows, n)) * 3).astype(np.float16) for _ in range(2)]
    tokens = r.integers(0, n, rows)
    temp = r.uniform(0.3, 1.5, rows).astype(np.float32)
    slab = (16 + 512) * rows * 5
    want = [_run(hip, x, temp, 0.0, tokens, top, slab) for x in xs]
    host = _want(xs[0][:20], temp, 0.0, tokens, top)
    assert np.array_equal(want[0][2][:20], host[2])
    _near(want[0][3][:20], *host[3])
    x = torch.from_numpy(xs[0]).cuda()
    td, tk = torch.from_numpy(temp).cuda(), torch.tensor(tokens, dtype=torch.int32, device="cuda")
    out = [torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"),
           torch.zeros((rows, top), dtype=torch.int32, device="cuda"), torch.zeros((rows, top), device="cuda")]
    work = torch.empty(slab, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    hip.set_stream(s)
    try:
        hip.capture_begin()
        try:
            hip.logprobs_rows(x, rows, n, tk, out[0], out[1], top, out[2], out[3], td, 1, 0.0, work)
        finally:
            g = hip.capture_end()
        for k in (0, 1, 0, 1):
            x.copy_(torch.from_numpy(xs[k]))
            for o in out:
                o.zero_()
            torch.cuda.synchronize()
            g.launch()
            torch.cuda.synchronize()
            for o, w in zip(out, want[k]):
                assert np.array_equal(o.cpu().numpy(), w)
    finally:
        hip.use_torch_stream()


@pytest.mark.parametrize("n", [2000, 8000, 20000, 60000, 151936])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_a_few_neighbours_may_be_taken(hip, dtype, n):
    """Rows of which one run of tokens is left, all of one sign, or as many as are
    wanted and one more or less."""
    r = np.random.default_rng(n)
    x = np.full((8, n), -np.inf)
    for i, (a, m) in enumerate(((0, 1000), (n // 3, 1500), (n - 31, 31), (5, 32), (n // 2, 33), (n // 2, 20), (7, 1993),
                                (0, n))):
        m = min(m, n - a)
        x[i, a:a + m] = -1 - np.abs(r.standard_normal(m)) * 3 if i % 2 else 100 + np.abs(r.standard_normal(m))
    x = x.astype(dtype)
    for top in (20, 32):
        _check(hip, x, np.full(8, 0.8, np.float32), 0.0, np.argmax(x, 1), top, slabs=(1 << 20,))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [8193, 12001, 32768])
def test_more_rows_than_compute_units(hip, dtype, n):
    """With a slab that holds their parts, one that does not and none."""
    r = np.random.default_rng(n)
    x = (r.standard_normal((270, n)) * 3).astype(dtype)
    x[5:100, ::2] = -np.inf
    temp = r.uniform(0.3, 1.5, 270).astype(np.float32)
    need = (16 + 256 * x.itemsize) * 270 * -(-n // 8192)
    _check(hip, x, temp, 0.0, r.integers(0, n, 270), 20, slabs=(need, need - 16, 0))


def test_refusals(hip):
    n = 40000
    x = torch.zeros((2, n), device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    lp, ent = torch.full((2,), 7.0, device="cuda"), torch.full((2,), 7.0, device="cuda")
    ids, alt = torch.full((2, 4), 7, dtype=torch.int32, device="cuda"), torch.full((2, 4), 7.0, device="cuda")
    slab = torch.empty(1040 * 2 * 5, dtype=torch.uint8, device="cuda")

    def no(*a, **kw):
        with pytest.raises(EngineError) as e:
            hip.logprobs_rows(*a, **kw)
        assert e.value.code == E_INVALID
    ok = dict(tokens=t, logprob=lp, entropy=ent, n_top=4, top_ids=ids, top_logprobs=alt, slab=slab)
    no(x, -1, n, **ok)
    no(x, 2, 0, **ok)
    no(x, 3, n, **ok)                                           # more rows than x holds
    no(x, 2, n, **{**ok, "n_top": 33})
    no(x, 2, n, **{**ok, "n_top": -1})
    no(x, 2, n, **{**ok, "n_top": 5})                           # more than top_ids holds
    no(x, 2, n, **{**ok, "top_ids": None})
    no(x, 2, n, **{**ok, "top_logprobs": None})
    no(x, 2, n, **{**ok, "tokens": None})                       # logprob wanted, of no tokens
    no(x, 2, n, **{**ok, "tokens": t.long()})
    no(x, 2, n, **{**ok, "logprob": lp.double()})
    no(x, 2, n, **{**ok, "slab": None})
    no(x, 2, n, **{**ok, "slab": slab[:-1]})
    no(x, 2, n, **{**ok, "slab": slab[1:]})
    no(x, 2, n, **ok, cap=-1.0)
    no(x, 2, n, **ok, cap=float("inf"))
    no(x, 2, n, **ok, rows_per_temp=0)
    no(x, 2, n, **ok, temp=torch.ones(1, device="cuda"))
    no(x.double(), 2, n, **ok)
    torch.cuda.synchronize()
    assert (lp == 7).all() and (ent == 7).all() and (ids == 7).all() and (alt == 7).all()
    hip.logprobs_rows(x, 0, n, **ok)                            # nothing to do
    torch.cuda.synchronize()
    assert (lp == 7).all()
    hip.logprobs_rows(x, 2, n, **ok)
    torch.cuda.synchronize()
    assert torch.equal(ids.cpu(), torch.arange(4, dtype=torch.int32).repeat(2, 1))
