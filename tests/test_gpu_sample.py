"""Row softmax and the verification of drafted tokens against plain
implementations in 64 bits on the host.

Tolerances.  An fp32 probability is e^z / sum: z = (x - m) / T is off by two
roundings (2^-23 |z|), the exponential and the division by 2^-22 together, the
sum by as much; 2^-20 (1 + |z|) of the value covers them.  With a cap, tanh is
off by 2^-22, the logit by cap times that and three roundings, the exponent by
that over T.  Verification's whole numbers are equal: its products are exact in
fp64 and its sums differ from the host's by 2^-52, which no case comes near.
"""
import numpy as np
import pytest

from cima_amd.hip import E_INVALID, EngineError

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _slab():
    return torch.empty(16 << 20, dtype=torch.uint8, device="cuda")


def _softmax_want(x, temp, per, cap):
    z = x.astype(np.float64)
    if cap:
        z = cap * np.tanh(z / cap)
    t = np.repeat(temp, per)[:len(x)].astype(np.float64)[:, None]
    want, tol = np.zeros_like(z), np.zeros_like(z)
    for r in range(len(z)):
        m = z[r].max()
        if m == -np.inf:
            continue
        if t[r, 0] <= 0:
            want[r, np.flatnonzero(z[r] == m)[0]] = 1.0
            continue
        e = (z[r] - m) / t[r, 0]
        want[r] = np.exp(e) / np.exp(e).sum()
        e = np.where(np.isfinite(e), e, 0)
        tol[r] = want[r] * (2.0 ** -20 * (1 + np.abs(e)) + cap * 2.0 ** -20 / t[r, 0]) + 2.0 ** -140
    return want, tol


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("n", [1, 7, 8, 255, 2049, 8191, 8192, 8193, 32003, 151936])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_softmax(hip, dtype, n, cap):
    r = np.random.default_rng(n)
    rows, per = 5, 2
    x = (r.standard_normal((rows, n)) * 4).astype(dtype)
    x[1, ::3] = -np.inf
    x[2, n // 2] = 60000
    temp = np.array([0.7, 1.3, 0.05], np.float32)
    y = torch.full((rows, n), 7.0, device="cuda")
    hip.softmax_rows(_cuda(x), y, rows, n, _cuda(temp), per, cap, _slab())
    torch.cuda.synchronize()
    want, tol = _softmax_want(x, temp, per, cap)
    assert (np.abs(y.cpu().numpy() - want) <= tol).all()


def test_softmax_of_strided_starts_and_no_temp(hip):
    """Rows of odd length begin at every alignment; no temperature is 1."""
    r = np.random.default_rng(3)
    for dtype in (np.float16, np.float32):
        whole = (r.standard_normal(9 * 4099 + 5) * 3).astype(dtype)
        dev, y = _cuda(whole), torch.full((9 * 4099 + 8,), -3.0, device="cuda")
        for off in (0, 1, 3):
            hip.softmax_rows(dev[off:], y[off:], 9, 4099, None, 1, 0.0, _slab())
            torch.cuda.synchronize()
            want, tol = _softmax_want(whole[off:off + 9 * 4099].reshape(9, 4099), np.ones(9), 1, 0.0)
            got = y.cpu().numpy()
            assert (np.abs(got[off:off + 9 * 4099].reshape(9, 4099) - want) <= tol).all()
            assert (got[off + 9 * 4099:] == -3.0).all() and (off == 0 or (got[:off] < 1.01).all())


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,n", [(130, 33001), (128, 65536), (127, 40000), (130, 65537), (3, 32768), (3, 32769)])
def test_softmax_on_both_sides_of_every_path(hip, dtype, rows, n):
    """Rows to a workgroup or in parts, by their length and number."""
    r = np.random.default_rng(rows + n)
    x = (r.standard_normal((rows, n), np.float32) * 3).astype(dtype)
    temp = np.where(np.arange(rows) % 5 == 1, 0, r.uniform(0.4, 1.4, rows)).astype(np.float32)
    y = torch.empty((rows, n), device="cuda")
    hip.softmax_rows(_cuda(x), y, rows, n, _cuda(temp), 1, 0.0, _slab())
    torch.cuda.synchronize()
    y = y.cpu().numpy()
    for i in range(0, rows, 3):
        want, tol = _softmax_want(x[i:i + 1], temp[i:i + 1], 1, 0.0)
        assert (np.abs(y[i:i + 1] - want) <= tol).all(), i
    assert np.allclose(y.sum(1, dtype=np.float64), 1, atol=1e-5)


@pytest.mark.parametrize("n", [100, 5000, 40000])
def test_softmax_of_extreme_temperatures(hip, n):
    """Next to nothing: the largest logits alone share the row; infinite: all
    that are not -inf do.  In between nothing overflows."""
    x = np.random.default_rng(n).standard_normal((4, n)).astype(np.float32)
    x[:, 7] = x[:, 90] = 9.0
    x[:, 11] = -np.inf
    temp = np.array([1e-40, 1e-30, np.inf, 1e30], np.float32)
    y = torch.empty((4, n), device="cuda")
    hip.softmax_rows(_cuda(x), y, 4, n, _cuda(temp), 1, 0.0, _slab())
    torch.cuda.synchronize()
    y = y.cpu().numpy()
    want = np.zeros(n)
    want[[7, 90]] = 0.5
    assert (y[0] == want).all() and (y[1] == want).all()
    want = np.full(n, 1 / (n - 1))
    want[11] = 0
    # n terms in fp32, at most n / 1024 of them one after the other, then a division
    assert np.abs(y[2:] / want.max() - want / want.max()).max() < 2.0 ** -23 * (n / 1024 + 20)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("n", [32769, 40960, 151936])
def test_softmax_of_few_rows_by_the_slab(hip, dtype, cap, n):
    """A slab of 16 bytes for each 8192 logits suffices, a larger one lets the
    row be split further."""
    r = np.random.default_rng(n)
    x = (r.standard_normal((3, n), np.float32) * 4).astype(dtype)
    temp = np.array([0.8, 0, 1.3], np.float32)
    want, tol = _softmax_want(x, temp, 1, cap)
    for size in (3 * 16 * -(-n // 8192), 3 * 16 * -(-n // 2048) - 8, 3 * 16 * -(-n // 2048), 1 << 16):
        y = torch.full((3, n), 7.0, device="cuda")
        slab = torch.full((size + 64,), 0x5a, dtype=torch.uint8, device="cuda")
        hip.softmax_rows(_cuda(x), y, 3, n, _cuda(temp), 1, cap, slab[:size])
        torch.cuda.synchronize()
        assert (np.abs(y.cpu().numpy() - want) <= tol).all(), size
        assert (slab[size:] == 0x5a).all()


@pytest.mark.parametrize("n", [5, 9000, 40000])
def test_softmax_edges(hip, n):
    """Rows of -inf become zeros, temperature 0 takes the first of equal
    largest, NaN and +inf make a row NaN."""
    r = np.random.default_rng(n)
    x = r.standard_normal((8, n)).astype(np.float16)
    x[0] = -np.inf
    x[1] = -np.inf
    x[1, n - 1] = -5
    x[2, [1, n - 1]] = 99
    x[3, n - 2] = np.nan
    x[4, 2] = np.inf
    x[5, 0] = np.nan
    x[6] = -np.inf
    x[7] = -65504
    temp = np.array([1, 1, 0, 1, 1, 0, -1, 0.5], np.float32)
    y = torch.empty((8, n), device="cuda")
    hip.softmax_rows(_cuda(x), y, 8, n, _cuda(temp), 1, 0.0, _slab())
    torch.cuda.synchronize()
    g = y.cpu().numpy()
    assert not g[0].any() and not g[6].any()
    assert g[1, n - 1] == 1 and g[1].sum() == 1
    assert g[2, 1] == 1 and g[2].sum() == 1
    assert np.isnan(g[3]).all() and np.isnan(g[4]).all()
    top = np.nanargmax(x[5].astype(np.float32))
    assert g[5, top] == 1 and g[5].sum() == 1
    assert np.allclose(g[7], 1 / n, rtol=2.0 ** -20)


# ------------------------------------------------------------- verification

def _verify_want(p, q, drafts, counts, u, lens):
    S, K = drafts.shape
    V = p.shape[2]
    tokens, accepted = np.full((S, K + 1), -1, np.int32), np.zeros(S, np.int32)
    for s in range(S):
        if lens is not None and lens[s] < 0:
            continue
        n, a = counts[s], 0
        while a < n:
            d = int(drafts[s, a])
            if not 0 <= d < V:
                break
            qd = 1.0 if q is None else float(q[s, a, d])
            if not float(u[s, a]) * qd < float(p[s, a, d]):
                break
            tokens[s, a] = d
            a += 1
        accepted[s] = a
        clean = lambda v: np.where(v > 0, v, np.float32(0))  # noqa: E731
        r = clean(p[s, a])
        if a < n:
            left = clean(p[s, a] - q[s, a]) if q is not None else r.copy()
            if q is None and 0 <= drafts[s, a] < V:
                left[drafts[s, a]] = 0
            if left.any():
                r = left
        c = np.cumsum(r.astype(np.float64))
        if c[-1] > 0:
            tokens[s, a] = np.searchsorted(c, float(u[s, K]) * c[-1], side="right")
    return tokens, accepted


def _verify(hip, p, q, drafts, counts, u, lens=None, counts_null=False):
    S, K = drafts.shape
    V = p.shape[2]
    tokens = torch.full((S, K + 1), 99, dtype=torch.int32, device="cuda")
    accepted = torch.full((S,), 99, dtype=torch.int32, device="cuda")
    ld = None if lens is None else _cuda(lens.astype(np.int32))
    hip.verify_drafts(_cuda(p), None if q is None else _cuda(q), _cuda(drafts.astype(np.int32)),
                      None if counts_null else _cuda(counts.astype(np.int32)), _cuda(u), accepted, tokens, ld, S, K, V,
                      _slab())
    torch.cuda.synchronize()
    wt, wa = _verify_want(p, q, drafts, counts, u, lens)
    assert np.array_equal(accepted.cpu().numpy(), wa)
    assert np.array_equal(tokens.cpu().numpy(), wt)
    if lens is not None:
        assert np.array_equal(ld.cpu().numpy(), np.where(lens < 0, lens, lens + wa + 1))
    return wa


def _probs(r, *shape):
    x = r.standard_normal(shape) * 3
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("V", [1, 5, 2047, 2048, 2049, 20003, 128256])
@pytest.mark.parametrize("K", [0, 1, 4])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(hip, V, K, certain):
    r = np.random.default_rng(V + K)
    S = 12 if V < 100000 else 4
    p = _probs(r, S, K + 1, V)
    q = None if certain else _probs(r, S, K, V)
    if q is not None and K:
        q[: S // 2] = 0.7 * p[: S // 2, :K] + 0.3 * q[: S // 2]
    drafts = r.integers(0, V, (S, K))
    for s in range(S):
        for i in range(K):
            if s % 2:
                drafts[s, i] = p[s, i].argmax()
    counts = r.integers(0, K + 1, S)
    u = r.random((S, K + 1), np.float32)
    u[0] = 0
    u[S - 1] = 1 - 2.0 ** -24
    a = _verify(hip, p, q, drafts, counts, u)
    if K == 4 and V > 1000 and not certain:
        assert a.max() > 0
    _verify(hip, p, q, drafts, np.full(S, K), u, r.integers(-1, 3, S), counts_null=True)


def test_verify_edges(hip):
    """Equal distributions keep every draft; nothing left of p draws from p
    itself; empty, negative and NaN probabilities; ids outside the vocabulary."""
    r = np.random.default_rng(8)
    V, K = 5000, 70                                     # more drafts than a wave looks at together
    p = _probs(r, 6, K + 1, V)
    q = p[:, :K].copy()
    drafts = np.stack([[r.choice(V, p=p[s, i].astype(np.float64) / p[s, i].sum(dtype=np.float64)) for i in range(K)]
                       for s in range(6)])
    counts = np.array([K, K, K, 66, K, 0])
    u = r.random((6, K + 1), np.float32)
    p[2, 68] = 0                                        # refused there, and p holds nothing: -1
    p[3, 65] = p[3, 65] * 0.5                           # below q everywhere: refused or kept by u, then from p
    u[3, 65] = 0.9
    drafts[4, 3] = V
    drafts[1, 69] = -7
    p[0, K] = np.nan
    p[0, K, 17] = 0.25
    p[0, K, 18] = -3
    a = _verify(hip, p, q, drafts, counts, u)
    assert a.tolist() == [70, 69, 68, 65, 3, 0]
    # more drafts given than there is room for are cut
    tokens = torch.empty((6, K + 1), dtype=torch.int32, device="cuda")
    acc = torch.empty(6, dtype=torch.int32, device="cuda")
    hip.verify_drafts(_cuda(p), _cuda(q), _cuda(drafts.astype(np.int32)), _cuda(np.full(6, 1000, np.int32)), _cuda(u),
                      acc, tokens, None, 6, K, V, _slab())
    assert int(acc.max().item()) <= K


def test_verify_draws_every_token_by_its_share(hip):
    """Uniform numbers on a fine grid draw each token as often as its share of
    the residual says, to one draw."""
    V, S = 37, 4000
    r = np.random.default_rng(2)
    p1, q1 = _probs(r, V), _probs(r, V)
    left = np.maximum(p1 - q1, 0).astype(np.float64)
    p = np.broadcast_to(p1, (S, 2, V)).copy()
    q = np.broadcast_to(q1, (S, 1, V)).copy()
    d = int(np.argmin(p1 / q1))
    u = np.stack([np.full(S, 1 - 2.0 ** -24), (np.arange(S) + 0.5) / S], 1).astype(np.float32)
    tokens = torch.empty((S, 2), dtype=torch.int32, device="cuda")
    acc = torch.empty(S, dtype=torch.int32, device="cuda")
    hip.verify_drafts(_cuda(p), _cuda(q), _cuda(np.full((S, 1), d, np.int32)), None, _cuda(u), acc, tokens, None, S, 1, V,
                      _slab())
    assert int(acc.sum().item()) == 0
    got = np.bincount(tokens[:, 0].cpu().numpy(), minlength=V)
    assert (np.abs(got - S * left / left.sum()) <= 1.001).all()


def test_a_sampling_step_in_a_graph(hip):
    """Logits to probabilities to kept tokens and lengths, captured and replayed
    on new logits, against the same calls made one by one."""
    r = np.random.default_rng(12)
    S, K, V = 5, 3, 9001
    f = dict(device="cuda")
    xt, xd = torch.zeros((S * (K + 1), V), dtype=torch.float16, **f), torch.zeros((S * K, V), dtype=torch.float16, **f)
    p, q = torch.empty((S, K + 1, V), **f), torch.empty((S, K, V), **f)
    temp = _cuda(np.array([0.8, 1.0, 0.0, 1.2, 0.6], np.float32))
    drafts, u = torch.zeros((S, K), dtype=torch.int32, **f), torch.zeros((S, K + 1), **f)
    acc, tokens = torch.zeros(S, dtype=torch.int32, **f), torch.zeros((S, K + 1), dtype=torch.int32, **f)
    lens, slab = torch.zeros(S, dtype=torch.int32, **f), _slab()

    def calls():
        hip.softmax_rows(xt, p, S * (K + 1), V, temp, K + 1, 0.0, slab)
        hip.softmax_rows(xd, q, S * K, V, temp, K, 0.0, slab)
        hip.verify_drafts(p, q, drafts, None, u, acc, tokens, lens, S, K, V, slab)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    hip.set_stream(s)
    try:
        hip.capture_begin()
        try:
            calls()
        finally:
            g = hip.capture_end()
        for k in range(3):
            new = (r.standard_normal((S * (K + 1), V)) * 3).astype(np.float16)
            xt.copy_(_cuda(new))
            xd.copy_(_cuda(new.reshape(S, K + 1, V)[:, :K].reshape(S * K, V) + np.float16(0.3) * r.standard_normal((S * K, V)).astype(np.float16)))
            drafts.copy_(xd.view(S, K, V).argmax(2).int())
            u.copy_(torch.from_numpy(r.random((S, K + 1), np.float32)))
            lens.copy_(_cuda(np.array([5, 0, -1, 9, 100], np.int32)))
            torch.cuda.synchronize()
            g.launch()
            torch.cuda.synchronize()
            got = [t.cpu().clone() for t in (p, q, acc, tokens, lens)]
            lens.copy_(_cuda(np.array([5, 0, -1, 9, 100], np.int32)))
            torch.cuda.synchronize()
            calls()
            torch.cuda.synchronize()
            for a, b in zip(got, (p, q, acc, tokens, lens)):
                assert torch.equal(a, b.cpu())
            wt, wa = _verify_want(got[0].numpy(), got[1].numpy(), drafts.cpu().numpy(), np.full(S, K), u.cpu().numpy(),
                                  np.array([5, 0, -1, 9, 100]))
            assert np.array_equal(got[2].numpy(), wa) and np.array_equal(got[3].numpy(), wt)
    finally:
        hip.use_torch_stream()


def test_rows_behind_2_to_31_elements(hip):
    """Offsets of rows and probabilities in 64 bits."""
    rows, n = 17000, 128256
    assert rows * n > 2 ** 31
    x = torch.empty((rows, n), dtype=torch.float16, device="cuda")
    x[:-5] = 0
    x[-5:] = torch.randn((5, n), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    y = torch.empty((rows, n), device="cuda")
    hip.softmax_rows(x, y, rows, n, None, 1, 0.0, torch.empty(rows * 16 * 16, dtype=torch.uint8, device="cuda"))
    want, tol = _softmax_want(x[-5:].cpu().numpy(), np.ones(5, np.float32), 1, 0.0)
    assert (np.abs(y[-5:].cpu().numpy() - want) <= tol).all()
    assert (y[:-5:500] - 1 / n).abs().max().item() < 2.0 ** -20 / n
    del x, y
    S, K, V = 9000, 1, 128256
    assert S * (K + 1) * V > 2 ** 31
    p = torch.zeros((S, K + 1, V), device="cuda")
    at = (torch.arange(S, device="cuda")[:, None] * 14 + torch.arange(2, device="cuda")) % V
    p.scatter_(2, at[:, :, None], 1.0)
    drafts = at[:, :1].clone()
    drafts[1::2] += 1                                   # refused: all of p is at another token
    f = dict(device="cuda", dtype=torch.int32)
    acc, tokens = torch.empty(S, **f), torch.empty((S, 2), **f)
    hip.verify_drafts(p, None, drafts.int(), None, torch.full((S, 2), 0.5, device="cuda"), acc, tokens, None, S, K, V,
                      torch.empty(8 * S * 64, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    want = torch.where((torch.arange(S, device="cuda") % 2 == 0)[:, None], at, torch.stack([at[:, 0], at[:, 0] * 0 - 1], 1))
    assert torch.equal(acc, 1 - torch.arange(S, **f) % 2) and torch.equal(tokens.long(), want)
    del p
    torch.cuda.empty_cache()


def test_refusals(hip):
    x, y, slab = torch.zeros((2, 100), device="cuda"), torch.zeros((2, 100), device="cuda"), _slab()
    i = torch.zeros(200, dtype=torch.int32, device="cuda")

    def no(f, *a):
        with pytest.raises(EngineError) as e:
            f(*a)
        assert e.value.code == E_INVALID
    hip.softmax_rows(x, y, 2, 100, None, 1, 0.0, slab)
    hip.softmax_rows(x, y, 0, 100, None, 1, 0.0, slab)
    no(hip.softmax_rows, x, y, 3, 100, None, 1, 0.0, slab)
    no(hip.softmax_rows, x, y, -1, 100, None, 1, 0.0, slab)
    no(hip.softmax_rows, x, y, 2, 0, None, 1, 0.0, slab)
    no(hip.softmax_rows, x, y, 2, 100, None, 0, 0.0, slab)
    no(hip.softmax_rows, x, y, 2, 100, None, 1, -1.0, slab)
    no(hip.softmax_rows, x, y, 2, 100, y[0, :1], 1, 0.0, slab)
    no(hip.softmax_rows, x, y.half(), 2, 100, None, 1, 0.0, slab)
    no(hip.softmax_rows, x.bfloat16(), y, 2, 100, None, 1, 0.0, slab)
    hip.softmax_rows(x, y, 2, 100)                      # short rows need no slab
    long = torch.zeros(2 * 40000, device="cuda")
    hip.softmax_rows(long, long.clone(), 2, 40000, None, 1, 0.0, slab[:160])
    no(hip.softmax_rows, long, long.clone(), 2, 40000, None, 1, 0.0, slab[:152])
    no(hip.softmax_rows, long, long.clone(), 2, 40000)
    no(hip.softmax_rows, long, long.clone(), 2, 40000, None, 1, 0.0, slab[4:])
    hip.verify_drafts(x, y, i, None, y, i, i, None, 1, 1, 100, slab)
    hip.verify_drafts(x, y, i, None, y, i, i, None, 0, 1, 100, slab)
    no(hip.verify_drafts, x, y, i, None, y, i, i, None, 2, 1, 100, slab)
    no(hip.verify_drafts, x, y, i.long(), None, y, i, i, None, 1, 1, 100, slab)
    no(hip.verify_drafts, x, y, i, i.float(), y, i, i, None, 1, 1, 100, slab)
    no(hip.verify_drafts, None, y, i, None, y, i, i, None, 1, 1, 100, slab)
    no(hip.verify_drafts, x, y, None, None, y, i, i, None, 1, 1, 100, slab)
    no(hip.verify_drafts, x, y, i, None, y, i, i, None, 1, -1, 100, slab)
    no(hip.verify_drafts, x, y, i, None, y, i, i, None, 1, 1, 100, slab[:4])
    torch.cuda.synchronize()
