"""Positions of a paged cache that have no page: they take no part in the
attention, whatever the pool holds, and a step whose reserve found too few pages
can be taken again.

Tolerances as in test_gpu_paged: 2^-10 max|v| for the weights' rounding and the
sums, 2^-11 |out| for the result's.
"""
import numpy as np
import pytest
from test_gpu_paged import EPS16, THETA, Batch, Pages, _attend, _i32, _some_cache

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _want(b, q, scale, window):
    """In 64 bits over the positions whose table entry names a page; zeros where
    a row has none."""
    g = b.q_heads // b.kvh
    out = np.zeros((b.rows, b.q_heads, b.D))
    tol = np.zeros_like(out)
    n_pages = b.pool.shape[1]
    for s, n in enumerate(b.lens):
        for j in range(b.n_new if n >= 0 else 0):
            p = np.arange(max(0, n + j + 1 - window) if window else 0, n + j + 1)
            ids = b.table[s, p // b.page]
            p, ids = p[(ids >= 0) & (ids < n_pages)], ids[(ids >= 0) & (ids < n_pages)]
            if not len(p):
                continue
            for h in range(b.kvh):
                k = b.pool[0, ids, h, p % b.page].astype(np.float64)
                v = b.pool[1, ids, h, p % b.page].astype(np.float64)
                z = q[s * b.n_new + j, h * g:(h + 1) * g].astype(np.float64) @ k.T * scale
                w = np.exp(z - z.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                sl = (s * b.n_new + j, slice(h * g, (h + 1) * g))
                out[sl] = w @ v
                tol[sl] = 2 * EPS16 * np.abs(v).max(0) + EPS16 * np.abs(out[sl])
    return out, tol


def _lose(b, entries, value=-1):
    """The table's `entries` (slot, entry) name no page any more.  The first and the
    last page, which such ids are nearest to, and those lost hold NaN: other pages
    take their place where a slot has them."""
    n = b.pool.shape[1]
    lost = {int(b.table[s, e]) for s, e in entries}
    for s, e in entries:
        b.table[s, e] = value
    held = set(b.table[(b.table >= 0) & (b.table < n)].tolist())
    spare = [p for p in range(1, n - 1) if p not in held]
    for page in sorted({0, n - 1} & held):
        other = spare.pop()
        b.pool[:, other] = b.pool[:, page]
        b.table[b.table == page] = other
        held = held - {page} | {other}
    for page in {0, n - 1, *lost} - held:
        b.pool[:, page] = np.nan
    b.kv.table.copy_(torch.from_numpy(b.table))
    b.kv.pool.copy_(torch.from_numpy(b.pool))


def _check(hip, b, window=0, slab_mb=32, extra=0.0):
    q = b.r.standard_normal((b.rows, b.q_heads, b.D)).astype(np.float16)
    got = _attend(hip, b, q, window, slab_mb)
    want, tol = _want(b, q, 1.0 / np.sqrt(b.D), window)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol + extra).all(), np.max(np.abs(got - want) / np.maximum(tol, 1e-9))


@pytest.mark.parametrize("value", [-1, -7, 10 ** 6, 2 ** 31 - 1])
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128), (12, 12, 64)], ids=str)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n_new", [1, 9])
def test_own_positions_without_a_page(hip, heads, page, value, n_new):
    """The first entry, one within, the last, several, all of a slot, and one
    behind the slot's tokens."""
    lens = [5 * page + 3, 9 * page, 3 * page - 1, 12 * page + 7, 40, 2 * page, 600]
    b = Batch(lens, n_new, heads, page, seed=31)
    last = [(n + n_new - 1) // page for n in lens]
    _lose(b, [(0, 0), (1, 4), (2, last[2]), (3, 0), (3, 1), (3, 5), (3, last[3]), (6, 2), (6, 3), (6, 4)]
          + [(4, e) for e in range(last[4] + 1)] + [(5, last[5] + 1)], value)
    _check(hip, b)
    _check(hip, b, window=3 * page + 5)
    _check(hip, b, slab_mb=0)


@pytest.mark.parametrize("seqs", [1, 2, 4, 9, 20])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 128])
def test_prefix_positions_without_a_page(hip, seqs, dim, page):
    """8 query heads a kv head: prefix tasks of 8 to 160 rows."""
    lens = [1024 + (7 * s) % 90 for s in range(seqs)]
    for lost in ([0], [3, 4], [1024 // page - 1], range(1024 // page)):
        b = Batch(lens, 1, (16, 2, dim), page, 1024, seed=seqs)
        _lose(b, [(s, e) for s in range(seqs) for e in lost])
        _check(hip, b)
        _check(hip, b, window=700)
        _check(hip, b, slab_mb=2.1 * seqs * 16 * (dim + 2) * 4 / (1 << 20))


@pytest.mark.parametrize("seqs", [3, 40, 70])
def test_positions_without_a_page_in_more_pages_than_are_kept(hip, seqs):
    """One part over 33008 positions in pages of 16, of which a task keeps 1024
    (64 a wave for few rows) at a time: pages missing at the ends of each."""
    b = Batch([33008 + s % 5 for s in range(seqs)], 1, (1, 1, 64), 16, 33008, seed=16)
    lost = [0, 63, 64, 65, 1022, 1023, 1024, 1025, 1026, 1027, 1500, 2046, 2047, 2048, 2062]
    _lose(b, [(s, e) for s in range(seqs) for e in lost])
    pick = [0, 33, seqs - 1] if seqs > 33 else [0, 1, 2]
    q = b.r.standard_normal((b.rows, 1, 64)).astype(np.float16)
    got = _attend(hip, b, q, slab_mb=2.2 * seqs * 66 * 4 / (1 << 20))
    assert np.isfinite(got).all()
    b.lens = [n if s in pick else -1 for s, n in enumerate(b.lens)]
    want, tol = _want(b, q, 1.0 / 8, 0)
    # fp32 sums of 33000 positions: 2^-24 a term, in the worst case all one way
    assert (np.abs(got - want)[pick] <= (tol + 33000 * 2.0 ** -24 * 4)[pick]).all()


def test_a_step_that_found_too_few_pages_is_taken_again(hip):
    """A captured step (reserve, append, attention, lengths) in a pool that runs
    out.  The failed step attends over the positions that have pages alone; its
    lengths are put back, a slot gives its pages up, and the same graph goes on:
    every step against the tokens' own history."""
    Q, H, D, page, S, n, V = 4, 2, 64, 16, 4, 5, 300
    kv = _some_cache(19, page, max_seqs=S, max_len=400, heads=H, dim=D, layers=1, seed=80)
    kv.pool.fill_(float("nan"))                                 # no token's values
    r = np.random.default_rng(81)
    z16, i32 = dict(dtype=torch.float16, device="cuda"), dict(dtype=torch.int32, device="cuda")
    qkv, q = torch.zeros((S * n, (Q + 2 * H) * D), **z16), torch.zeros((S * n, Q, D), **z16)
    out, status = torch.zeros((S * n, Q, D), **z16), torch.zeros(1, **i32)
    slab = torch.empty(8 << 20, dtype=torch.uint8, device="cuda")
    # certain drafts of probability 1: all n - 1 are kept, lengths grow by n
    p = torch.zeros((S, n, V), device="cuda")
    p[..., 5] = 1
    drafts, u = torch.full((S, n - 1), 5, **i32), torch.full((S, n), 0.5, device="cuda")
    acc, tok = torch.zeros(S, **i32), torch.zeros((S, n), **i32)
    kv.lens[:] = 0
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    hip.set_stream(st)
    try:
        hip.capture_begin()
        try:
            hip.kv_pages_reserve(kv, S, n, status)
            hip.rope_append_paged(kv, 0, qkv, q, S, n, Q, THETA)
            hip.attn_paged(kv, 0, q, out, S, n, Q, 0.125, slab)
            hip.verify_drafts(p, None, drafts, None, u, acc, tok, kv.lens, S, n - 1, V, slab)
        finally:
            g = hip.capture_end()
    finally:
        hip.use_torch_stream()
    freq = THETA ** (-np.arange(0, D, 2) / D)

    def rotate(x, pos):
        z = (x[..., :D // 2] + 1j * x[..., D // 2:]) * np.exp(1j * pos * freq)
        return np.concatenate([z.real, z.imag], -1)

    history, host, failed = {s: ([], []) for s in range(S)}, Pages(kv), 0
    for k in range(40):
        x = r.standard_normal((S * n, Q + 2 * H, D)).astype(np.float16)
        qkv.copy_(torch.from_numpy(x.reshape(S * n, -1)))
        before = kv.lens.clone()
        lens = before.tolist()
        torch.cuda.synchronize()
        g.launch()
        torch.cuda.synchronize()
        missing = int(status.item())
        assert missing == host.reserve(S, n)
        assert np.array_equal(kv.table.cpu().numpy(), host.table) and np.array_equal(kv.refs.cpu().numpy(), host.refs)
        got, x = out.cpu().numpy().astype(np.float64), x.astype(np.float64)
        for s in range(S):
            ks, vs = (list(h) for h in history[s])
            for j in range(n if lens[s] >= 0 else 0):
                pos = lens[s] + j
                if host.table[s, pos // page] >= 0:             # else the token is dropped
                    ks.append(rotate(x[s * n + j, Q:Q + H], pos).astype(np.float16).astype(np.float64))
                    vs.append(x[s * n + j, Q + H:])
                for h in range(Q):
                    want, tol = np.zeros(D), 0.0
                    if ks:
                        K, V_ = np.array(ks)[:, h // (Q // H)], np.array(vs)[:, h // (Q // H)]
                        z = K @ rotate(x[s * n + j, h], pos).astype(np.float16).astype(np.float64) * 0.125
                        w = np.exp(z - z.max())
                        want = w @ V_ / w.sum()
                        # once more the rounding of q and of the keys, as for several steps in test_gpu_paged
                        tol = 4 * EPS16 * np.abs(V_).max() + EPS16 * np.abs(want)
                    assert (np.abs(got[s * n + j, h] - want) <= tol).all(), (k, s, j, h)
            if not missing and lens[s] >= 0:
                history[s] = (ks, vs)
        if missing:
            failed += 1
            kv.lens.copy_(before)                               # as if the step had not been
            s = max(range(S), key=lambda s: lens[s])
            hip.kv_pages_free(kv, _i32([s]), 1)
            host.lens = before.cpu().numpy()
            host.free([s])
            kv.lens[s] = host.lens[s] = 0                       # another request takes the slot
            history[s] = ([], [])
        else:
            host.lens = kv.lens.cpu().numpy()
            assert host.lens.tolist() == [m + n for m in lens]
        torch.cuda.synchronize()
    assert failed >= 3
