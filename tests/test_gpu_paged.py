"""A batch over the paged cache: RoPE with append, attention with a shared
prefix, page operations, and a run of them together, against plain
implementations in 64 bits on the host.

Tolerances.  A result rounded to f16 is off by half a step, 2^-11 of its value.
Attention also rounds each probability to f16 (2^-11 of it) before the product
with the values: the weighted sum is then off by at most 2^-11 sum(w |v|) /
sum(w), and its fp32 sums by far less (2^-24 times the number of positions,
below 2^-11 up to 8192 of them); 2^-10 max|v| covers both, 2^-11 |out| the
last rounding.  The rotation is rounded once, its fp32 products and the fp32
sine and cosine (2^-23 each) are covered by 2^-20 (|a| + |b|).
"""
import numpy as np
import pytest

from cima_amd.hip import E_INVALID, EngineError

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS16 = 2.0 ** -11
THETA = 1e6


def _i32(v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


class Batch:
    """A host-side cache of seqs slots with the given lengths, whose first
    `prefix` positions are shared pages; `n_new` tokens are held on top.  Rows of
    the table have `spare` entries more than the longest slot needs."""

    def __init__(self, lens, n_new, heads, page, prefix=0, layers=1, seed=0, poison=None, spare=1):
        from cima_amd.paged import PagedKV

        r = np.random.default_rng(seed)
        self.q_heads, kvh, D = heads
        self.lens, self.n_new, self.page, self.pp = list(lens), n_new, page, prefix // page
        S = len(lens)
        held = [max(0, -(-(n + n_new) // page) - self.pp) if n >= 0 else 0 for n in lens]
        stride = self.pp + max(held + [1]) + spare
        n_pages = self.pp + sum(held) + 3
        ids = r.permutation(n_pages)
        self.table = np.full((S, stride), -1, np.int32)
        at = self.pp
        for s in range(S):
            if lens[s] < 0:
                continue
            self.table[s, :self.pp] = ids[:self.pp]
            self.table[s, self.pp:self.pp + held[s]] = ids[at:at + held[s]]
            at += held[s]
        pool = r.standard_normal((2 * layers, n_pages, kvh, page, D)).astype(np.float16)
        if poison is not None:  # what no row sees
            seen = np.zeros((n_pages, page), bool)
            for s in range(S):
                if lens[s] >= 0:
                    for p in range(max(0, poison[s]), lens[s] + n_new):
                        seen[self.table[s, p // page], p % page] = True
            pool[:, ~seen[:, None, :, None].repeat(kvh, 1)[..., 0]] = np.nan
        self.pool = pool
        refs = np.zeros(n_pages, np.int32)
        np.add.at(refs, self.table[self.table >= 0], 1)
        self.refs = refs
        self.kv = PagedKV(torch.from_numpy(pool).cuda(), _i32(refs), _i32(self.table), _i32(lens))
        self.rows = S * n_new
        self.D, self.kvh, self.r = D, kvh, r

    def want(self, q, scale, window, layer=0):
        """[rows, q_heads, D] in float64 and the bound on the error."""
        g = self.q_heads // self.kvh
        out = np.zeros((self.rows, self.q_heads, self.D))
        tol = np.zeros_like(out)
        for s, n in enumerate(self.lens):
            if n < 0:
                continue
            for j in range(self.n_new):
                hi = n + j + 1
                lo = max(0, hi - window) if window else 0
                p = np.arange(lo, hi)
                ids = self.table[s, p // self.page]
                for h in range(self.kvh):
                    k = self.pool[2 * layer, ids, h, p % self.page].astype(np.float64)
                    v = self.pool[2 * layer + 1, ids, h, p % self.page].astype(np.float64)
                    z = q[s * self.n_new + j, h * g:(h + 1) * g].astype(np.float64) @ k.T * scale
                    w = np.exp(z - z.max(1, keepdims=True))
                    w /= w.sum(1, keepdims=True)
                    sl = (s * self.n_new + j, slice(h * g, (h + 1) * g))
                    out[sl] = w @ v
                    tol[sl] = 2 * EPS16 * np.abs(v).max(0) + EPS16 * np.abs(out[sl])
        return out, tol


def _attend(hip, b, q, window=0, slab_mb=32, scale=None, prefix_slot=None, layer=0):
    scale = scale or 1.0 / np.sqrt(b.D)
    out = torch.full((b.rows, b.q_heads, b.D), float("nan"), dtype=torch.float16, device="cuda")
    slab = torch.full((int(slab_mb * (1 << 20)) // 4,), float("nan"), device="cuda") if slab_mb else None
    slot = prefix_slot if prefix_slot is not None else next((i for i, n in enumerate(b.lens) if n >= 0), 0)
    hip.attn_paged(b.kv, layer, torch.from_numpy(q).cuda(), out, len(b.lens), b.n_new, b.q_heads, scale, slab,
                   prefix_pages=b.pp, prefix_slot=slot, window=window)
    torch.cuda.synchronize()
    return out.cpu().numpy().astype(np.float64)


def _check(hip, b, window=0, slab_mb=32, layer=0):
    q = b.r.standard_normal((b.rows, b.q_heads, b.D)).astype(np.float16)
    got = _attend(hip, b, q, window, slab_mb, layer=layer)
    want, tol = b.want(q, 1.0 / np.sqrt(b.D), window, layer)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / np.maximum(tol, 1e-9))


HEADS = [(14, 2, 64), (32, 8, 128), (12, 12, 64), (16, 1, 128), (8, 8, 128)]


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attention_own_pages_only(hip, heads, page):
    _check(hip, Batch([0, 1, 15, 16, 63, 130, 517], 1, heads, page, seed=1))


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("page,prefix", [(16, 16), (16, 48), (32, 320), (128, 1024), (256, 2048)])
def test_attention_shared_prefix(hip, heads, page, prefix):
    _check(hip, Batch([prefix, prefix + 1, prefix + 40, prefix + 200, prefix + page], 1, heads, page, prefix, seed=2))


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("page,prefix", [(16, 16), (16, 48), (32, 320)])
def test_attention_short_prefix_in_a_long_table(hip, heads, page, prefix):
    """The same slots in tables of more than 640 positions: the prefix has tasks
    of its own."""
    for seqs in (1, 5):
        lens = [prefix, prefix + 1, prefix + 40, prefix + 200, prefix + page][:seqs]
        _check(hip, Batch(lens, 1, heads, page, prefix, seed=2, spare=700 // page))
    _check(hip, Batch([prefix + 3, prefix + 90, -1], 4, heads, page, prefix, seed=23, spare=700 // page), window=60)


@pytest.mark.parametrize("seqs", [1, 9, 20, 40, 80])
def test_attention_every_row_tile(hip, seqs):
    """8 query heads a kv head: 8 to 640 rows, every tile of the prefix tasks."""
    lens = [640 + (7 * s) % 90 for s in range(seqs)]
    for dim in (64, 128):
        _check(hip, Batch(lens, 1, (16, 2, dim), 64, 640, seed=seqs))


@pytest.mark.parametrize("n_new", [2, 5, 8, 33])
def test_attention_drafts(hip, n_new):
    _check(hip, Batch([96, 100, 111, 250], n_new, (14, 2, 64), 32, 96, seed=3))
    _check(hip, Batch([0, 5, 31], n_new, (8, 2, 128), 32, 0, seed=4))


@pytest.mark.parametrize("window", [1, 7, 64, 100, 300, 5000])
def test_attention_window(hip, window):
    lens = [256, 300, 333, 480, 700]
    for n_new in (1, 4):
        _check(hip, Batch(lens, n_new, (14, 2, 64), 64, 256, seed=5), window)
        _check(hip, Batch(lens, n_new, (8, 2, 128), 64, 256, seed=6), window)


def test_attention_free_slots_and_short_ones(hip):
    """Free slots give zeros, also first, last and all of them; a slot shorter
    than the prefix sees what it has of it."""
    for lens in ([-1, 70, -1, 90], [64, -1, 64], [-1, -1]):
        b = Batch(lens, 2, (8, 2, 128), 32, 64 if max(lens) > 0 else 0, seed=7)
        _check(hip, b)
    _check(hip, Batch([10, 64, 130, 0], 1, (14, 2, 64), 32, 64, seed=8))


@pytest.mark.parametrize("window", [0, 50])
def test_attention_ignores_what_no_row_sees(hip, window):
    """Rows behind a slot's last token, whole unused pages and what lies before
    every row's window hold NaN."""
    lens, n_new = [200, 131, 160], 3
    low = [n + 1 - window if window else 0 for n in lens]
    b = Batch(lens, n_new, (8, 2, 128), 64, 0, seed=9, poison=low)
    assert np.isnan(b.pool).any()
    _check(hip, b, window)


@pytest.mark.parametrize("slab_mb", [0.07, 0.15, 0.5, 64])
def test_attention_with_small_and_large_slabs(hip, slab_mb):
    _check(hip, Batch([512, 700, 600, 555], 1, (14, 2, 64), 64, 512, seed=10), slab_mb=slab_mb)
    _check(hip, Batch([512, 700, 600, 555], 1, (14, 2, 64), 64, 0, seed=10), slab_mb=slab_mb)


def test_attention_without_a_slab(hip):
    _check(hip, Batch([512, 700, 60], 1, (14, 2, 64), 64, 0, seed=11), slab_mb=0)


def test_attention_second_layer_and_many_pages(hip):
    """More pages than a task keeps ids of at a time (1024), unsplit."""
    b = Batch([17000], 1, (2, 2, 64), 16, 0, layers=2, seed=12)
    _check(hip, b, slab_mb=0, layer=1)
    _check(hip, Batch([33000, 32768], 1, (2, 2, 64), 16, 32768, seed=13), slab_mb=0.01)


@pytest.mark.parametrize("seqs", [40, 70])
def test_attention_of_many_rows_over_more_pages_than_are_kept(hip, seqs):
    """One part over 33000 positions in pages of 16, tiles of 64 and 128 rows."""
    b = Batch([33008 + s % 5 for s in range(seqs)], 1, (1, 1, 64), 16, 33008, seed=16)
    q = b.r.standard_normal((b.rows, 1, 64)).astype(np.float16)
    got = _attend(hip, b, q, slab_mb=2.2 * seqs * 66 * 4 / (1 << 20))
    pick = [0, 33, seqs - 1]
    b.lens = [n if s in pick else -1 for s, n in enumerate(b.lens)]
    want, tol = b.want(q, 1.0 / 8, 0)
    # fp32 sums of 33000 positions: 2^-24 a term, in the worst case all one way
    assert (np.abs(got - want)[pick] <= (tol + 33000 * 2.0 ** -24 * 4)[pick]).all()


def test_attention_leaves_rows_behind_the_last_slot(hip):
    b = Batch([100, 64, 90], 2, (8, 2, 128), 32, 64, seed=17)
    q = torch.from_numpy(b.r.standard_normal((20, 8, 128)).astype(np.float16)).cuda()
    out = torch.full((20, 8, 128), 5.0, dtype=torch.float16, device="cuda")
    hip.attn_paged(b.kv, 0, q, out, 2, 2, 8, 0.1, torch.empty(1 << 20, dtype=torch.uint8, device="cuda"), prefix_pages=2)
    torch.cuda.synchronize()
    assert (out[4:] == 5.0).all() and not (out[:4] == 5.0).all()


def test_lengths_and_entries_out_of_range_do_no_harm(hip):
    """Lengths behind the table, entries that name no page: nothing is written
    outside, and the other slots' results are what they are alone."""
    big = 2 ** 31 - 2
    b = Batch([70, 64, 90], 3, (8, 2, 64), 32, 64, seed=18)
    q = b.r.standard_normal((b.rows, 8, 64)).astype(np.float16)
    want = _attend(hip, b, q)
    b.kv.lens[1] = big
    b.kv.table[2, 2:] = torch.tensor([10 ** 6] * (b.table.shape[1] - 2), dtype=torch.int32, device="cuda")
    got = _attend(hip, b, q)
    assert np.array_equal(got[:3], want[:3])
    pool = b.kv.pool.clone()
    qkv = torch.zeros((9, 12 * 64), dtype=torch.float16, device="cuda")
    hip.rope_append_paged(b.kv, 0, qkv, torch.empty((9, 8, 64), dtype=torch.float16, device="cuda"), 3, 3, 8, 1e4)
    status = _i32([3])
    hip.kv_pages_reserve(b.kv, 3, 5, status)
    assert int(status.item()) > 0                       # behind the row
    b.kv.lens[0] = -1
    refs = b.kv.refs.clone()
    hip.kv_pages_fork(b.kv, _i32([1]), _i32([0]), 1, status)
    assert int(status.item()) == -1 and int(b.kv.lens[0].item()) == -1
    torch.cuda.synchronize()
    same = (b.kv.pool == pool).all(-1)                  # [planes, pages, heads, rows]
    mine = torch.zeros_like(same)
    for p in range(70, 73):
        mine[:, int(b.table[0, p // 32]), :, p % 32] = True
    assert (same | mine).all() and torch.equal(refs, b.kv.refs)


def test_attention_scores_far_apart(hip):
    """Scores over hundreds of powers of two, rising and falling along the
    positions: the running maximum is raised often, old sums vanish."""
    for order in (1, -1):
        b = Batch([700, 650], 1, (8, 2, 128), 64, 512, seed=14)
        q = b.r.standard_normal((b.rows, b.q_heads, b.D)).astype(np.float16)
        ramp = np.linspace(-30, 30, 12 * 64)[::order].reshape(12, 1, 64, 1)
        for s in range(2):
            n = (b.table[s] >= 0).sum()
            b.pool[0, b.table[s, :n]] = (ramp[:n] * np.sign(q[0, 0]) + b.pool[0, b.table[s, :n]] * 0.1).astype(np.float16)
        b.kv.pool.copy_(torch.from_numpy(b.pool))
        got = _attend(hip, b, q)
        want, tol = b.want(q, 1.0 / np.sqrt(b.D), 0)
        # a score of size z in fp32 is off by 2^-22 |z| (its products and their
        # sum), a probability by as much
        z = 30 * np.abs(q).astype(np.float64).sum(-1, keepdims=True) / np.sqrt(b.D)
        assert (np.abs(got - want) <= tol + 2.0 ** -21 * z * 5).all()


@pytest.mark.parametrize("prefix", [0, 128])
def test_attention_of_many_new_tokens(hip, prefix):
    """A prompt's own tokens in one call: tiles of 32 rows behind each other."""
    _check(hip, Batch([prefix, prefix + 3, -1], 150, (8, 2, 128), 32, prefix, seed=16))
    _check(hip, Batch([prefix + 17], 201, (14, 2, 64), 64, prefix, seed=17), window=90)


@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 8, 128)], ids=str)
def test_attention_of_a_ragged_batch(hip, heads):
    """Short and long slots side by side: every part of a slot has its share."""
    r = np.random.default_rng(18)
    lens = list((700 ** r.random(70)).astype(int)) + [-1, 1500, 0]
    _check(hip, Batch(lens, 1, heads, 16, 0, seed=19))


def test_attention_ignores_a_prefix_before_every_window(hip):
    lens, n_new, window = [300, 331, 280], 3, 50
    b = Batch(lens, n_new, (14, 2, 64), 64, 256, seed=20, poison=[n + 1 - window for n in lens])
    assert np.isnan(b.pool).any()
    _check(hip, b, window)


def test_attention_on_two_streams_at_once(hip):
    """Two calls that may run together, a slab each."""
    a, b = (Batch([512, 700, 513, 999], 2, (14, 2, 64), 64, 512, seed=s) for s in (21, 22))
    qs = [x.r.standard_normal((x.rows, x.q_heads, x.D)).astype(np.float16) for x in (a, b)]
    alone = [_attend(hip, x, q) for x, q in zip((a, b), qs)]
    dev = [torch.from_numpy(q).cuda() for q in qs]
    outs = [torch.zeros((x.rows, x.q_heads, x.D), dtype=torch.float16, device="cuda") for x in (a, b)]
    slabs = [torch.empty(8 << 20, dtype=torch.uint8, device="cuda") for _ in (a, b)]
    streams = [torch.cuda.Stream() for _ in (a, b)]
    torch.cuda.synchronize()
    try:
        for _ in range(10):
            for x, q, out, slab, st in zip((a, b), dev, outs, slabs, streams):
                hip.set_stream(st)
                hip.attn_paged(x.kv, 0, q, out, 4, 2, 14, 1.0 / np.sqrt(64), slab, prefix_pages=x.pp)
    finally:
        hip.use_torch_stream()
    torch.cuda.synchronize()
    # the slabs are smaller: fewer parts, another order of the same sums
    for x, q, out, want in zip((a, b), qs, outs, alone):
        same = _attend(hip, x, q, slab_mb=8)
        assert np.array_equal(out.cpu().numpy().astype(np.float64), same)
        assert np.abs(same - want).max() < 2.0 ** -9 * np.abs(x.pool[1]).max()


def test_attention_is_deterministic_and_replays(hip):
    b = Batch([520, 700, 513, -1, 999], 2, (14, 2, 64), 64, 512, seed=15)
    q = b.r.standard_normal((b.rows, b.q_heads, b.D)).astype(np.float16)
    first = _attend(hip, b, q)
    assert np.array_equal(first, _attend(hip, b, q))
    qd = torch.from_numpy(q).cuda()
    out = torch.zeros((b.rows, b.q_heads, b.D), dtype=torch.float16, device="cuda")
    slab = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    hip.set_stream(s)
    try:
        hip.capture_begin()
        try:
            hip.attn_paged(b.kv, 0, qd, out, 5, 2, 14, 1.0 / np.sqrt(64), slab, prefix_pages=b.pp)
        finally:
            g = hip.capture_end()
        for k in range(3):
            out.fill_(float("nan"))
            slab.fill_(255)
            torch.cuda.synchronize()
            g.launch()
            torch.cuda.synchronize()
            assert np.array_equal(first, out.cpu().numpy().astype(np.float64)), k
    finally:
        hip.use_torch_stream()


# ------------------------------------------------------------- RoPE + append

def _rope_want(b, qkv, theta):
    """Rotated q, pool after the append (float64) and the error bound of each."""
    D, Q, H, n = b.D, b.q_heads, b.kvh, b.n_new
    x = qkv.astype(np.float64).reshape(len(b.lens), n, -1, D)
    q = np.full((len(b.lens), n, Q, D), np.nan)
    qt = np.zeros_like(q)
    pool, pt = b.pool.astype(np.float64), np.zeros(b.pool.shape)
    freq = THETA ** (-np.arange(0, D, 2) / D) if theta else np.zeros(D // 2)
    for s, length in enumerate(b.lens):
        for j in range(n if length >= 0 else 0):
            z = x[s, j, :Q + H, :D // 2] + 1j * x[s, j, :Q + H, D // 2:]
            y = z * np.exp(1j * (length + j) * freq)
            y = np.concatenate([y.real, y.imag], -1)
            bound = 2.0 ** -20 * np.tile(np.abs(z.real) + np.abs(z.imag), 2) + EPS16 * np.abs(y) + 2.0 ** -25
            q[s, j], qt[s, j] = y[:Q], bound[:Q]
            e = (length + j) // b.page
            if e < b.table.shape[1] and b.table[s, e] >= 0:
                at = (b.table[s, e], slice(None), (length + j) % b.page)
                pool[(0,) + at], pt[(0,) + at] = y[Q:], bound[Q:]
                pool[(1,) + at] = x[s, j, Q + H:]
    return q.reshape(-1, Q, D), qt.reshape(-1, Q, D), pool, pt


@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("n_new,theta", [(1, THETA), (3, THETA), (20, THETA), (2, 0.0)])
def test_rope_append(hip, heads, n_new, theta):
    b = Batch([0, 15, 16, 131, -1, 500], n_new, heads, 16, seed=20)
    b.table[3, -1] = b.table[5, -1] = -1
    qkv = b.r.standard_normal((b.rows, (b.q_heads + 2 * b.kvh) * b.D)).astype(np.float16)
    q = torch.full((b.rows, b.q_heads, b.D), float("nan"), dtype=torch.float16, device="cuda")
    hip.rope_append_paged(b.kv, 0, torch.from_numpy(qkv).cuda(), q, 6, n_new, b.q_heads, theta)
    torch.cuda.synchronize()
    wq, tq, wp, tp = _rope_want(b, qkv, theta)
    gq, gp = q.cpu().numpy().astype(np.float64), b.kv.pool.cpu().numpy().astype(np.float64)
    free = np.isnan(wq)
    assert np.array_equal(np.isnan(gq), free)          # rows of a free slot are left as they were
    assert (np.abs(gq - wq)[~free] <= tq[~free]).all()
    assert (np.abs(gp - wp) <= tp).all()               # zero bound: every other row of the pool is untouched


def test_rope_append_far_positions_and_missing_pages(hip):
    """Position 130000 keeps its angle; positions without a page write no key."""
    b = Batch([40, 90], 2, (4, 2, 64), 16, seed=21)
    b.lens = [130001, 90]
    b.kv.lens.copy_(_i32(b.lens))
    b.table[1, 5] = -1
    b.kv.table.copy_(torch.from_numpy(b.table))
    qkv = b.r.standard_normal((b.rows, 8 * 64)).astype(np.float16)
    q = torch.empty((b.rows, 4, 64), dtype=torch.float16, device="cuda")
    hip.rope_append_paged(b.kv, 0, torch.from_numpy(qkv).cuda(), q, 2, 2, 4, THETA)
    torch.cuda.synchronize()
    wq, tq, wp, tp = _rope_want(b, qkv, THETA)
    assert (np.abs(q.cpu().numpy() - wq) <= tq).all()
    assert (np.abs(b.kv.pool.cpu().numpy() - wp) <= tp).all()


# ------------------------------------------------------------ page operations

class Pages:
    """The host's idea of the cache: lists and counts."""

    def __init__(self, kv):
        self.refs, self.table = kv.refs.cpu().numpy().copy(), kv.table.cpu().numpy().copy()
        self.lens, self.pool = kv.lens.cpu().numpy().copy(), kv.pool.cpu().numpy().copy()
        self.page = kv.page

    def lowest(self, n):
        free = np.flatnonzero(self.refs == 0)
        return None if len(free) < n else free[:n]

    def free(self, slots):
        for s in slots:
            if 0 <= s < len(self.lens):
                for e in self.table[s][self.table[s] >= 0]:
                    self.refs[e] -= 1
                self.table[s] = -1
                self.lens[s] = -1

    def fork(self, parents, children):
        ok = all(0 <= p < len(self.lens) and self.lens[p] >= 0 for p in parents)
        ok = ok and all(0 <= c < len(self.lens) and self.lens[c] == -1 for c in children)
        if not ok or len(set(children)) < len(children):
            return -1
        need = sum(self.lens[p] % self.page > 0 for p in parents)
        got = self.lowest(need)
        if got is None:
            return need - int((self.refs == 0).sum())
        got = list(got)
        for p, c in zip(parents, children):
            full, rest = divmod(int(self.lens[p]), self.page)
            self.table[c] = -1
            self.table[c, :full] = self.table[p, :full]
            self.refs[self.table[p, :full]] += 1
            if rest:
                e = got.pop(0)
                self.table[c, full], self.refs[e] = e, 1
                self.pool[:, e, :, :rest] = self.pool[:, self.table[p, full], :, :rest]
            self.lens[c] = self.lens[p]
        return 0

    def reserve(self, seqs, n_new):
        want, behind = [], 0
        for s in range(seqs):
            if self.lens[s] < 0:
                continue
            first, end = self.lens[s] // self.page, -(-(self.lens[s] + n_new) // self.page)
            behind += max(0, end - max(first, self.table.shape[1]))
            want += [(s, e) for e in range(first, min(end, self.table.shape[1])) if self.table[s, e] < 0]
        got = self.lowest(len(want))
        missing = (0 if got is not None else len(want) - int((self.refs == 0).sum())) + behind
        if missing:
            return missing
        for (s, e), p in zip(want, got):
            self.table[s, e], self.refs[p] = p, 1
        return 0

    def compact(self):
        live = int((self.refs != 0).sum())
        src = [p for p in range(live, len(self.refs)) if self.refs[p]]
        dst = [p for p in range(live) if not self.refs[p]]
        for a, b in zip(src, dst):
            self.pool[:, b] = self.pool[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.table[self.table == a] = b
        return live

    def same(self, kv):
        torch.cuda.synchronize()
        assert np.array_equal(kv.refs.cpu().numpy(), self.refs)
        assert np.array_equal(kv.table.cpu().numpy(), self.table)
        assert np.array_equal(kv.lens.cpu().numpy(), self.lens)
        assert np.array_equal(kv.pool.cpu().numpy().view(np.uint16), self.pool.view(np.uint16))


def _some_cache(n_pages, page=16, max_seqs=12, max_len=600, heads=2, dim=64, layers=2, seed=30):
    from cima_amd.paged import PagedKV

    kv = PagedKV.empty(layers, n_pages, heads, page, dim, max_seqs, max_len)
    kv.pool.copy_(torch.from_numpy(np.random.default_rng(seed).standard_normal(tuple(kv.pool.shape)).astype(np.float16)))
    return kv


@pytest.mark.parametrize("n_pages", [40, 1000, 1024, 5000])
@pytest.mark.parametrize("page", [16, 64])
def test_pages_random_history(hip, n_pages, page):
    """A few dozen operations in a row, each compared with the host's: enough
    and too little room, slots that are not as they must be, compaction in place."""
    kv = _some_cache(n_pages, page)
    host, r = Pages(kv), np.random.default_rng(n_pages + page)
    status, slab = _i32([77]), torch.empty(12 * n_pages + 64, dtype=torch.uint8, device="cuda")
    live = _i32([0])
    seen = set()
    for step in range(40):
        op = r.integers(0, 6)
        if op == 0:                                     # a request starts
            s, n = int(r.integers(0, 12)), int(r.integers(0, 400))
            if host.lens[s] < 0:
                host.lens[s] = 0
                kv.lens[s] = 0
            hip.kv_pages_reserve(kv, 12, n, status)
            got = host.reserve(12, n)
            assert int(status.item()) == got
            if got == 0:                                # its tokens are there now
                for i in range(12):
                    if host.lens[i] >= 0:
                        host.lens[i] += n
                kv.lens.copy_(torch.from_numpy(host.lens))
            seen.add(("reserve", got > 0))
        elif op in (1, 2):
            k = int(r.integers(1, 6))
            parents = r.integers(0, 12, k) if op == 1 else r.choice(np.append(np.flatnonzero(host.lens >= 0), 0), k)
            children = r.permutation(np.append(np.flatnonzero(host.lens < 0), 0))[:k] if op == 2 else r.integers(-1, 13, k)
            parents = parents[:len(children)]
            hip.kv_pages_fork(kv, _i32(parents), _i32(children), len(children), status)
            got = host.fork(parents.tolist(), children.tolist())
            assert int(status.item()) == got
            seen.add(("fork", got))
        elif op == 3:
            slots = r.integers(-1, 13, int(r.integers(1, 5)))
            hip.kv_pages_free(kv, _i32(slots), len(slots))
            host.free(slots.tolist())
        elif op == 4:
            hip.kv_pages_compact(kv, kv.refs, kv.table, live, slab)
            assert int(live.item()) != -5 and host.compact() == int(live.item())
        else:
            a = r.permutation(n_pages)[:6]
            free = [p for p in a[3:] if host.refs[p] == 0]
            src = a[:len(free)]
            hip.kv_pages_copy(kv, _i32(list(src) + [-1, n_pages, 0]), _i32(list(free) + [0, 0, -3]), len(free) + 3)
            host.pool[:, free] = host.pool[:, src]
        host.same(kv)
    assert ("fork", -1) in seen


def test_pages_fork_many_from_one_and_free_twice(hip):
    kv = _some_cache(300, max_seqs=80, max_len=700)
    host = Pages(kv)
    status = _i32([5])
    for at in (0, 1):
        kv.lens[at] = host.lens[at] = 0
    hip.kv_pages_reserve(kv, 2, 200, status)
    assert host.reserve(2, 200) == int(status.item()) == 0
    kv.lens[0] = host.lens[0] = 200                     # 12 pages and 8 rows
    kv.lens[1] = host.lens[1] = 192                     # 12 pages
    kids = list(range(2, 72))
    hip.kv_pages_fork(kv, _i32([i % 2 for i in kids]), _i32(kids), 70, status)
    assert host.fork([i % 2 for i in kids], kids) == int(status.item()) == 0
    host.same(kv)
    hip.kv_pages_free(kv, _i32([5, 5, 6, 5, 79]), 5)    # named three times, and one not in use
    host.free([5, 6, 79])
    host.same(kv)
    # the same child twice: refused, nothing claimed
    hip.kv_pages_fork(kv, _i32([0, 1]), _i32([5, 5]), 2, status)
    assert int(status.item()) == -1
    host.same(kv)
    # free slots give the pages back
    hip.kv_pages_free(kv, _i32(list(range(80))), 80)
    host.free(range(80))
    host.same(kv)
    assert not host.refs.any()


def test_pages_planes_apart_and_out_of_place_compaction(hip):
    """The pool as a view with room between its planes; the old counts and table stay."""
    from cima_amd.paged import PagedKV

    whole = torch.from_numpy(np.random.default_rng(3).standard_normal((4, 30, 2, 16, 64)).astype(np.float16)).cuda()
    kv = PagedKV(whole[:, :25], _i32([0, 1, 0, 0, 2] * 5), _i32(np.array([[1, 4, 6, 9, 24, -1], [4, 9, 11, 14, -1, -1]])),
                 _i32([70, 60]))
    host, keep = Pages(kv), whole.cpu().numpy().copy()
    refs, table, live = torch.empty_like(kv.refs), torch.empty_like(kv.table), _i32([0])
    hip.kv_pages_compact(kv, refs, table, live, torch.empty(1 << 16, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    before = Pages(kv)
    assert host.compact() == int(live.item()) == 10
    assert np.array_equal(refs.cpu().numpy(), host.refs) and np.array_equal(table.cpu().numpy(), host.table)
    assert before.refs.tolist() == [0, 1, 0, 0, 2] * 5 and before.table[0, 4] == 24
    got = whole.cpu().numpy()
    assert np.array_equal(got[:, :25], host.pool) and np.array_equal(got[:, 25:], keep[:, 25:])


# ---------------------------------------------------------------- together

def test_a_batch_of_continuations_step_by_step(hip):
    """One prompt, forked into four continuations that each take steps of one to
    three tokens, one freed and its pages used again, the pool compacted in
    between: every step's attention against the tokens' own history on the host."""
    heads, D, page, layers = (8, 2, 64), 64, 16, 2
    Q, H, _ = heads
    kv = _some_cache(64, page, max_seqs=6, max_len=400, heads=H, dim=D, layers=layers, seed=40)
    r = np.random.default_rng(41)
    status, live = _i32([1]), _i32([0])
    slab = torch.empty(8 << 20, dtype=torch.uint8, device="cuda")
    history = {}                                        # slot -> per layer (keys, values) float64
    freq = THETA ** (-np.arange(0, D, 2) / D)

    def rotate(x, pos):
        z = (x[..., :D // 2] + 1j * x[..., D // 2:]) * np.exp(1j * pos * freq)
        return np.concatenate([z.real, z.imag], -1)

    def step(seqs, n, prefix_pages, slot):
        hip.kv_pages_reserve(kv, seqs, n, status)
        assert int(status.item()) == 0
        lens = kv.lens.cpu().numpy()
        for layer in range(layers):
            qkv = r.standard_normal((seqs * n, (Q + 2 * H), D)).astype(np.float16)
            q = torch.zeros((seqs * n, Q, D), dtype=torch.float16, device="cuda")
            out = torch.empty_like(q)
            hip.rope_append_paged(kv, layer, torch.from_numpy(qkv).cuda(), q, seqs, n, Q, THETA)
            hip.attn_paged(kv, layer, q, out, seqs, n, Q, 1 / np.sqrt(D), slab, prefix_pages, slot)
            torch.cuda.synchronize()
            got = out.cpu().numpy().astype(np.float64)
            for s in range(seqs):
                for j in range(n):
                    if lens[s] < 0:
                        assert not got[s * n + j].any()
                        continue
                    x, pos = qkv[s * n + j].astype(np.float64), lens[s] + j
                    k, v = history[s][layer]
                    k.append(rotate(x[Q:Q + H], pos).astype(np.float16).astype(np.float64))
                    v.append(x[Q + H:])
                    K, V, qq = np.array(k), np.array(v), rotate(x[:Q], pos).astype(np.float16).astype(np.float64)
                    for h in range(Q):
                        z = K[:, h // (Q // H)] @ qq[h] / np.sqrt(D)
                        w = np.exp(z - z.max())
                        want = w @ V[:, h // (Q // H)] / w.sum()
                        # the bound of one attention, and once more the rounding of q and of
                        # the keys (half a step each, where sine and cosine differ in fp32)
                        tol = 4 * EPS16 * np.abs(V).max() + EPS16 * np.abs(want)
                        assert (np.abs(got[s * n + j, h] - want) <= tol).all()
        kv.lens.add_((kv.lens >= 0).int() * n)

    kv.lens[0] = 0
    history[0] = [([], []) for _ in range(layers)]
    step(1, 37, 0, 0)                                   # the prompt: two pages and five rows
    kids = [3, 1, 2]
    hip.kv_pages_fork(kv, _i32([0, 0, 0]), _i32(kids), 3, status)
    assert int(status.item()) == 0
    for c in kids:
        history[c] = [(list(k), list(v)) for k, v in history[0]]
    step(4, 1, 2, 0)
    step(4, 3, 2, 3)
    hip.kv_pages_free(kv, _i32([1]), 1)
    step(4, 2, 2, 0)
    hip.kv_pages_compact(kv, kv.refs, kv.table, live, slab)
    assert int(live.item()) == int((kv.refs > 0).sum())
    hip.kv_pages_fork(kv, _i32([2]), _i32([1]), 1, status)
    assert int(status.item()) == 0
    history[1] = [(list(k), list(v)) for k, v in history[2]]
    for n in (1, 2, 1):
        step(5, n, 2, 2)
    hip.kv_pages_free(kv, _i32([0, 1, 2, 3]), 4)
    torch.cuda.synchronize()
    assert not kv.refs.any() and (kv.table == -1).all() and (kv.lens == -1).all()


def test_a_captured_step_replays_as_the_batch_grows(hip):
    """Reserve, append, attention, softmax and verification of a step recorded
    once and replayed while lengths, pages and slots change; an eager twin on
    another cache gives the same bits after every step."""
    Q, H, D, page, layers, S, n, V = 14, 2, 64, 16, 2, 4, 3, 5000
    r = np.random.default_rng(70)
    twins = [_some_cache(96, page, max_seqs=S, max_len=900, heads=H, dim=D, layers=layers, seed=71) for _ in range(2)]
    f32, i32 = dict(device="cuda"), dict(device="cuda", dtype=torch.int32)
    qkv = torch.zeros((layers, S * n, (Q + 2 * H) * D), dtype=torch.float16, device="cuda")
    logits = torch.zeros((S * n, V), dtype=torch.float16, device="cuda")
    drafts, u = torch.zeros((S, n - 1), **i32), torch.zeros((S, n), **f32)
    temp = torch.tensor([0.7, 0.0, 1.2, 1.0], **f32)
    bufs = [dict(q=torch.zeros((S * n, Q, D), dtype=torch.float16, device="cuda"),
                 out=torch.zeros((layers, S * n, Q, D), dtype=torch.float16, device="cuda"),
                 p=torch.zeros((S * n, V), **f32), acc=torch.zeros(S, **i32), tok=torch.zeros((S, n), **i32),
                 status=torch.zeros(1, **i32), slab=torch.zeros(16 << 20, dtype=torch.uint8, device="cuda"))
            for _ in twins]

    def step(kv, b):
        hip.kv_pages_reserve(kv, S, n, b["status"])
        for layer in range(layers):
            hip.rope_append_paged(kv, layer, qkv[layer], b["q"], S, n, Q, THETA)
            hip.attn_paged(kv, layer, b["q"], b["out"][layer], S, n, Q, 0.125, b["slab"], prefix_pages=2, window=200)
        hip.softmax_rows(logits, b["p"], S * n, V, temp, n, 0.0, b["slab"])
        hip.verify_drafts(b["p"], None, drafts, None, u, b["acc"], b["tok"], kv.lens, S, n - 1, V, b["slab"])

    for kv, b in zip(twins, bufs):                      # a prompt of 37 tokens in slot 0, forked into 1 and 2
        kv.lens[0] = 0
        hip.kv_pages_reserve(kv, 1, 37, b["status"])
        for layer in range(layers):
            x = torch.from_numpy(np.random.default_rng(layer).standard_normal((37, (Q + 2 * H) * D)).astype(np.float16))
            hip.rope_append_paged(kv, layer, x.cuda(), torch.zeros((37, Q * D), dtype=torch.float16, device="cuda"), 1, 37,
                                  Q, THETA)
        kv.lens[0] = 37
        hip.kv_pages_fork(kv, _i32([0, 0]), _i32([1, 2]), 2, b["status"])
        torch.cuda.synchronize()
        assert b["status"].item() == 0
    st = torch.cuda.Stream()
    hip.set_stream(st)
    try:
        hip.capture_begin()
        try:
            step(twins[0], bufs[0])
        finally:
            g = hip.capture_end()
    finally:
        hip.use_torch_stream()
    for k in range(8):
        qkv.copy_(torch.from_numpy(r.standard_normal(qkv.shape).astype(np.float16)))
        logits.copy_(torch.from_numpy((r.standard_normal(logits.shape) * 3).astype(np.float16)))
        drafts.copy_(logits.view(S, n, V)[:, :n - 1].argmax(-1))
        u.copy_(torch.from_numpy(r.random((S, n)).astype(np.float32)))
        torch.cuda.synchronize()
        before = twins[1].lens.tolist()
        g.launch()
        torch.cuda.synchronize()
        step(twins[1], bufs[1])
        torch.cuda.synchronize()
        for key in ("out", "p", "acc", "tok", "status"):
            assert torch.equal(bufs[0][key], bufs[1][key]), (k, key)
        for key in ("lens", "table", "refs", "pool"):
            assert torch.equal(getattr(twins[0], key), getattr(twins[1], key)), (k, key)
        assert bufs[0]["status"].item() == 0
        assert twins[0].lens.tolist() == [m + a + 1 if m >= 0 else -1 for m, a in zip(before, bufs[0]["acc"].tolist())]
        for kv, b in zip(twins, bufs):                  # the batch changes between the steps
            if k == 2:
                hip.kv_pages_fork(kv, _i32([2]), _i32([3]), 1, b["status"])
            if k == 4:
                hip.kv_pages_free(kv, _i32([1]), 1)
            if k == 5:
                hip.kv_pages_compact(kv, kv.refs, kv.table, b["status"], b["slab"])
            if k == 6:
                hip.kv_pages_fork(kv, _i32([3]), _i32([1]), 1, b["status"])
        torch.cuda.synchronize()


# --------------------------------------------------------------- refusals

def test_pages_behind_4_gib(hip):
    """The same slots in the first pages and in the last ones of planes of 6 GB:
    every operator gives the same bits."""
    from cima_amd.paged import PagedKV

    heads, H, D, page, S = 8, 2, 128, 256, 3
    lens, stride = [700, 512, 3], 5
    r = np.random.default_rng(60)
    rows = r.standard_normal((2, 12, H, page, D)).astype(np.float16)
    qkv = torch.from_numpy(r.standard_normal((S, (heads + 2 * H) * D)).astype(np.float16)).cuda()
    results = []
    for n_pages, first in ((40, 0), (50000, 50000 - 40)):
        pool = torch.empty((2, n_pages, H, page, D), dtype=torch.float16, device="cuda")
        assert first == 0 or pool[0].numel() * 2 > 6 << 30
        pool[:, first:first + 12] = torch.from_numpy(rows).cuda()
        table = np.full((S + 1, stride), -1, np.int32)
        table[0, :4], table[1, :4], table[2, :1] = [0, 1, 5, 9], [0, 1, 11, 7], [3]
        table[table >= 0] += first
        refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        refs += 1                                       # free pages lie at the end alone
        refs[first + 20:first + 30] = 0
        kv = PagedKV(pool, refs, _i32(table), _i32(lens + [-1]))
        q, out = (torch.zeros((S, heads, D), dtype=torch.float16, device="cuda") for _ in range(2))
        slab = torch.empty(8 << 20, dtype=torch.uint8, device="cuda")
        status = _i32([9])
        hip.kv_pages_fork(kv, _i32([0]), _i32([3]), 1, status)   # the page begun: first + 20
        torch.cuda.synchronize()
        assert status.item() == 0 and kv.table[3].tolist() == [first, first + 1, first + 20, -1, -1]
        hip.rope_append_paged(kv, 0, qkv, q, S, 1, heads, 1e6)
        hip.attn_paged(kv, 0, q, out, S, 1, heads, 0.1, slab)
        shared = torch.zeros_like(out)
        hip.attn_paged(kv, 0, q[:2], shared[:2], 2, 1, heads, 0.1, slab, prefix_pages=2)
        hip.kv_pages_copy(kv, _i32([first + 11]), _i32([first + 33]), 1)
        torch.cuda.synchronize()
        results.append([t.cpu() for t in (q, out, shared, pool[:, first:first + 12], pool[:, first + 33],
                                          pool[:, first + 20, :, :700 - 512])])
        del pool, kv
        torch.cuda.empty_cache()
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    assert torch.isfinite(results[0][1]).all() and results[0][1].abs().max() > 0


def test_refusals(hip):
    b = Batch([64, 70], 1, (8, 2, 64), 32, 64, seed=50)
    q = torch.zeros((2, 8, 64), dtype=torch.float16, device="cuda")
    slab = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    one = _i32([0])

    def no(f, *a, **k):
        with pytest.raises(EngineError) as e:
            f(*a, **k)
        assert e.value.code == E_INVALID
    at = lambda **k: (b.kv, k.get("layer", 0), k.get("q", q), q, k.get("seqs", 2), 1, k.get("heads", 8),  # noqa: E731
                      k.get("scale", 0.1), k.get("slab", slab))
    hip.attn_paged(*at(), prefix_pages=2)
    for bad in ({"layer": 1}, {"layer": -1}, {"seqs": 3}, {"heads": 7}, {"heads": 16}, {"scale": 0.0},
                {"scale": float("inf")}, {"scale": 1e9}, {"q": q.float()}, {"q": q[:1]}, {"slab": 4096}):
        no(hip.attn_paged, *at(**bad), prefix_pages=2)
    no(hip.attn_paged, *at(), prefix_pages=99)
    no(hip.attn_paged, *at(), prefix_pages=2, prefix_slot=2)
    no(hip.attn_paged, *at(), prefix_pages=2, window=-1)
    no(hip.attn_paged, *at(slab=None), prefix_pages=2)
    no(hip.attn_paged, *at(slab=slab[:1000]), prefix_pages=2)
    no(hip.attn_paged, *at(slab=slab[8:]), prefix_pages=2)
    qkv = torch.zeros((2, 12 * 64), dtype=torch.float16, device="cuda")
    hip.rope_append_paged(b.kv, 0, qkv, q, 2, 1, 8, 1e4)
    no(hip.rope_append_paged, b.kv, 0, qkv, q, 2, 1, 8, -1.0)
    no(hip.rope_append_paged, b.kv, 0, qkv, q, 3, 1, 8, 1e4)
    no(hip.rope_append_paged, b.kv, 0, qkv.float(), q, 2, 1, 8, 1e4)
    no(hip.kv_pages_reserve, b.kv, 3, 1, one)
    no(hip.kv_pages_reserve, b.kv, 2, 1, one.long())
    no(hip.kv_pages_fork, b.kv, one, one, 2, one)
    no(hip.kv_pages_fork, b.kv, _i32([0] * 3), _i32([1] * 3), 3, one)
    no(hip.kv_pages_compact, b.kv, b.kv.refs, b.kv.table, one, slab[:64])
    no(hip.kv_pages_copy, b.kv, one, one.long(), 1)
    # nothing to do is no error
    hip.attn_paged(b.kv, 0, q, q, 0, 1, 8, 0.1, None)
    hip.kv_pages_free(b.kv, one, 0)
    hip.kv_pages_copy(b.kv, one, one, 0)
    torch.cuda.synchronize()
