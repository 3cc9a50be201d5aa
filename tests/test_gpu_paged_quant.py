"""The paged cache with 4- and 8-bit elements: append, read back, attention and page
operations, against plain implementations in 64 bits on the host.

Tolerances.  Codes and scales are whole numbers by definition: they are equal.  So
are values read back, each the f16 nearest to its code's.  The attention takes those
values, so that its error is what it is over an f16 cache (test_gpu_paged.py).
"""
import numpy as np
import pytest

from cima_amd.gguf import DType
from cima_amd.hip import E_FORMAT, E_INVALID, EngineError
from test_gpu_paged import THETA, Batch, _attend, _check, _i32, _rope_want

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [DType.Q4_1, DType.Q8_0]
HEADS = [(14, 2, 64), (32, 8, 128), (12, 12, 64), (16, 1, 128), (8, 8, 128)]


def quantise(x, t):
    """f16 rows [..., D] -> (codes uint8 [..., D], scales f16 [..., D / 32, 2 or 1]), in 64 bits.
    A least value of -0 is 0."""
    g = x.astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    low = g.min(-1, keepdims=True) + 0.0 if t == DType.Q4_1 else np.zeros((*g.shape[:-1], 1))
    steps = 15 if t == DType.Q4_1 else 127
    width = g.max(-1, keepdims=True) - low + 0.0 if t == DType.Q4_1 else np.abs(g).max(-1, keepdims=True)
    d = (width / steps).astype(np.float16)
    d = np.where(d.astype(np.float64) * steps < width, np.nextafter(d, np.float16(np.inf)), d)
    c = np.rint(np.divide(g - low, d.astype(np.float64), out=np.zeros_like(g), where=d > 0))
    codes = (c + (0 if t == DType.Q4_1 else 128)).astype(np.uint8).reshape(x.shape)
    return codes, np.concatenate([d, low.astype(np.float16)], -1) if t == DType.Q4_1 else d


def values(codes, scales, t):
    g = codes.astype(np.float64).reshape(*codes.shape[:-1], -1, 32)
    s = scales.astype(np.float64)
    x = g * s[..., :1] + s[..., 1:] if t == DType.Q4_1 else (g - 128) * s
    return x.astype(np.float16).reshape(codes.shape)


def pack(codes, scales, t):
    """Codes [..., page, D] and scales as heads' pages of bytes."""
    if t == DType.Q4_1:
        e = codes.reshape(*codes.shape[:-1], -1, 8).astype(np.uint32)
        w = sum(e[..., j] << (j // 2 * 4 + j % 2 * 16) for j in range(8))
        codes = w.astype("<u4").view(np.uint8)
    lead = codes.shape[:-2]
    return np.concatenate([codes.reshape(*lead, -1), np.ascontiguousarray(scales).view(np.uint8).reshape(*lead, -1)], -1)


def unpack(pool, t, page, D):
    """Bytes of heads' pages -> (codes [..., page, D], scales)."""
    lead, n = pool.shape[:-1], page * D // (2 if t == DType.Q4_1 else 1)
    codes = np.ascontiguousarray(pool[..., :n])
    if t == DType.Q4_1:
        w = codes.view("<u4").reshape(*lead, page, D // 8)
        codes = np.stack([w >> (j // 2 * 4 + j % 2 * 16) & 15 for j in range(8)], -1).astype(np.uint8)
    scales = np.ascontiguousarray(pool[..., n:]).view(np.float16).reshape(*lead, page, D // 32, -1)
    return codes.reshape(*lead, page, D), scales


class QBatch(Batch):
    """A Batch whose cache is quantised: ``pool`` holds the values that it stands for,
    rows that no one sees any codes and scales that are no number."""

    def __init__(self, t, *args, poison=None, **kw):
        from cima_amd.paged import PagedKV

        super().__init__(*args, poison=poison, **kw)
        self.t = t
        unseen = np.isnan(self.pool).any(-1)
        codes, scales = quantise(np.nan_to_num(self.pool), t)
        codes[unseen] = self.r.integers(0, 16, codes[unseen].shape)
        scales[unseen] = np.nan
        self.bytes = pack(codes, scales, t)
        self.pool = values(codes, scales, t)
        old = self.kv
        self.kv = PagedKV(torch.from_numpy(self.bytes).cuda(), old.refs, old.table, old.lens, ggml_type=t,
                          page=self.page, head_dim=self.D)

    def now(self):
        """The values that the cache stands for now."""
        return values(*unpack(self.kv.pool.cpu().numpy(), self.t, self.page, self.D), self.t)


# --------------------------------------------------------------- attention

@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attention_own_pages_only(hip, t, heads, page):
    _check(hip, QBatch(t, [0, 1, 15, 16, 63, 130, 517], 1, heads, page, seed=1))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("page,prefix", [(16, 16), (16, 48), (32, 320), (128, 1024), (256, 2048)])
def test_attention_shared_prefix(hip, t, heads, page, prefix):
    _check(hip, QBatch(t, [prefix, prefix + 1, prefix + 40, prefix + 200, prefix + page], 1, heads, page, prefix, seed=2))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", [(14, 2, 64), (16, 1, 128)], ids=str)
@pytest.mark.parametrize("page,prefix", [(16, 48), (32, 320)])
def test_attention_short_prefix_in_a_long_table(hip, t, heads, page, prefix):
    for seqs in (1, 5):
        lens = [prefix, prefix + 1, prefix + 40, prefix + 200, prefix + page][:seqs]
        _check(hip, QBatch(t, lens, 1, heads, page, prefix, seed=2, spare=2000 // page))
    _check(hip, QBatch(t, [prefix + 3, prefix + 90, -1], 4, heads, page, prefix, seed=23, spare=2000 // page), window=60)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("seqs", [1, 9, 20, 40, 80])
def test_attention_every_row_tile(hip, t, seqs):
    lens = [640 + (7 * s) % 90 for s in range(seqs)]
    for dim in (64, 128):
        _check(hip, QBatch(t, lens, 1, (16, 2, dim), 64, 640, seed=seqs, spare=20))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("n_new", [2, 5, 8, 33])
def test_attention_drafts(hip, t, n_new):
    _check(hip, QBatch(t, [96, 100, 111, 250], n_new, (14, 2, 64), 32, 96, seed=3))
    _check(hip, QBatch(t, [0, 5, 31], n_new, (8, 2, 128), 32, 0, seed=4))
    _check(hip, QBatch(t, [96, 100, 111, 250], n_new, (8, 2, 128), 32, 96, seed=5, spare=70))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("window", [1, 7, 64, 100, 300, 5000])
def test_attention_window(hip, t, window):
    lens = [256, 300, 333, 480, 700]
    for n_new in (1, 4):
        _check(hip, QBatch(t, lens, n_new, (14, 2, 64), 64, 256, seed=5), window)
        _check(hip, QBatch(t, lens, n_new, (8, 2, 128), 64, 256, seed=6, spare=20), window)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_free_slots_and_short_ones(hip, t):
    for lens in ([-1, 70, -1, 90], [64, -1, 64], [-1, -1]):
        _check(hip, QBatch(t, lens, 2, (8, 2, 128), 32, 64 if max(lens) > 0 else 0, seed=7))
    _check(hip, QBatch(t, [10, 64, 130, 0], 1, (14, 2, 64), 32, 64, seed=8))
    _check(hip, QBatch(t, [10, 64, 130, 0], 1, (14, 2, 64), 32, 64, seed=8, spare=70))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("window", [0, 50])
def test_attention_ignores_what_no_row_sees(hip, t, window):
    """Rows behind a slot's last token, unused pages and what lies before every row's
    window have scales that are no number; also behind a prefix, in tiles of rows."""
    lens, n_new = [200, 131, 160], 3
    low = [n + 1 - window if window else 0 for n in lens]
    for prefix in (0, 128):
        for spare in (1, 20):
            b = QBatch(t, lens, n_new, (8, 2, 128), 64, prefix, seed=9, poison=low, spare=spare)
            assert np.isnan(b.pool).any()
            _check(hip, b, window)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_between_windows_that_lie_apart(hip, t, dim):
    """Slots that end within the prefix: what is between their rows' windows may be anything."""
    lens, window = [30, 620, 300, 40], 20
    for heads in ((4, 2, dim), (32, 2, dim)):
        b = QBatch(t, lens, 1, heads, 32, 640, seed=10, poison=[n + 1 - window for n in lens], spare=60)
        assert np.isnan(b.pool).any()
        _check(hip, b, window)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_heads", [4, 40])
def test_attention_positions_without_a_page_are_not_seen(hip, t, dim, q_heads):
    """Entries that name no page, of the prefix and of slots: as if those positions were not there."""
    lens, page, prefix = [300, 290, 330], 32, 256
    b = QBatch(t, lens, 1, (q_heads, 2, dim), page, prefix, seed=11, spare=60)
    q = b.r.standard_normal((b.rows, q_heads, dim)).astype(np.float16)
    table = b.table.copy()
    table[:, 3] = -1                                       # of the prefix, in every slot
    table[1, 8], table[2, 9] = b.kv.n_pages, -7
    b.kv.table.copy_(_i32(table))
    got = _attend(hip, b, q)
    for s, n in enumerate(lens):
        ids = table[s, np.arange(n + 1) // page]
        ok = np.flatnonzero((ids >= 0) & (ids < b.kv.n_pages))
        for h in range(2):
            k, v = (b.pool[c, ids[ok], h, ok % page].astype(np.float64) for c in (0, 1))
            sl = slice(h * q_heads // 2, (h + 1) * q_heads // 2)
            z = q[s, sl].astype(np.float64) @ k.T / np.sqrt(dim)
            w = np.exp(z - z.max(1, keepdims=True))
            want = w / w.sum(1, keepdims=True) @ v
            tol = 2.0 ** -10 * np.abs(v).max(0) + 2.0 ** -11 * np.abs(want)
            assert (np.abs(got[s, sl] - want) <= tol).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("slab_mb", [0.07, 0.15, 0.5, 64])
def test_attention_with_small_and_large_slabs(hip, t, slab_mb):
    _check(hip, QBatch(t, [512, 700, 600, 555], 1, (14, 2, 64), 64, 512, seed=10, spare=20), slab_mb=slab_mb)
    _check(hip, QBatch(t, [512, 700, 600, 555], 1, (14, 2, 64), 64, 0, seed=10), slab_mb=slab_mb)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_without_a_slab(hip, t):
    _check(hip, QBatch(t, [512, 700, 60], 1, (14, 2, 64), 64, 0, seed=11), slab_mb=0)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_second_layer_and_many_pages(hip, t):
    """More pages than a task keeps ids of at a time (1024), unsplit; also in tiles of rows."""
    _check(hip, QBatch(t, [17000], 1, (2, 2, 64), 16, 0, layers=2, seed=12), slab_mb=0, layer=1)
    _check(hip, QBatch(t, [33000, 32768], 1, (2, 2, 64), 16, 32768, seed=13), slab_mb=0.01)
    _check(hip, QBatch(t, [17000], 1, (24, 1, 64), 16, 16992, seed=14), slab_mb=0.013)
    _check(hip, QBatch(t, [17000], 1, (70, 1, 128), 16, 16992, seed=15), slab_mb=0.08)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("prefix", [0, 128])
def test_attention_of_many_new_tokens(hip, t, prefix):
    _check(hip, QBatch(t, [prefix, prefix + 3, -1], 150, (8, 2, 128), 32, prefix, seed=16))
    _check(hip, QBatch(t, [prefix + 17], 201, (14, 2, 64), 64, prefix, seed=17), window=90)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", [(14, 2, 64), (8, 8, 128)], ids=str)
def test_attention_of_a_ragged_batch(hip, t, heads):
    r = np.random.default_rng(18)
    lens = list((700 ** r.random(70)).astype(int)) + [-1, 1500, 0]
    _check(hip, QBatch(t, lens, 1, heads, 16, 0, seed=19))


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_of_values_at_the_ends_of_f16(hip, t):
    """Groups of one value, of zeros, of f16's smallest numbers and of large ones."""
    b = QBatch(t, [90, 100], 1, (4, 2, 64), 32, 0, seed=24)
    pool = np.zeros_like(b.pool)
    r = np.random.default_rng(25)
    pool[0] = r.standard_normal(pool[0].shape)
    for i, (a, z) in enumerate([(0, 0), (3.5, 0), (0, 2.0 ** -24), (1, 2.0 ** -22), (0, 2.0 ** -14), (-56000, 3000),
                                (0, 20000)]):
        rows = (pool[1].reshape(-1, 64))[i::7]
        rows[:] = a + z * r.integers(-3, 4, rows.shape)
        pool[1].reshape(-1, 64)[i::7] = rows
    codes, scales = quantise(pool, t)
    b.pool = values(codes, scales, t)
    assert np.isfinite(b.pool).all()
    # half a step of the group and a rounding to f16
    step = np.repeat(scales[..., 0].astype(np.float64), 32, -1)
    assert (np.abs(b.pool - pool.astype(np.float64)) <= step / 2 + 2.0 ** -11 * np.abs(pool) + 2.0 ** -11 * step).all()
    b.kv.pool.copy_(torch.from_numpy(pack(codes, scales, t)))
    _check(hip, b)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_is_deterministic_and_replays(hip, t):
    b = QBatch(t, [520, 700, 513, -1, 999], 2, (14, 2, 64), 64, 512, seed=15)
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


# ---------------------------------------------------------- append, read back

def _append_want(b, qkv, theta):
    """Queries (float64, with their bound), and the pages' bytes after the append."""
    wq, tq, wp, tp = _rope_want(b, qkv, theta)
    codes, scales = unpack(b.bytes.copy(), b.t, b.page, b.D)
    x = qkv.reshape(len(b.lens), b.n_new, -1, b.D)
    freq = THETA ** (-np.arange(0, b.D, 2) / b.D) if theta else np.zeros(b.D // 2)
    for s, length in enumerate(b.lens):
        for j in range(b.n_new if length >= 0 else 0):
            e = (length + j) // b.page
            if e >= b.table.shape[1] or b.table[s, e] < 0:
                continue
            k = x[s, j, b.q_heads:b.q_heads + b.kvh].astype(np.float64)
            z = (k[:, :b.D // 2] + 1j * k[:, b.D // 2:]) * np.exp(1j * (length + j) * freq)
            rows = (np.concatenate([z.real, z.imag], -1).astype(np.float16), x[s, j, b.q_heads + b.kvh:])
            for plane, row in enumerate(rows):
                at = (plane, b.table[s, e], slice(None), (length + j) % b.page)
                codes[at], scales[at] = quantise(row, b.t)
    return wq, tq, pack(codes, scales, b.t)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("n_new,theta", [(1, THETA), (3, THETA), (20, THETA), (2, 0.0)])
def test_rope_append(hip, t, heads, n_new, theta):
    """Codes and scales as the definition gives them, every other byte as it was."""
    b = QBatch(t, [0, 15, 16, 131, -1, 500], n_new, heads, 16, seed=20)
    b.table[3, -1] = b.table[5, -1] = -1
    qkv = b.r.standard_normal((b.rows, (b.q_heads + 2 * b.kvh) * b.D)).astype(np.float16)
    q = torch.full((b.rows, b.q_heads, b.D), float("nan"), dtype=torch.float16, device="cuda")
    hip.rope_append_paged(b.kv, 0, torch.from_numpy(qkv).cuda(), q, 6, n_new, b.q_heads, theta)
    torch.cuda.synchronize()
    wq, tq, want = _append_want(b, qkv, theta)
    gq = q.cpu().numpy().astype(np.float64)
    free = np.isnan(wq)
    assert np.array_equal(np.isnan(gq), free)
    assert (np.abs(gq - wq)[~free] <= tq[~free]).all()
    assert np.array_equal(b.kv.pool.cpu().numpy(), want)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_append_of_every_kind_of_group(hip, t):
    """Ties between two codes, equal elements, zeros of both signs, f16's smallest and largest:
    as the definition says."""
    b = QBatch(t, [0, 3], 40, (2, 2, 128), 16, seed=21)
    r = b.r
    x = r.standard_normal((b.rows, 6, 128))
    x[0], x[1], x[2] = 0, -1.25, 65000
    x[3] = r.integers(-15, 16, x[3].shape)                # whole steps and halves of them
    x[4] = r.integers(0, 31, x[4].shape) / 2
    x[5] = r.integers(-254, 255, x[5].shape) / 2
    x[6] = r.integers(-5, 6, x[6].shape) * 2.0 ** -24
    x[7] = r.integers(-200, 201, x[7].shape) * 2.0 ** -24
    x[8] = np.where(r.random(x[8].shape) < 0.5, -65000, 65000)
    x[9] = np.where(r.random(x[9].shape) < 0.05, -30000, r.standard_normal(x[9].shape) * 2.0 ** -20)
    x[10] = -np.abs(x[10])
    x[11:20] *= 2.0 ** np.arange(-18, 9, 3)[:, None, None]
    x[20], x[21] = np.where(r.random(x[20].shape) < 0.5, 0.0, -0.0), -0.0
    x[22] = np.where(r.random(x[22].shape) < 0.5, -0.0, 3.5)
    qkv = x.reshape(b.rows, -1).astype(np.float16)
    q = torch.empty((b.rows, 2, 128), dtype=torch.float16, device="cuda")
    hip.rope_append_paged(b.kv, 0, torch.from_numpy(qkv).cuda(), q, 2, 40, 2, 0.0)
    torch.cuda.synchronize()
    want = _append_want(b, qkv, 0.0)[2]
    assert np.array_equal(b.kv.pool.cpu().numpy(), want)
    assert np.isfinite(b.now()).all()
    assert np.array_equal(q.cpu().numpy().reshape(b.rows, -1), qkv[:, :256])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_a_group_that_is_not_finite_reads_back_as_nan(hip, t):
    b = QBatch(t, [0], 3, (1, 1, 64), 16, seed=22)
    x = b.r.standard_normal((3, 3, 64)).astype(np.float16)
    x[0, 2, 5], x[1, 1, 40], x[2, 2, 63] = np.nan, np.inf, -np.inf
    hip.rope_append_paged(b.kv, 0, torch.from_numpy(x.reshape(3, -1)).cuda(),
                          torch.empty((3, 1, 64), dtype=torch.float16, device="cuda"), 1, 3, 1, 0.0)
    k, v = (torch.empty((1, 1, 3, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    hip.kv_pages_read(b.kv, 0, k, v, 1, 3)
    torch.cuda.synchronize()
    bad = torch.zeros((2, 3, 64), dtype=torch.bool)
    bad[1, 0, :32] = bad[0, 1] = bad[1, 2, 32:] = True    # a key's element 40 turns with element 8
    assert torch.equal(torch.stack([k[0, 0], v[0, 0]]).isnan().cpu(), bad)


@pytest.mark.parametrize("t", [0, *TYPES], ids=str)
@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128), (16, 1, 128)], ids=str)
@pytest.mark.parametrize("page", [16, 256])
def test_read_back(hip, t, heads, page):
    """Positions of slots in any order, one of them twice, in one that is free and in none."""
    lens = [0, 15, 16, 131, -1, 500]
    b = QBatch(t, lens, 1, heads, page, layers=2, seed=26) if t else Batch(lens, 1, heads, page, layers=2, seed=26)
    D, H = b.D, b.kvh
    table, n_pages = b.table.copy(), b.kv.n_pages
    table[3, 0] = n_pages + 5
    b.kv.table.copy_(_i32(table))
    for slots, first, n, room in (([5, 3, 5, 4, 1, 6, -1], None, 501, 501), ([5, 3], [100, -7], 97, 130),
                                  (None, [0, 1, 2, 3, 4, 2 ** 31 - 3], 1, 2), (None, None, 33, 33)):
        S = len(slots) if slots else len(first) if first else 6
        k, v = (torch.full((S, H, room, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
        hip.kv_pages_read(b.kv, 1, k, v, S, n, slots=_i32(slots) if slots else None, first=_i32(first) if first else None,
                          max_seq=room)
        torch.cuda.synchronize()
        want = np.zeros((2, S, H, room, D), np.float16)
        want[:, :, :, n:] = 7.0
        for i in range(S):
            s = slots[i] if slots else i
            for j in range(n):
                p = (first[i] if first else 0) + j
                if not (0 <= s < 6 and 0 <= p < table.shape[1] * page):
                    continue
                e = table[s, p // page]
                if 0 <= e < n_pages:
                    want[:, i, :, j] = b.pool[2:, e, :, p % page]
        assert np.array_equal(k.cpu().numpy(), want[0]) and np.array_equal(v.cpu().numpy(), want[1])


@pytest.mark.parametrize("t", [0, *TYPES], ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_read_back_of_many_rows(hip, t, dim):
    """As many rows as are read one a thread, one more of each head, and more: slots again and
    again, from positions before the first and behind the last."""
    lens, page, H = [700, 33, -1, 512], 64, 8
    b = QBatch(t, lens, 1, (8, H, dim), page, seed=38) if t else Batch(lens, 1, (8, H, dim), page, seed=38)
    most = 8 * torch.cuda.get_device_properties(0).multi_processor_count * 256 // (dim // 8)
    r = np.random.default_rng(39)
    for n in (most // (8 * H), most // (8 * H) + 1, 1300):
        slots, first = r.integers(-1, 5, 8), r.integers(-200, 300, 8)
        k, v = (torch.full((8, H, n + 3, dim), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
        hip.kv_pages_read(b.kv, 0, k, v, 8, n, slots=_i32(slots), first=_i32(first), max_seq=n + 3)
        torch.cuda.synchronize()
        want = np.zeros((2, 8, H, n + 3, dim), np.float16)
        want[:, :, :, n:] = 7.0
        for i, (s, f) in enumerate(zip(slots, first)):
            if not 0 <= s < 4:
                continue
            p = f + np.arange(n)
            ok = (p >= 0) & (p < b.table.shape[1] * page)
            e = np.where(ok, b.table[s, np.where(ok, p, 0) // page], -1)
            ok &= e >= 0
            want[:, i][:, :, np.flatnonzero(ok)] = b.pool[:, e[ok], :, p[ok] % page].transpose(1, 2, 0, 3)
        assert np.array_equal(k.cpu().numpy(), want[0]) and np.array_equal(v.cpu().numpy(), want[1])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_far_positions_and_pages_behind_4_gib(hip, t):
    """A pool of which a page lies behind 2^32 bytes: append, read back and attention find it."""
    from cima_amd.paged import PagedKV, head_page_bytes

    page, H, D = 256, 8, 128
    n_pages = (5 << 30) // (H * head_page_bytes(t, page, D))
    pool = torch.empty((2, n_pages, H, head_page_bytes(t, page, D)), dtype=torch.uint8, device="cuda")
    kv = PagedKV(pool, torch.zeros(n_pages, dtype=torch.int32, device="cuda"),
                 torch.full((1, 600), -1, dtype=torch.int32, device="cuda"), _i32([130000]), ggml_type=t, page=page,
                 head_dim=D)
    kv.table[0, 130000 // page] = n_pages - 1
    r = np.random.default_rng(27)
    qkv = r.standard_normal((3, 24, D)).astype(np.float16)
    q = torch.empty((3, 8, D), dtype=torch.float16, device="cuda")
    k, v = (torch.empty((1, H, 3, D), dtype=torch.float16, device="cuda") for _ in range(2))
    out = torch.empty_like(q)
    hip.rope_append_paged(kv, 0, torch.from_numpy(qkv.reshape(3, -1)).cuda(), q, 1, 3, 8, THETA)
    hip.kv_pages_read(kv, 0, k, v, 1, 3, first=kv.lens)
    hip.attn_paged(kv, 0, q, out, 1, 3, 8, 0.1, None, window=1)      # a row sees its own position alone
    torch.cuda.synchronize()
    z = (qkv[:, 8:16, :64] + 1j * qkv[:, 8:16, 64:].astype(np.float64)) * np.exp(
        1j * (130000 + np.arange(3))[:, None, None] * THETA ** (-np.arange(0, D, 2) / D))
    wk = values(*quantise(np.concatenate([z.real, z.imag], -1).astype(np.float16), t), t)
    wv = values(*quantise(qkv[:, 16:], t), t)
    assert np.array_equal(k[0].cpu().numpy(), wk.transpose(1, 0, 2))
    assert np.array_equal(v[0].cpu().numpy(), wv.transpose(1, 0, 2))
    got = out.cpu().numpy().astype(np.float64)
    assert (np.abs(got - wv) <= 2.0 ** -10 * np.abs(wv)).all()


# ------------------------------------------------------------ page operations

@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads,page", [((2, 2, 64), 16), ((8, 8, 128), 64)])
def test_page_operations_move_codes_and_scales(hip, t, heads, page):
    """Fork, copy and compact: the same slots read the same values as before, the
    children what their parents hold, and no other byte changes."""
    lens = [3 * page + 5, -1, 7, -1, 2 * page, -1]
    b = QBatch(t, lens, 1, heads, page, layers=3, seed=28, spare=2)
    slots = [0, 2, 4]

    def read(s, n):
        out = []
        for layer in range(3):
            k, v = (torch.empty((1, b.kvh, n, b.D), dtype=torch.float16, device="cuda") for _ in range(2))
            hip.kv_pages_read(b.kv, layer, k, v, 1, n, slots=_i32([s]))
            out += [k.cpu().numpy(), v.cpu().numpy()]
        return np.stack(out)
    before = {s: read(s, lens[s]) for s in slots}
    assert all(np.isfinite(x).all() for x in before.values())
    # a page begun is copied as far as it is filled
    held = set(np.flatnonzero(b.refs))
    was = b.kv.pool.cpu().numpy()
    status = _i32([9])
    free = [i for i in range(b.kv.n_pages) if i not in held]
    if len(free) < 2:
        pytest.fail("the cache has to have two free pages")
    hip.kv_pages_fork(b.kv, _i32([0, 2]), _i32([5, 1]), 2, status)
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    table, now = b.kv.table.cpu().numpy(), b.kv.pool.cpu().numpy()
    assert np.array_equal(read(5, lens[0]), before[0]) and np.array_equal(read(1, lens[2]), before[2])
    c0, s0 = unpack(was, t, page, b.D)
    c1, s1 = unpack(now, t, page, b.D)
    for parent, child in ((0, 5), (2, 1)):
        full, rest = divmod(lens[parent], page)
        src, dst = table[parent, full], table[child, full]
        assert dst in free and src != dst
        for a0, a1 in ((c0, c1), (s0.view(np.uint16), s1.view(np.uint16))):
            a0[:, dst, :, :rest] = a0[:, src, :, :rest]
    assert np.array_equal(c0, c1) and np.array_equal(s0.view(np.uint16), s1.view(np.uint16))
    # whole pages copied
    left = [i for i in free if i not in table]
    if left:
        hip.kv_pages_copy(b.kv, _i32([table[0, 0]]), _i32([left[0]]), 1)
        now[:, left[0]] = now[:, table[0, 0]]
        assert np.array_equal(b.kv.pool.cpu().numpy(), now)
    # slots freed, the others' pages moved together
    hip.kv_pages_free(b.kv, _i32([4, 5]), 2)
    live = _i32([0])
    hip.kv_pages_compact(b.kv, b.kv.refs, b.kv.table, live, torch.empty(1 << 16, dtype=torch.uint8, device="cuda"))
    n = int(live.item())
    assert (b.kv.refs[:n] > 0).all() and not b.kv.refs[n:].any() and int(b.kv.table.max()) < n
    for s, p in ((0, 0), (2, 2), (1, 2)):
        assert np.array_equal(read(s, lens[p]), before[p])


# ------------------------------------------------------------------ refusals

def test_refusals(hip):
    import ctypes

    from cima_amd.hip import KvPages

    b = QBatch(DType.Q4_1, [40], 1, (4, 2, 64), 16, seed=29)
    k = torch.zeros((1, 2, 40, 64), dtype=torch.float16, device="cuda")

    def no(code, f, *a, **kw):
        with pytest.raises(EngineError) as e:
            f(*a, **kw)
        assert e.value.code == code
    # a type that no cache has, planes of odd sizes
    for field, value, code in (("ggml_type", 12, E_FORMAT), ("ggml_type", 2, E_FORMAT), ("plane_elems", 8, E_INVALID),
                               ("plane_elems", b.kv.desc.plane_elems + 8, E_INVALID), ("head_dim", 96, E_INVALID),
                               ("pool", b.kv.desc.pool + 8, E_INVALID)):
        old = getattr(b.kv.desc, field)
        setattr(b.kv.desc, field, value)
        try:
            no(code, hip.kv_pages_read, b.kv, 0, k, k.clone(), 1, 40)
            no(code, hip.kv_pages_reserve, b.kv, 1, 1, _i32([0]))
        finally:
            setattr(b.kv.desc, field, old)
    assert ctypes.sizeof(KvPages) == 72
    v = k.clone()
    no(E_INVALID, hip.kv_pages_read, b.kv, 1, k, v, 1, 40)                    # a layer that is not there
    no(E_INVALID, hip.kv_pages_read, b.kv, 0, k, v, 1, 41)                    # more than k holds
    no(E_INVALID, hip.kv_pages_read, b.kv, 0, k, v, 1, 20, max_seq=10)
    no(E_INVALID, hip.kv_pages_read, b.kv, 0, k, v, -1, 20)
    no(E_INVALID, hip.kv_pages_read, b.kv, 0, k, v, 1, -1)
    no(E_INVALID, hip.kv_pages_read, b.kv, 0, k.float(), v, 1, 20)
    no(E_INVALID, hip.kv_pages_read, b.kv, 0, k, None, 1, 20)
    no(E_INVALID, hip.kv_pages_read, b.kv, 0, k.data_ptr() + 2, v, 1, 20)
    no(E_INVALID, hip.kv_pages_read, b.kv, 0, k, v, 1, 20, slots=torch.zeros(1, device="cuda", dtype=torch.int64))
    no(E_INVALID, hip.kv_pages_read, b.kv, 0, k, v, 1, 20, first=_i32([]))
    torch.cuda.synchronize()
    assert not k.any() and not v.any()
    hip.kv_pages_read(b.kv, 0, k, v, 0, 40)                                   # nothing to do
    hip.kv_pages_read(b.kv, 0, k, v, 1, 0)
    assert not k.any() and not v.any()
