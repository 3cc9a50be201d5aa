"""Attention over a quantised cache where the prefix is taken in tiles of 128 rows (more
than 64 rows of a kv head of 128, or 256 of one of 64): what no row sees, windows that lie apart
and entries that name no page.  Tolerances as in test_gpu_paged.
"""
import numpy as np
import pytest

from cima_amd.gguf import DType
from test_gpu_paged import _attend, _check, _i32
from test_gpu_paged_quant import QBatch

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = [DType.Q4_1, DType.Q8_0]
# heads whose four slots are a tile and a part of one, and more
HEADS = [(80, 2, 128), (33, 1, 128), (200, 2, 64), (70, 1, 64)]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("window", [0, 50])
def test_attention_ignores_what_no_row_sees(hip, t, heads, window):
    """Scales that are no number behind the slots' last tokens and before every row's window,
    inside the prefix too."""
    for lens, prefix, n_new in (([200, 131, 160, 150], 128, 1), ([700, 650, 641, 660], 640, 2)):
        low = [n + 1 - window if window else 0 for n in lens]
        for spare in (20, 90):
            b = QBatch(t, lens, n_new, heads, 32, prefix, seed=9, poison=low, spare=spare)
            assert np.isnan(b.pool).any()
            _check(hip, b, window)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_attention_between_windows_that_lie_apart(hip, t, heads):
    """Slots that end within the prefix: what is between their rows' windows may be anything."""
    window = 20
    for lens, slab in (([30, 620, 300, 40], 32), ([50, 610, -1, 330], 32), ([30, 620, 300, 40], 1.7)):
        b = QBatch(t, lens, 1, heads, 32, 640, seed=10, poison=[max(n + 1 - window, 0) for n in lens], spare=60)
        assert np.isnan(b.pool).any()
        _check(hip, b, window, slab_mb=slab)


def _without(hip, b, table, lens, window=0, slab_mb=32):
    """The attention where `table` names no page at some entries: as if those positions were not."""
    q = b.r.standard_normal((b.rows, b.q_heads, b.D)).astype(np.float16)
    b.kv.table.copy_(_i32(table))
    got = _attend(hip, b, q, window, slab_mb)
    g = b.q_heads // b.kvh
    for s, n in enumerate(lens):
        for j in range(b.n_new):
            p = np.arange(max(0, n + j + 1 - window) if window else 0, n + j + 1)
            ids = table[s, p // b.page]
            ok = (ids >= 0) & (ids < b.kv.n_pages)
            row = s * b.n_new + j
            if not ok.any():
                assert not got[row].any()
                continue
            for h in range(b.kvh):
                k, v = (b.pool[c, ids[ok], h, p[ok] % b.page].astype(np.float64) for c in (0, 1))
                sl = slice(h * g, (h + 1) * g)
                z = q[row, sl].astype(np.float64) @ k.T / np.sqrt(b.D)
                w = np.exp(z - z.max(1, keepdims=True))
                want = w / w.sum(1, keepdims=True) @ v
                tol = 2.0 ** -10 * np.abs(v).max(0) + 2.0 ** -11 * np.abs(want)
                assert (np.abs(got[row, sl] - want) <= tol).all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("page", [16, 64])
def test_attention_positions_without_a_page_are_not_seen(hip, t, heads, page):
    """Entries of the prefix and of slots that name no page; page 0, which is read in their
    place, holds scales that are no number."""
    lens, prefix = [700, 660, 690, 642], 640
    b = QBatch(t, lens, 1, heads, page, prefix, seed=11, spare=2000 // page)
    table = b.table.copy()
    zero = np.argwhere(table == 0)                         # wherever page 0 is: gone with the others
    table[table == 0] = -1
    table[:, 3] = table[:, 5] = -1                         # of the prefix, in every slot
    table[1, 640 // page], table[2, 1 + 640 // page] = b.kv.n_pages, -7
    b.kv.pool[:, 0].fill_(255)
    b.pool[:, 0] = np.nan
    assert len(zero) <= 4
    _without(hip, b, table, lens)
    table[:, :prefix // page] = -1                         # a prefix of which nothing is left
    _without(hip, b, table, lens)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", [(70, 1, 128), (264, 1, 64)], ids=str)
def test_attention_without_a_page_behind_the_ids_kept(hip, t, heads):
    """Of 1062 pages of the prefix, in one part, more than a task keeps ids of at a time: entries that
    name no page among the first, about the change and behind it, or behind it alone."""
    n, page = 17000, 16
    b = QBatch(t, [n], 1, heads, page, 16992, seed=15)
    rows, dim = heads[0], heads[2]
    slab = 2 * rows * (dim + 2) * 4 / (1 << 20) + 0.001    # two parts: the prefix's and the slot's
    for gone in ([1040, 1061], [2, 5, 500, 1018, 1019, 1020, 1023, 1024, 1025, 1050]):
        table = b.table.copy()
        table[:, gone[::2]], table[:, gone[1::2]] = -1, b.kv.n_pages
        _without(hip, b, table, [n], slab_mb=slab)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("window", [1, 64, 300])
def test_attention_windows_over_several_tiles(hip, t, heads, window):
    """Two tokens a slot, windows that end within the prefix, slots that are free."""
    _check(hip, QBatch(t, [700, 641, -1, 655, 640], 2, heads, 64, 640, seed=5, spare=20), window)
