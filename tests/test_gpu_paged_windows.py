"""Attention over a shared prefix by rows whose windows lie apart: what no row
sees may hold anything.  Tolerances as in test_gpu_paged_absent."""
import numpy as np
import pytest
from test_gpu_paged import Batch
from test_gpu_paged_absent import _check, _lose

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_new", [1, 3])
@pytest.mark.parametrize("lens", [[10, 540], [540, 3, 700, 200], [0, 90, 91, 250, 400, 550] * 2, [5 + 37 * s for s in range(30)]],
                         ids=len)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [50, 9])
def test_what_lies_between_the_rows_windows(hip, lens, n_new, dim, window):
    """Slots that end within the prefix beside longer ones: the windows of a
    task's rows lie apart, and what is between them holds NaN."""
    b = Batch(lens, n_new, (8, 2, dim), 16, 512, seed=33, poison=[n + 1 - window for n in lens], spare=60)
    assert np.isnan(b.pool).any()
    _check(hip, b, window)
    gaps = [e for e in range(32) if not any(e * 16 < n + n_new and e * 16 + 16 > n + 1 - window for n in lens)]
    _lose(b, [(s, e) for s in range(len(lens)) for e in gaps])       # given back, as a window's past may be
    _check(hip, b, window)
