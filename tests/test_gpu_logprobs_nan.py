"""Log probabilities of rows with signalling NaN: as of rows with any other NaN, it hides no
token from the likeliest."""
import numpy as np
import pytest

from test_gpu_logprobs import _check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("rows,n", [(12, 700), (12, 5000), (12, 20011), (12, 50001), (150, 40000)])
def test_a_signalling_nan_hides_no_token(hip, dtype, cap, rows, n):
    """The largest logits before, behind and beside them, in the same and other words of a lane."""
    r = np.random.default_rng(n)
    x = (r.standard_normal((rows, n)) * 2).astype(dtype)
    bits = x.view(np.uint16 if dtype == np.float16 else np.uint32)
    nan = 0x7C01 if dtype == np.float16 else 0x7F800001
    sign = 0x8000 if dtype == np.float16 else 0x80000000
    for i in range(rows):
        for at in r.integers(0, n - 40, 6):
            x[i, at] = 10 + r.random()
            for gap in r.choice([1, 2, 3, 4, 6, 7, 8, 30], 3):
                bits[i, at + gap] = nan | (sign if r.random() < 0.5 else 0)
    temp = np.array([1.0, 0.0, 0.5, -1.0], np.float32)[np.arange(rows) % 4]
    tokens = np.where(np.isnan(x), -np.inf, x).argmax(1)
    for top in (0, 1, 8, 32):
        _check(hip, x, temp, cap, tokens, top)
