"""softmax_rows at temperatures that leave one token, of rows with signalling NaN: NaN ranks as the
lowest, of either kind."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("rows,n", [(9, 700), (9, 5000), (9, 20011), (9, 50001), (300, 60001), (150, 70001)])
def test_a_signalling_nan_hides_no_logit(hip, dtype, cap, rows, n):
    r = np.random.default_rng(n)
    x = (r.standard_normal((rows, n)) * 2).astype(dtype)
    bits = x.view(np.uint16 if dtype == np.float16 else np.uint32)
    nan = 0x7C01 if dtype == np.float16 else 0x7F800001
    for i in range(rows):
        at = int(r.integers(0, n - 40))
        x[i, at] = 12
        bits[i, at + r.choice(np.arange(1, 33), 12, False)] = nan
    temp = np.array([0.0, -1.0, np.nan], np.float32)[np.arange(rows) % 3]
    y = torch.empty((rows, n), device="cuda")
    hip.softmax_rows(torch.from_numpy(x).cuda(), y, rows, n, torch.from_numpy(temp).cuda(), 1, cap,
                     torch.empty(8 << 20, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    want = np.zeros((rows, n), np.float32)
    want[np.arange(rows), np.where(np.isnan(x), -np.inf, x).argmax(1)] = 1
    assert np.array_equal(y.cpu().numpy(), want)
