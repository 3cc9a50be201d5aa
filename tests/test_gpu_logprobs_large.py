"""Log probabilities of rows behind 2^31 logits: the same as of those rows alone."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,few", [(131071, 9), (30001, 9)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_rows_behind_2_31_logits(hip, n, few, cap):
    rows, top = (1 << 31) // n + few, 7
    r = np.random.default_rng(n)
    some = torch.from_numpy((r.standard_normal((few, n)) * 4).astype(np.float16)).cuda()
    x = torch.zeros((rows, n), dtype=torch.float16, device="cuda")
    x[-few:] = some
    temp = torch.ones(rows, device="cuda")
    temp[-few:] = torch.tensor(r.uniform(0.3, 2, few), device="cuda")
    temp[-2] = 0
    slab = torch.empty(528 * rows * -(-n // 8192), dtype=torch.uint8, device="cuda")

    def run(x, temp):
        m = len(x)
        tokens = torch.arange(m, 0, -1, dtype=torch.int32, device="cuda") % n
        out = [torch.zeros(m, device="cuda"), torch.zeros(m, device="cuda"),
               torch.zeros((m, top), dtype=torch.int32, device="cuda"), torch.zeros((m, top), device="cuda")]
        hip.logprobs_rows(x, m, n, tokens, out[0], out[1], top, out[2], out[3], temp, 1, cap, slab)
        torch.cuda.synchronize()
        return out
    got, want = run(x, temp), run(some, temp[-few:].contiguous())
    assert torch.equal(got[2][-few:], want[2])
    # the sums of a few rows are split otherwise: 2^-24 for each of 40 additions on both sides, 2^-20 of their exponents
    for a, b in zip(got[:2] + got[3:], want[:2] + want[3:]):
        a, b = a[-few:].double(), b.double()
        odd = ~b.isfinite()
        assert torch.equal(a[odd], b[odd])
        assert ((a - b)[~odd].abs() <= 2.0 ** -17 * (1 + b[~odd].abs())).all()
    # rows of zeros: all are as likely
    assert (got[0][:-few] + np.log(n)).abs().max() < 1e-5 and (got[1][:-few] - np.log(n)).abs().max() < 1e-5
    assert (got[2][:-few] == torch.arange(top, dtype=torch.int32, device="cuda")).all()
