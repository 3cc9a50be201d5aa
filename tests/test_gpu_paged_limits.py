"""The paged cache's counts and launches at their limits."""
import pytest
from test_gpu_paged import _i32

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_reserve_counts_more_missing_pages_than_an_int_holds(hip):
    """4096 slots that want 500000 entries each and 262144 behind their rows: the
    count stops at 2^31 - 1 and nothing is changed."""
    from cima_amd.paged import PagedKV

    slots, stride = 4096, 500000
    i32 = dict(dtype=torch.int32, device="cuda")
    kv = PagedKV(torch.zeros((2, 8, 1, 16, 64), dtype=torch.float16, device="cuda"), torch.zeros(8, **i32),
                 torch.full((slots, stride), -1, **i32), torch.zeros(slots, **i32))
    status = _i32([5])
    hip.kv_pages_reserve(kv, slots, 2 ** 30, status)
    torch.cuda.synchronize()
    assert status.item() == 2 ** 31 - 1
    assert not kv.refs.any() and int(kv.table.max().item()) == -1 and not kv.lens.any()
    hip.kv_pages_reserve(kv, 100, 16 * stride + 1, status)
    torch.cuda.synchronize()
    assert status.item() == 100 * stride - 8 + 100
    del kv
    torch.cuda.empty_cache()
