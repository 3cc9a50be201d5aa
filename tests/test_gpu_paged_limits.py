"""The paged cache's counts and launches at their limits."""
import numpy as np
import pytest
from test_gpu_paged import EPS16, _i32, _some_cache

from cima_amd.hip import E_INVALID, EngineError

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


def test_attention_of_more_workgroups_than_a_launch_takes(hip):
    """4096 slots of 4096 heads, each a task of its own: 2^24 workgroups of 256
    threads pass the 2^32 of a launch and are refused; 4095 slots are served, the
    first, one within and the last of them in use."""
    kv = _some_cache(1, 16, max_seqs=4096, max_len=16, heads=4096, dim=64, layers=1)
    q = torch.empty((4096, 4096, 64), dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    with pytest.raises(EngineError) as e:
        hip.attn_paged(kv, 0, q, out, 4096, 1, 4096, 0.1, None)
    assert e.value.code == E_INVALID
    used = [0, 2222, 4094]
    r = np.random.default_rng(90)
    x = r.standard_normal((4096, 64)).astype(np.float16)
    for s in used:
        kv.lens[s], kv.table[s, 0] = 5, 0
        q[s] = torch.from_numpy(x).cuda()
    hip.attn_paged(kv, 0, q, out, 4095, 1, 4096, 0.1, None)
    torch.cuda.synchronize()
    got = out[used].cpu().numpy()
    k, v = kv.pool[:, 0, :, :6].cpu().numpy().astype(np.float64)
    z = np.einsum("hd,hpd->hp", x.astype(np.float64), k) * 0.1
    w = np.exp(z - z.max(1, keepdims=True))
    want = np.einsum("hp,hpd->hd", w / w.sum(1, keepdims=True), v)
    assert (np.abs(got - want) <= 2 * EPS16 * np.abs(v).max(1) + EPS16 * np.abs(want)).all()
    assert (out[4095] == 7.0).all()                     # behind the last slot
    out[used] = 0
    assert not out[:4095].any()
    del kv, q, out
    torch.cuda.empty_cache()
