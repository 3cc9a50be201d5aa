"""Elements of a cache of 8 bits at the ends of f16: what is written finite reads back finite,
off by half a step."""
import numpy as np
import pytest

from cima_amd.gguf import DType
from test_gpu_paged_quant import QBatch, pack, quantise, unpack, values

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
def test_the_largest_elements_of_8_bits(hip, dim):
    """127 d is no f16 where d is 516, the least not below 65472 / 127: d is 515.5 there."""
    b = QBatch(DType.Q8_0, [0], 12, (2, 2, dim), 16, seed=31)
    r, groups = b.r, dim // 32
    x = (r.standard_normal((12, 6, dim)) * 30000).clip(-65000, 65000).astype(np.float16)
    most = np.array([65408, 65440, 65472, 65504, -65440, -65472, -65504], np.float16)
    for i, m in enumerate(most):
        for g in range(groups):
            x[i, :, 32 * g + (5 * i + g) % 32] = m
    x[7], x[8] = 65504, -65504
    x[9] = np.where(r.random(x[9].shape) < 0.5, -65504, 65504)
    x[10] = np.where(r.random(x[10].shape) < 0.1, 65472, r.standard_normal(x[10].shape))
    q = torch.empty((12, 2, dim), dtype=torch.float16, device="cuda")
    hip.rope_append_paged(b.kv, 0, torch.from_numpy(x.reshape(12, -1)).cuda(), q, 1, 12, 2, 0.0)
    k, v = (torch.empty((1, 2, 12, dim), dtype=torch.float16, device="cuda") for _ in range(2))
    hip.kv_pages_read(b.kv, 0, k, v, 1, 12)
    torch.cuda.synchronize()
    got = np.stack([k[0].cpu().numpy(), v[0].cpu().numpy()])             # [2, heads, rows, dim]
    want = x[:, 2:].reshape(12, 2, 2, dim).transpose(1, 2, 0, 3)
    assert np.isfinite(got).all()
    # the definition, with d of at most 515.5
    g = want.astype(np.float64).reshape(*want.shape[:-1], groups, 32)
    d = np.minimum(quantise(want, DType.Q8_0)[1].astype(np.float64), 515.5)
    c = np.rint(g / d)
    assert np.abs(c).max() == 127
    assert np.array_equal(got, (c * d).astype(np.float16).reshape(want.shape))
    # half a step, and half an f16's step (of 32 at most)
    assert (np.abs(got.astype(np.float64) - want) <= np.repeat(d[..., 0], 32, -1) / 2 + 16).all()
    # the bytes
    codes, scales = unpack(b.bytes.copy(), b.t, b.page, dim)
    ids = b.table[0, np.arange(12) // 16]
    for p in range(12):
        codes[:, ids[p], :, p] = (c[:, :, p].reshape(2, 2, dim) + 128).astype(np.uint8)
        scales[:, ids[p], :, p] = d[:, :, p].astype(np.float16)
    assert np.array_equal(b.kv.pool.cpu().numpy(), pack(codes, scales, b.t))
    assert np.array_equal(values(codes, scales, b.t)[:, ids[0], :, :12], got)
