"""The quantised paged cache without a device: descriptor, sizes, kernels in the
code objects, and what PagedKV and a missing context refuse."""
import ctypes

import pytest

from cima_amd import build as cbuild
from cima_amd import hip as hipmod
from cima_amd.gguf import DType
from test_paged_fields import _OnDevice

torch = pytest.importorskip("torch")


def _tensors(t, planes=4, pages=6, heads=2, page=16, dim=64, slots=3, stride=5):
    from cima_amd.paged import head_page_bytes

    i32 = torch.int32
    return [torch.zeros((planes, pages, heads, head_page_bytes(t, page, dim)), dtype=torch.uint8),
            torch.zeros(pages, dtype=i32), torch.full((slots, stride), -1, dtype=i32), torch.full((slots,), -1, dtype=i32)]


@pytest.mark.parametrize("t,page,dim,size", [(DType.Q4_1, 16, 64, 640), (DType.Q4_1, 256, 128, 20480),
                                             (DType.Q8_0, 16, 64, 1088), (DType.Q8_0, 64, 128, 8704)])
def test_sizes_and_descriptor(t, page, dim, size):
    from cima_amd.paged import PagedKV, head_page_bytes

    assert head_page_bytes(t, page, dim) == size and size % 16 == 0
    kv = PagedKV(*(x.as_subclass(_OnDevice) for x in _tensors(t, page=page, dim=dim)), ggml_type=t, page=page,
                 head_dim=dim)
    d = kv.desc
    assert (d.ggml_type, d.page, d.head_dim, d.kv_heads, d.n_planes, d.n_pages) == (t, page, dim, 2, 4, 6)
    assert d.plane_elems == 6 * 2 * size and kv.layers == 2
    assert ctypes.sizeof(hipmod.KvPages) == 72        # as large as it was without the type


def test_paged_kv_refuses_wrong_tensors():
    from cima_amd.paged import PagedKV, head_page_bytes

    t = DType.Q4_1

    def no(ts, text, **kw):
        with pytest.raises(hipmod.EngineError, match=text) as e:
            PagedKV(*ts, **{"ggml_type": t, "page": 16, "head_dim": 64, **kw})
        assert e.value.code == hipmod.E_INVALID
    good = _tensors(t)
    no(good, "not on a HIP device")                   # all else is as it must be
    no([good[0].half()] + good[1:], "pool")
    no([good[0][:3]] + good[1:], "pool")
    no([good[0][..., :-1]] + good[1:], "pool")
    no([good[0][:, :, ::2]] + good[1:], "contiguous")
    no(good, "pool", ggml_type=DType.Q8_0)
    no(good, "pool", page=32)
    no(good, "pool", head_dim=128)
    no(good, "ggml type", ggml_type=DType.Q4_K)
    no(good, "a page", page=0)
    no(good, "a page", head_dim=48)
    no(_tensors(t)[:1] + [good[1].long()] + good[2:], "refs")
    with pytest.raises(hipmod.EngineError, match="ggml type"):
        head_page_bytes(0, 16, 64)
    # an f16 pool may name its sizes, if they are its own
    f16 = [torch.zeros((4, 6, 2, 16, 64), dtype=torch.float16), *good[1:]]
    no(f16, "not on a HIP device", ggml_type=0)
    no(f16, "pages of", ggml_type=0, page=32)
    no(f16, "pages of", ggml_type=0, head_dim=128)


def test_code_objects_hold_every_kernel():
    want = {"paged": [f"cima_rope_append_paged_q{b}_d{d}" for b in (4, 8) for d in (64, 128)]
            + [f"cima_kv_pages_read{f}_b{b}_d{d}" for f in ("", "_few") for b in (4, 8, 16) for d in (64, 128)]}
    for b in (4, 8):
        want[f"paged_attn_q{b}"] = [f"cima_attn_paged_q{b}_d{d}_m{m}_n{n}" for d in (64, 128) for m in (0, 2, 3, 4)
                                    for n in (1, 2)]
    for name, kernels in want.items():
        blob = open(cbuild.HSACOS[name], "rb").read()
        for k in kernels:
            assert k.encode() in blob, k


def test_quantised_kernels_do_not_spill():
    """Attention, append, read back and log probabilities keep every value in registers."""
    from test_abi import _kernel_notes

    notes = {}
    for name in ("paged", "paged_attn_q4", "paged_attn_q8", "sample"):
        notes.update(_kernel_notes(cbuild.HSACOS[name]))
    mine = {k: v for k, v in notes.items() if "paged_q" in k or "kv_pages_read" in k or "logprobs" in k}
    assert len(mine) == 2 * 16 + 4 + 12 + 28
    assert not {k: v for k, v in mine.items() if v[1] > 0}


def test_read_back_refuses_a_missing_context():
    L = hipmod.load_library()
    rc = L.cima_hip_kv_pages_read(None, ctypes.byref(hipmod.KvPages()), 0, None, None, None, None, 1, 1, 1)
    assert rc == hipmod.E_NOT_INIT and b"not initialised" in L.cima_hip_last_error()


def test_logprobs_kernels_and_a_missing_context():
    blob = open(cbuild.HSACOS["sample"], "rb").read()
    for t in ("f16", "f32", "cap_f16", "cap_f32"):
        for k in ("t256_w2", "t256_w8", "t1024_w8", "part_w2", "part_w8", "join_w2", "join_w8"):
            assert f"cima_logprobs_{k}_{t}".encode() in blob
    L = hipmod.load_library()
    rc = L.cima_hip_logprobs_rows(None, None, 1, 1, None, None, None, 0, None, None, None, 1, 0.0, 0, None, 0)
    assert rc == hipmod.E_NOT_INIT and b"not initialised" in L.cima_hip_last_error()
