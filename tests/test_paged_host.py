"""The paged cache's and sampling's host side without a device: struct layout,
kernels in the code objects, refusals of a missing context, and what PagedKV
and the binding refuse."""
import ctypes
import os
import subprocess

import pytest

from cima_amd import build as cbuild
from cima_amd import hip as hipmod

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_kv_pages_layout_matches_header(tmp_path):
    fields = [f[0] for f in hipmod.KvPages._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cima_hip.h"\nint main(void){'
                   + "".join(f'printf("%zu ", offsetof(cima_kv_pages, {f}));' for f in fields)
                   + 'printf("%zu", sizeof(cima_kv_pages));return 0;}')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(hipmod.KvPages, f).offset for f in fields] + [ctypes.sizeof(hipmod.KvPages)]


def test_code_objects_hold_every_kernel():
    want = {"paged": ["cima_rope_append_paged_d64", "cima_rope_append_paged_d128", "cima_kv_pages_copy",
                      "cima_kv_pages_reserve", "cima_kv_pages_fork", "cima_kv_pages_free", "cima_kv_pages_compact"],
            "paged_attn": [f"cima_attn_paged_{k}" for d in (64, 128)
                           for k in (f"join_d{d}", *(f"d{d}_m{m}_n{n}" for m in (0, 1, 2) for n in (1, 2)))],
            "sample": ["cima_softmax", "cima_verify"]}
    for name, kernels in want.items():
        blob = open(cbuild.HSACOS[name], "rb").read()
        for k in kernels:
            assert k.encode() in blob, k


def test_every_entry_point_refuses_a_missing_context():
    L = hipmod.load_library()
    kv = ctypes.byref(hipmod.KvPages())
    for rc in (L.cima_hip_rope_append_paged(None, kv, 0, None, None, 1, 1, 1, 1e4),
               L.cima_hip_attn_paged(None, kv, 0, None, None, 1, 1, 1, 1.0, 0, 0, 0, None, 0),
               L.cima_hip_kv_pages_copy(None, kv, None, None, 1), L.cima_hip_kv_pages_reserve(None, kv, 1, 1, None),
               L.cima_hip_kv_pages_fork(None, kv, None, None, 1, None), L.cima_hip_kv_pages_free(None, kv, None, 1),
               L.cima_hip_kv_pages_compact(None, kv, None, None, None, None, 0),
               L.cima_hip_softmax_rows(None, None, None, 1, 1, None, 1, 0.0, 0, None, 0),
               L.cima_hip_verify_drafts(None, *[None] * 8, 1, 1, 1, None, 0)):
        assert rc == hipmod.E_NOT_INIT
        assert b"not initialised" in L.cima_hip_last_error()


def _tensors(planes=4, pages=6, heads=2, page=16, dim=64, slots=3, stride=5):
    i32 = torch.int32
    return [torch.zeros((planes, pages, heads, page, dim), dtype=torch.float16), torch.zeros(pages, dtype=i32),
            torch.full((slots, stride), -1, dtype=i32), torch.full((slots,), -1, dtype=i32)]


def test_paged_kv_refuses_wrong_tensors():
    from cima_amd.paged import PagedKV

    def no(t, text):
        with pytest.raises(hipmod.EngineError, match=text) as e:
            PagedKV(*t)
        assert e.value.code == hipmod.E_INVALID
    good = _tensors()
    no(good, "not on a HIP device")                     # all else is as it must be
    no([good[0].float()] + good[1:], "pool")
    no([good[0][0]] + good[1:], "pool")
    no([good[0][:3]] + good[1:], "pool")
    no([good[0].transpose(2, 3)] + good[1:], "contiguous")
    no([good[0], good[1].long(), *good[2:]], "refs")
    no([good[0], good[1][:5], *good[2:]], "refs")
    no([*good[:2], good[2][:, ::2], good[3]], "table")
    no([*good[:2], good[2][:2], good[3]], "table")
    no([*good[:3], good[3].float()], "lens")


def test_binding_checks_element_types_and_sizes(monkeypatch):
    monkeypatch.setattr(hipmod, "_ptr", lambda a: 4096)
    t = torch.zeros(6, dtype=torch.int32)
    assert hipmod._ptr_of(t, hipmod._I32, 6, "x", -1) in (4096, t.data_ptr())
    assert hipmod._ptr_of(None, hipmod._I32, 6, "x") is None and hipmod._ptr_of(64, hipmod._I32, 6, "x") == 64
    for a, n, device in ((t, 7, -1), (t.long(), 6, -1), (t.float(), 6, -1), (t, 6, 0), (t, 6, 1)):
        with pytest.raises(hipmod.EngineError):
            hipmod._ptr_of(a, hipmod._I32, n, "x", device)


def test_kernels_do_not_spill():
    """The attention's tiles, the copies and sampling keep their values in registers."""
    from test_abi import _kernel_notes

    for name in ("paged", "paged_attn", "sample"):
        notes = _kernel_notes(cbuild.HSACOS[name])
        assert notes and not {k: v for k, v in notes.items() if v[1] > 0}
