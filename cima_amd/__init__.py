"""cima_amd -- MI355X (gfx950) GGUF dequant-GEMV hot path of the cima engine.

Native parts (built by ``cima_amd.build`` into ``cima_amd/lib``):
  * ``cima_gemv_{a,b,c}.hsaco``, ``cima_gemm.hsaco``, ``cima_gemm_wide.hsaco``,
    ``cima_dequant.hsaco``, ``cima_decode.hsaco``, ``cima_bnb4.hsaco``,
    ``cima_paged.hsaco``, ``cima_paged_attn{,_q4,_q8}.hsaco``,
    ``cima_sample.hsaco`` -- hand-written HIP kernels for gfx950
  * ``libcima_hip.so``  -- the C ABI of ``include/cima_hip.h``
  * ``libcima_synth.so`` -- seeded synthetic weights (``include/cima_synth.h``)

``cima_amd.hip.HipCtx`` is the Python mirror of the reference's ``CudaCtx``
GGUF methods; ``cima_amd.paged.PagedKV`` is the cache of its batch methods.
"""
from . import gguf  # noqa: F401
from .gguf import DType, block_elems, storage_bytes  # noqa: F401

__all__ = ["gguf", "DType", "block_elems", "storage_bytes"]
