"""A paged KV cache for a batch of sequences, over the C ABI's ``cima_kv_pages``.

The reference serves one sequence from contiguous caches
(``src/models/transformer.rs:1100-1160``); several continuations of one prompt,
or drafted tokens, share its pages here.  ``PagedKV`` holds the tensors and the
descriptor that ``HipCtx``'s paged methods take:

    kv = PagedKV.empty(layers, n_pages, kv_heads, page, head_dim, max_seqs, max_len)
    kv.lens[0] = 0                                   # slot 0 starts a sequence
    hip.kv_pages_reserve(kv, 1, prompt_len, status)  # pages for the prompt
    ... per layer: hip.rope_append_paged, hip.attn_paged; then kv.lens[0] = prompt_len
    hip.kv_pages_fork(kv, parents, children, n, status)   # more continuations of it
    hip.kv_pages_free(kv, slots, n)

A cache of 4- or 8-bit elements (``ggml_type=DType.Q4_1`` or ``Q8_0``) takes the same
calls; ``hip.kv_pages_read`` gives its rows, or an f16 cache's, as f16.
"""
from __future__ import annotations

import ctypes

from .gguf import DType, storage_bytes
from .hip import E_INVALID, EngineError, KvPages


def _bad(msg: str):
    raise EngineError("hip", E_INVALID, f"paged cache: {msg}")


def head_page_bytes(ggml_type: int, page: int, head_dim: int) -> int:
    """Bytes of one head's page of a quantised cache: its codes, then its scales."""
    if ggml_type not in (DType.Q4_1, DType.Q8_0):
        _bad(f"ggml type {ggml_type} is not Q4_1 or Q8_0")
    if page <= 0 or head_dim <= 0 or head_dim % 32:
        _bad(f"a page of {page} rows of {head_dim} elements")
    return page * storage_bytes(ggml_type, head_dim)


class PagedKV:
    """The tensors of a paged cache: ``pool`` f16 [2 * layers, n_pages, kv_heads,
    page, head_dim] (planes may lie apart), ``refs`` [n_pages], ``table``
    [max_seqs, entries] and ``lens`` [max_seqs] int32.  They are written in place:
    the descriptor holds their addresses, so none is exchanged for another.

    With ``ggml_type`` Q4_1 or Q8_0 the pool is uint8 [2 * layers, n_pages,
    kv_heads, head_page_bytes(...)], and ``page`` and ``head_dim`` have to be named."""

    def __init__(self, pool, refs, table, lens, ggml_type: int = 0, page: int = 0, head_dim: int = 0):
        import torch

        if ggml_type:
            size = head_page_bytes(ggml_type, page, head_dim)
            if pool.dim() != 4 or pool.dtype != torch.uint8 or pool.shape[0] % 2 or pool.shape[3] != size:
                _bad(f"pool is not uint8 [2 * layers, n_pages, kv_heads, {size}]")
            planes, n_pages, heads = pool.shape[:3]
            dim, inner = head_dim, (heads * size, size, 1)
        else:
            if pool.dim() != 5 or pool.dtype != torch.float16 or pool.shape[0] % 2:
                _bad("pool is not f16 [2 * layers, n_pages, kv_heads, page, head_dim]")
            if (page or pool.shape[3], head_dim or pool.shape[4]) != tuple(pool.shape[3:]):
                _bad(f"pool has pages of {tuple(pool.shape[3:])}, not {(page, head_dim)}")
            planes, n_pages, heads, page, dim = pool.shape
            inner = (heads * page * dim, page * dim, dim, 1)
        if pool.stride()[1:] != inner:
            _bad("a plane of the pool is not contiguous")
        for name, t, shape in (("refs", refs, (n_pages,)), ("table", table, (lens.shape[0], table.shape[-1])),
                               ("lens", lens, lens.shape[:1])):
            if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
                _bad(f"{name} is not a contiguous int32 tensor of shape {tuple(shape)}")
            if t.device != pool.device:
                _bad(f"{name} is on {t.device}, the pool on {pool.device}")
        if not pool.is_cuda:
            _bad("the pool is not on a HIP device")
        self.pool, self.refs, self.table, self.lens = pool, refs, table, lens
        self.layers, self.n_pages, self.kv_heads, self.page, self.head_dim = planes // 2, n_pages, heads, page, dim
        self.max_seqs, self.device = lens.shape[0], pool.get_device()
        self.ggml_type = int(ggml_type)
        self.desc = KvPages(pool.data_ptr(), pool.stride(0), refs.data_ptr(), table.data_ptr(), lens.data_ptr(), planes,
                            n_pages, heads, page, dim, self.max_seqs, table.shape[1], self.ggml_type)
        self.ref = ctypes.byref(self.desc)

    def __setattr__(self, name, value):
        if name in ("pool", "refs", "table", "lens") and self.__dict__.get(name, value) is not value:
            _bad(f"{name} stays the tensor that the descriptor points to: write into it, or make another PagedKV")
        super().__setattr__(name, value)

    @classmethod
    def empty(cls, layers: int, n_pages: int, kv_heads: int, page: int, head_dim: int, max_seqs: int, max_len: int,
              device: str = "cuda", ggml_type: int = 0) -> "PagedKV":
        """A cache without sequences: no page held, every slot free."""
        import torch

        i32 = dict(dtype=torch.int32, device=device)
        if ggml_type:
            pool = torch.empty((2 * layers, n_pages, kv_heads, head_page_bytes(ggml_type, page, head_dim)),
                               dtype=torch.uint8, device=device)
        else:
            pool = torch.empty((2 * layers, n_pages, kv_heads, page, head_dim), dtype=torch.float16, device=device)
        return cls(pool, torch.zeros(n_pages, **i32), torch.full((max_seqs, -(-max_len // page)), -1, **i32),
                   torch.full((max_seqs,), -1, **i32), ggml_type, page, head_dim)
