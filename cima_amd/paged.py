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
"""
from __future__ import annotations

import ctypes

from .hip import E_INVALID, EngineError, KvPages


def _bad(msg: str):
    raise EngineError("hip", E_INVALID, f"paged cache: {msg}")


class PagedKV:
    """The tensors of a paged cache: ``pool`` f16 [2 * layers, n_pages, kv_heads,
    page, head_dim] (planes may lie apart), ``refs`` [n_pages], ``table``
    [max_seqs, entries] and ``lens`` [max_seqs] int32.  They are written in place:
    the descriptor holds their addresses, so none is exchanged for another."""

    def __init__(self, pool, refs, table, lens):
        import torch

        if pool.dim() != 5 or pool.dtype != torch.float16 or pool.shape[0] % 2:
            _bad("pool is not f16 [2 * layers, n_pages, kv_heads, page, head_dim]")
        planes, n_pages, heads, page, dim = pool.shape
        if pool.stride()[1:] != (heads * page * dim, page * dim, dim, 1):
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
        self.desc = KvPages(pool.data_ptr(), pool.stride(0), refs.data_ptr(), table.data_ptr(), lens.data_ptr(), planes,
                            n_pages, heads, page, dim, self.max_seqs, table.shape[1])
        self.ref = ctypes.byref(self.desc)

    def __setattr__(self, name, value):
        if name in ("pool", "refs", "table", "lens") and self.__dict__.get(name, value) is not value:
            _bad(f"{name} stays the tensor that the descriptor points to: write into it, or make another PagedKV")
        super().__setattr__(name, value)

    @classmethod
    def empty(cls, layers: int, n_pages: int, kv_heads: int, page: int, head_dim: int, max_seqs: int, max_len: int,
              device: str = "cuda") -> "PagedKV":
        """A cache without sequences: no page held, every slot free."""
        import torch

        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.empty((2 * layers, n_pages, kv_heads, page, head_dim), dtype=torch.float16, device=device),
                   torch.zeros(n_pages, **i32), torch.full((max_seqs, -(-max_len // page)), -1, **i32),
                   torch.full((max_seqs,), -1, **i32))
