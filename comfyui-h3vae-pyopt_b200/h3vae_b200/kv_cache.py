"""Paged INT8 key/value cache of one attention layer.

Tokens lie in pages of `page_size`; a page table int32 [batch, pages] says which pages hold a sequence, so
sequences of different lengths share one pool.  Keys and values are INT8 codes with one fp32 scale per
(page, head); k_sum holds, for each complete page, the sum of its K codes (what page selection scores).
The operations are h3vae_b200.kernels: kv_write_i8, kv_read_i8, attention_kv_i8, kv_select_i8.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)


class KVCacheI8:
    """The pool's tensors: k, v int8 [pages, heads, page_size, head_dim]; k_scale, v_scale fp32 [pages, heads];
    k_sum int16 [pages, heads, head_dim].  All contiguous on one CUDA device; they are updated in place and not
    replaced for the life of the object."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "k_sum", "num_pages", "kv_heads", "page_size", "head_dim", "device",
                 "struct", "_struct")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 k_sum: torch.Tensor):
        if k.ndim != 4 or v.shape != k.shape:
            raise ValueError("k and v must both be int8 [pages, heads, page_size, head_dim]")
        pages, heads, page, dim = k.shape
        if page not in PAGE_SIZES or dim not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}, got {page}, {dim}")
        for name, t, dtype, shape in (("k", k, torch.int8, k.shape), ("v", v, torch.int8, k.shape),
                                      ("k_scale", k_scale, torch.float32, (pages, heads)),
                                      ("v_scale", v_scale, torch.float32, (pages, heads)),
                                      ("k_sum", k_sum, torch.int16, (pages, heads, dim))):
            if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dtype} {list(shape)}")
            if t.device != k.device or t.device.type != "cuda":
                raise ValueError("the cache's tensors must be on one CUDA device")
        self.k, self.v, self.k_scale, self.v_scale, self.k_sum = k, v, k_scale, v_scale, k_sum
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page, dim
        self.device = k.device
        self._struct = _lib.KvCacheStruct(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                          k_sum.data_ptr(), pages, heads, page, dim)
        self.struct = ctypes.addressof(self._struct)     # what the library takes

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, head_dim: int = 64, page_size: int = 64,
              device="cuda") -> "KVCacheI8":
        """A pool of zeroed pages."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        z = lambda s, t: torch.zeros(s, dtype=t, device=device)  # noqa: E731
        return cls(z(shape, torch.int8), z(shape, torch.int8), z(shape[:2], torch.float32), z(shape[:2], torch.float32),
                   z((num_pages, kv_heads, head_dim), torch.int16))
