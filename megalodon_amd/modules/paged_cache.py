"""`PagedCache`: the pools of a paged key / value cache of one attention layer, and the operators on them."""
from typing import Optional, Tuple

import torch
from torch import Tensor

from ..fused_ops import paged_attention, paged_cache_read, paged_cache_write


class PagedCache:
    """Keys and values of `pages` pages of `page_size` positions (fused_ops/paged_cache.py says how they lie).
    `quantized`: e4m3 codes with an exponent a row, half the bytes of `dtype`, which stays the type of
    the rows that go in and come out.  Which page belongs to whom is the caller's to say, call by call."""

    def __init__(self, pages: int, page_size: int, n_heads: int, z_head_dim: int, v_head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, quantized: bool = False, device=None):
        if dtype not in (torch.bfloat16, torch.float16):
            raise RuntimeError(f"PagedCache: dtype must be bfloat16 or float16 (got {dtype})")
        self.page_size, self.dtype, self.quantized = page_size, dtype, quantized
        stored = torch.float8_e4m3fn if quantized else dtype
        shape = (pages, page_size, n_heads)
        self.k_pages = torch.zeros(*shape, z_head_dim, dtype=stored, device=device)
        self.v_pages = torch.zeros(*shape, v_head_dim, dtype=stored, device=device)
        self.k_exponents = torch.full(shape, 127, dtype=torch.uint8, device=device) if quantized else None
        self.v_exponents = torch.full(shape, 127, dtype=torch.uint8, device=device) if quantized else None

    def write(self, k: Tensor, v: Tensor, block_table: Tensor, lengths: Tensor, cu_new: Tensor) -> None:
        paged_cache_write(k, v, self.k_pages, self.v_pages, block_table, lengths, cu_new, self.k_exponents, self.v_exponents)

    def read(self, block_table: Tensor, begins: Tensor, cu_rows: Tensor, rows: int) -> Tuple[Tensor, Tensor]:
        return paged_cache_read(self.k_pages, self.v_pages, block_table, begins, cu_rows, rows, self.k_exponents,
                                self.v_exponents, self.dtype)

    def attend(self, q: Tensor, block_table: Tensor, lengths: Tensor, cu_new: Tensor, scale: float = 1.0, chunk_size: int = 0,
               out: Optional[Tensor] = None) -> Tensor:
        return paged_attention(q, self.k_pages, self.v_pages, block_table, lengths, cu_new, scale, chunk_size,
                               self.k_exponents, self.v_exponents, out)

    def __repr__(self) -> str:
        pages, size, heads, width = self.k_pages.shape
        return (f"PagedCache(pages={pages}, page_size={size}, heads={heads}, z_head_dim={width}, "
                f"v_head_dim={self.v_pages.shape[3]}, dtype={self.dtype}, quantized={self.quantized})")
