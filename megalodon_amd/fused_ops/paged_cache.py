"""A paged key / value cache: writing to it, reading it back, attention over it.

The contiguous cache of the attention layer (megalodon/modules/moving_average_gated_attention.py:92-101)
has one length for a whole batch.  Here sequences of any lengths share pools of pages:

* ``k_pages`` (pages, page_size, heads, k_width), ``v_pages`` (pages, page_size, heads, v_width); a page
  holds ``page_size`` consecutive positions of a sequence.  bfloat16 or float16; or float8_e4m3fn with
  ``k_exponents``, ``v_exponents`` (pages, page_size, heads) uint8: the row of a position and head is
  its codes times 2 ** (exponent - 127).  Any strides with a contiguous last axis, multiples of 16 elements;
* ``block_table`` (sequences, pages of one) int32: the pages of each sequence in their order.  Entries
  behind a sequence's last page are not looked at; a number that is no page has nothing behind it
  (writes to it are dropped, reads give zeros, attention does not see its keys);
* ``cu_new`` (sequences + 1) int32, from 0, not decreasing: rows cu_new[b] .. cu_new[b + 1] - 1 of a packed operand
  (rows, heads, width) belong to sequence b;
* ``lengths`` (sequences) int32: positions of each sequence, its new ones included, so that new row i of n is
  position lengths[b] - n + i.

page_size is a power of two from 16 on; widths are multiples of 16, up to 4096 (keys under attention: 512);
a row of block_table holds up to 2 ** 30 positions.
All metadata stays on the device: the calls do not synchronise and may be captured into a graph whose
replays follow new lengths and tables.  Pages may belong to several sequences as long as only one writes.
Inference only: a gradient that is asked for raises."""
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _lib


def paged_cache_write(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, lengths: Tensor, cu_new: Tensor,
                      k_exponents: Optional[Tensor] = None, v_exponents: Optional[Tensor] = None) -> None:
    """New rows k (rows, heads, k_width), v (rows, heads, v_width) to their positions, in place.

    8 bits: a row's exponent is the smallest that keeps its largest finite magnitude at or below 448 codes;
    codes are rounded to nearest, ties to even; infinities and NaN become NaN.  Two new rows of one call
    must not have one place.  Pools and exponents may be slices of one tensor, but not of the same memory."""
    _lib.host().paged_cache_write(k, v, k_pages, v_pages, block_table, lengths, cu_new, k_exponents, v_exponents)


def paged_cache_read(k_pages: Tensor, v_pages: Tensor, block_table: Tensor, begins: Tensor, cu_rows: Tensor, rows: int,
                     k_exponents: Optional[Tensor] = None, v_exponents: Optional[Tensor] = None,
                     dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Tensor]:
    """(k, v), `rows` contiguous rows each: row cu_rows[b] + i is position begins[b] + i of sequence b; zeros behind the
    last sequence.  `dtype` for an 8-bit cache: bfloat16 (the default) or float16."""
    return _lib.host().paged_cache_read(k_pages, v_pages, block_table, begins, cu_rows, rows, k_exponents, v_exponents, dtype)


def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, lengths: Tensor, cu_new: Tensor,
                    scale: float = 1.0, chunk_size: int = 0, k_exponents: Optional[Tensor] = None,
                    v_exponents: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """softmax(scale q k^T) v of new tokens q (rows, query heads, k_width) over their sequences' stored positions.

    The token at position p sees positions from the start of its chunk of `chunk_size` (0: from the first) to p; its own key
    and value have been written before.  The number of query heads is a multiple of the cache's: h reads head
    h // (query heads // heads).  A token that sees no key, or whose scores are all -inf, gets zeros.  What 8-bit rows stand
    for is rounded to q's dtype as paged_cache_read does (infinite past its largest number).  Returns
    (rows, query heads, v_width): rows behind the last sequence are zeros, or left as they are in a given `out`."""
    return _lib.host().paged_attention(q, k_pages, v_pages, block_table, lengths, cu_new, scale, chunk_size, k_exponents, v_exponents, out)
