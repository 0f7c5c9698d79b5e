"""The gated half of a feed-forward network as one operator.

`F.silu(self.fc1(x)) * self.fc3(x)` (megalodon/modules/normalized_feedforward_network.py:82) with both projections inside
(csrc/gated_linear.hip); the autograd node is C++ (csrc/host/ops.cpp)."""
from typing import Optional

import torch

from .. import _lib


def gated_linear(x: torch.Tensor, w1: torch.Tensor, w3: torch.Tensor, kept: Optional[torch.dtype] = None) -> torch.Tensor:
    """`F.silu(x @ w1.T) * (x @ w3.T)`: x (..., n_in), w1 and w3 (n_out, n_in) -> (..., n_out).

    bfloat16 or float16, one dtype for all three, any sizes; the products and the gate in float32, one rounding.  With gradients
    the two products are kept in `kept`: float32 (the default), or x's dtype for half the memory and one rounding more on the
    gradients' way.  The products' gradients are rounded to x's dtype before those of x and the weights are formed from them, so that these are off
    by 1.4 times what rounding them once takes (up to 64 tokens: rounded to two terms, and off by their own rounding alone).  In float16
    they have its range as well, as between separate layers: one beyond 65504 makes its token's and its feature's gradients infinite or NaN, and below 2 ** -14 they are off
    by 2 ** -25 each.  The gradients may be differentiated again; they are the same with `create_graph`.  The two matrices together hold fewer than
    2 ** 30 elements (n_in and n_out rounded up to 64)."""
    return _lib.host().gated_linear(x, w1, w3, kept)
