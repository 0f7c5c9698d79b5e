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
    gradients' way.  The products' gradients are rounded to x's dtype before those of x and the weights are formed from them (up to 64
    tokens: to two terms, so that the results are off by their own rounding alone).  The two matrices together hold fewer than
    2 ** 30 elements (n_in and n_out rounded up to 64)."""
    return _lib.host().gated_linear(x, w1, w3, kept)
