"""Rows of a table by token (the reference's ParallelEmbedding at model-parallel world size 1,
megalodon/modules/model_parallel/layers.py), with a scale; the kernels are csrc/embedding.hip, the autograd node
csrc/host/embedding.cpp."""
from typing import Optional

import torch

from .. import _lib


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """`scale * weight[tokens]`: tokens of any shape, int64 or int32; weight (vocabulary, width) -> (*tokens.shape, width).

    float32, bfloat16 or float16; the product and the gradient's sums in float32, one rounding.  The gradient is dense, written whole,
    and the same from call to call.  `padding_idx` (negative: from the end) names a row whose tokens have no gradient.  A token that is
    no row of the table gives zeros and has no gradient: nothing on the device can raise for it."""
    return _lib.host().embedding(tokens, weight, scale, padding_idx)
