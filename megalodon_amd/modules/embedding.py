"""`Embedding`: the reference's ParallelEmbedding (megalodon/modules/model_parallel/layers.py) at model-parallel world size 1."""
from typing import Optional

import torch
from torch import nn

from ..fused_ops import embedding


class Embedding(nn.Embedding):
    """`nn.Embedding` (same parameters, same state dict) with a scale on its rows, on the framework's kernels
    (fused_ops/embedding.py).  `max_norm`, `scale_grad_by_freq` and `sparse` are not offered."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: Optional[int] = None, scale: float = 1.0, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device, dtype=dtype)
        self.scale = scale

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True, padding_idx: Optional[int] = None, scale: float = 1.0):
        layer = cls(*embeddings.shape, padding_idx=padding_idx, scale=scale, device="meta")
        layer.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return layer

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return embedding(tokens, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return super().extra_repr() + (f", scale={self.scale}" if self.scale != 1.0 else "")
