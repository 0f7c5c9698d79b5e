"""`NormalizedFeedForwardNetwork` (megalodon/modules/normalized_feedforward_network.py:15-98)
for model-parallel world size 1: Column/RowParallelLinear are plain `nn.Linear`
(megalodon/modules/model_parallel/layers.py:222-235,321-341); the two dropouts
sit where the reference has them (:83-90).  `fused_gate`: with `swiglu` and 16-bit rows the two projections and the gate
(:82) are one operator, `fused_ops.gated_linear`, whose gate sees the products in float32; elsewhere, and by default, they are two
products and `silu_mul`.  The operator is ahead without gradients, and with them on ordinary sizes; its products are kept in float32, which costs the largest trainings
more than the gate's pass (32768 tokens, 4096 -> 11008 13.6 ms forward and backward, 13.0 without; 4096 tokens, 1024 -> 2752 0.197, 0.193)."""
import torch
import torch.nn.functional as F
from torch import nn

from ..fused_ops import gated_linear, memory_efficient_dropout, silu_mul
from .linear import Linear, is_bare, linear_group
from .layer_norm import FusedLayerNorm


class NormalizedFeedForwardNetwork(nn.Module):
    fused_gate = False  # (modules that were pickled without it)

    def __init__(self, model_dim, ffn_hidden_dim, dropout=0.0, hidden_dropout=0.0, swiglu=False,
                 norm_affine=True, norm_eps=1e-5, rescale=None, init_std=0.02, fused_gate=False):
        super().__init__()
        self.fused_gate = fused_gate
        self.dropout = dropout
        self.hidden_dropout = hidden_dropout
        self.model_dim = model_dim
        self.hidden_dim = ffn_hidden_dim
        self.swiglu = swiglu
        self.rescale_init = rescale
        self.norm = FusedLayerNorm(model_dim, elementwise_affine=norm_affine, eps=norm_eps)
        self.fc1 = Linear(model_dim, ffn_hidden_dim, bias=False)
        self.fc2 = Linear(ffn_hidden_dim, model_dim, bias=False)
        self.fc3 = Linear(model_dim, ffn_hidden_dim, bias=False) if swiglu else None
        for lin in (self.fc1, self.fc2, self.fc3):
            if lin is not None:
                nn.init.normal_(lin.weight, mean=0.0, std=init_std)
        if rescale is None:
            self.register_parameter('alpha', None)
        else:
            assert rescale > 0., 'Layer scale init value should be positive.'
            self.alpha = nn.Parameter(torch.full((model_dim,), rescale))

    def rescale(self, x: torch.Tensor) -> torch.Tensor:
        return x if self.alpha is None else (self.alpha * x)

    def takes_fused_gate(self, x: torch.Tensor) -> bool:
        """Rows and weights of one 16-bit type on the GPU, of sizes that the operator takes, and layers whose call is nothing but `Linear.forward`."""
        layers = (self.fc1, self.fc3)
        if not (x.is_cuda and x.dtype in (torch.bfloat16, torch.float16) and all(is_bare(l) and l.bias is None and l.weight.dtype == x.dtype for l in layers)):
            return False
        n_out, n_in = (-(-n // 64) * 64 for n in self.fc1.weight.shape)
        return 2 * n_in * n_out < 1 << 30 and max(n_in, n_out) <= 1 << 20 and not torch.is_autocast_enabled("cuda")

    def forward(self, x, residual):
        x = self.norm(x)
        if self.swiglu and self.fused_gate and self.takes_fused_gate(x):
            hidden = gated_linear(x, self.fc1.weight, self.fc3.weight)
        elif self.swiglu:
            hidden = silu_mul(*linear_group(x, (self.fc1, self.fc3)))
        else:
            hidden = F.silu(self.fc1(x))
        hidden = memory_efficient_dropout(hidden, self.hidden_dropout, self.training)
        if self.alpha is None and (self.dropout == 0.0 or not self.training):
            return self.fc2(hidden, residual=residual)   # fc2(hidden) + residual, the sum formed inside the GEMM
        x = self.fc2(hidden)
        x = memory_efficient_dropout(x, self.dropout, self.training)
        return self.rescale(x) + residual

    def extra_repr(self) -> str:
        return 'dim={}, hdim={}, swiglu={}, rescale={}'.format(self.model_dim, self.hidden_dim, self.swiglu,
                                                             self.rescale_init)
