"""The norm of all gradients together, and clipping by it (`clip_grad_norm_` of the reference's training,
megalodon/distributed/fairscale_fsdp.py, on one device); the kernels are csrc/clip.hip.

Tensors are float32, bfloat16 or float16, types mixed as they come, dense (any order of the axes, no gaps), on one
device; norm_type is 2 or infinity.  Squares and sums are float64, the same bits from call to call.  Nothing is recorded for autograd and nothing
synchronises; the calls may be captured into a graph."""
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from .. import _lib


def grad_norm(tensors: Sequence[Tensor], norm_type: float = 2.0) -> Tensor:
    """The norm of all elements of all tensors: float32, no axes.  Without tensors 0, on the CPU."""
    tensors = list(tensors)
    return _lib.host().grad_norm(tensors, norm_type, False) if tensors else torch.tensor(0.0)


def clip_grads(tensors: Sequence[Tensor], max_norm: float, norm_type: float = 2.0,
               out: Optional[Sequence[Tensor]] = None) -> Tuple[Tensor, List[Tensor]]:
    """(norm, clipped): each tensor times min(1, max_norm / (norm + 1e-6)), in `out` (shapes, strides and dtypes of the tensors; the
    tensors themselves for clipping in place) or in new tensors.  In place, nothing is written where nothing is to be scaled."""
    tensors = list(tensors)
    out = [torch.empty_like(t) for t in tensors] if out is None else list(out)
    if not tensors and not out:
        return torch.tensor(0.0), out
    return _lib.host().clip_grads(tensors, out, max_norm, norm_type, False), out


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float, norm_type: float = 2.0) -> Tensor:
    """`torch.nn.utils.clip_grad_norm_` for what this module takes: clips the `.grad` of the parameters (those that have one) in place, returns their norm.

    Raises for other norms, gradients of float64 or with gaps, and parameters that share a gradient; there is no `error_if_nonfinite`: as
    nothing synchronises, a norm that is not finite is returned, and the gradients are scaled by it (NaN, or zeros for an infinite norm's finite ones)."""
    parameters = [parameters] if isinstance(parameters, Tensor) else parameters
    grads = [p.grad for p in parameters if p.grad is not None]
    return _lib.host().clip_grads(grads, grads, max_norm, norm_type, True) if grads else torch.tensor(0.0)
