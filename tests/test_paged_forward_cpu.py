"""`_InnerAttention.forward_paged` refuses a gradient that it would have to drop, before anything is written."""
import pytest
import torch
from torch.autograd import forward_ad

from megalodon_amd.modules import PagedCache, _InnerAttention


def call(attn, q, k, v):
    cache = PagedCache(2, 16, 2, 16, 32)
    ints = [torch.tensor(t, dtype=torch.int32) for t in ([[0, 1]], [3], [0, 3])]
    return attn.forward_paged(q, k, v, cache, *ints)


def rows():
    return [torch.zeros(3, 2 * w, dtype=torch.bfloat16) for w in (16, 16, 32)]


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("which", range(3))
def test_a_gradient_is_refused(which, training):
    attn = _InnerAttention(16, 32, 2, 64, 0.0, "fused").train(training)
    x = rows()
    x[which].requires_grad_(True)
    with pytest.raises(RuntimeError, match="forward_paged has no gradient"):
        call(attn, *x)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # (past that: the operators want GPU tensors)
        call(attn, *x)


@pytest.mark.parametrize("which", range(3))
def test_a_tangent_is_refused(which):
    attn = _InnerAttention(16, 32, 2, 64, 0.0, "fused").eval()
    with forward_ad.dual_level():
        x = rows()
        x[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError, match="forward_paged has no gradient"):
            call(attn, *x)


def test_dropout_is_refused():
    with pytest.raises(RuntimeError, match="dropout"):
        call(_InnerAttention(16, 32, 2, 64, 0.1, "fused").train(), *rows())
