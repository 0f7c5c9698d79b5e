"""The gated product at the ends of what its callers may do."""
import pytest
import torch

from megalodon_amd import fused_ops

pytestmark = pytest.mark.gpu


def operands(tokens, n_in, n_out, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + tokens + 7 * n_in + 11 * n_out)
    rows = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return (rows(tokens, n_in).to(dtype), (rows(n_out, n_in) / n_in ** 0.5).to(dtype), (rows(n_out, n_in) / n_in ** 0.5).to(dtype), rows(tokens, n_out).to(dtype))


def leaves_of(*tensors):
    return [t.clone().requires_grad_(True) for t in tensors]


# x (70, 72), w1 and w3 (36, 72), a and b (70, 40) float32: what a hook makes of the tensors that it recognises
SAVED = {
    "weights in another type": lambda t: t.float() if t.shape == (36, 72) else t,
    "weights in the other 16 bits": lambda t: t.half() if t.shape == (36, 72) else t,
    "rows in another type": lambda t: t.double() if t.shape == (70, 72) else t,
    "products in the other 16 bits": lambda t: t.half() if t.dtype == torch.float32 else t,
    "products in 64 bits": lambda t: t.double() if t.dtype == torch.float32 else t,
    "weights on the host": lambda t: t.cpu() if t.shape == (36, 72) else t,
    "rows on the host": lambda t: t.cpu() if t.shape == (70, 72) else t,
    "products on the host": lambda t: t.cpu() if t.dtype == torch.float32 else t,
    "fewer rows": lambda t: t[1:] if t.shape == (70, 72) else t,
    "narrower products": lambda t: t[:, :36] if t.dtype == torch.float32 else t,
}


@pytest.mark.parametrize("what", list(SAVED))
def test_saved_tensors_that_came_back_as_something_else(what):
    """What hooks hand back is refused where it is not what was saved any more, before anything is launched."""
    x, w1, w3, dh = operands(70, 72, 36, torch.bfloat16)
    leaves = leaves_of(x, w1, w3)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, SAVED[what]):
        h = fused_ops.gated_linear(*leaves)
        with pytest.raises(RuntimeError, match="saved tensor"):
            torch.autograd.grad(h, leaves, dh)


def test_saved_tensors_in_other_forms():
    """Negated on reading, in another layout: as they were."""
    x, w1, w3, dh = operands(70, 72, 36, torch.bfloat16)
    leaves = leaves_of(x, w1, w3)
    want = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
    for pack, back in ((lambda t: -t, torch._neg_view), (lambda t: t.t().contiguous(), lambda t: t.t())):
        with torch.autograd.graph.saved_tensors_hooks(pack, back):
            got = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
        assert all(torch.equal(g, w) for g, w in zip(got, want))
