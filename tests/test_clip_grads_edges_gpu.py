"""Clipping by the gradients' norm at the ends of float32's range."""
import pytest
import torch

from megalodon_amd import fused_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_norm", [1e-3, 1e-7, 1e-20, 1e-38])
def test_factors_below_the_normal_numbers(max_norm, dtype, in_place):
    """Gradients near the largest numbers, whose norm only float64 holds, clipped to a small one: max_norm / norm is below 2^-126, down to where float32 has
    zero for it, and the clipped values are ordinary numbers.  The bar is that of ordinary factors: the norm's, the factor's and the product's roundings, half a
    step of the type (below its normal numbers of the smallest)."""
    g = torch.Generator("cuda").manual_seed(4)
    ts = [(6e37 * torch.randn(n, generator=g, device="cuda")).to(dtype) for n in (70001, 8, 40000)]
    wide = [t.double() for t in ts]
    norm = sum(t.square().sum() for t in wide).sqrt().item()
    assert norm > 3.5e38 and max_norm / norm < 2.0 ** -126
    got, new = fused_ops.clip_grads(ts, max_norm, out=ts if in_place else None)
    assert got.isinf()  # (float32 has no other number for it)
    info = torch.finfo(dtype)
    for n, t in zip(new, wide):
        v = t * (max_norm / (norm + 1e-6))
        bar = v.abs() * (3 * U + info.eps / 2) + info.smallest_normal * info.eps / 2 + 2.0 ** -149
        assert bool(((n.double() - v).abs() <= bar).all())
        if max_norm > 1e-30:
            assert n.any()


def test_offsets_beyond_32_bits():
    """A gradient of more than 2^32 elements between small ones: all counted, all scaled."""
    n = (1 << 32) + 100_001
    ts = [torch.ones(7, device="cuda"), torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda"), torch.ones(9, device="cuda")]
    ts[1][-3:] = 64.0
    want = (16 + (n - 3) * 0.25 + 3 * 4096) ** 0.5
    norm, out = fused_ops.clip_grads(ts, want / 4, out=ts)
    assert abs(norm.item() - want) <= 2 * U * want
    for t, v in zip(out, (0.25, 0.125, 0.25)):
        assert (t[:-3] - v).abs().max() <= 2.0 ** -8 * v
    assert (out[1][-3:] - 16).abs().max() <= 2.0 ** -8 * 16
