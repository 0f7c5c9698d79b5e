"""Embedding's gradient at the ends of its ranges.

Where gradients are small whole numbers, every sum of them below 2^24 is exact in float32, in any order, and a result is that sum rounded once."""
import pytest
import torch

from megalodon_amd import fused_ops

pytestmark = pytest.mark.gpu


def test_more_pieces_than_a_launch_has_threads_for():
    """Rows of 8 columns have pieces of 4 positions: from 2^26 tokens on a workgroup for each, of 256 threads, would be 2^32 threads and more."""
    n, V, D = (1 << 26) + 12345, 1009, 8
    g = torch.Generator("cuda").manual_seed(1)
    tokens = torch.randint(0, V, (n,), generator=g, device="cuda", dtype=torch.int32)
    tokens[::5] = 77  # one that has a fifth of the positions
    dy = torch.randint(-1, 3, (n, D), generator=g, device="cuda", dtype=torch.int8).bfloat16()
    weight = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    junk = torch.full((V, D), 7.0, dtype=torch.bfloat16, device="cuda")  # (what the gradient's memory held)
    y = fused_ops.embedding(tokens, weight)
    del junk
    dw, = torch.autograd.grad(y, weight, dy)
    del y
    want = torch.stack([torch.bincount(tokens, dy[:, d].double(), minlength=V) for d in range(D)], 1)
    assert want.abs().max() < 1 << 24
    assert torch.equal(dw, want.to(torch.float32).bfloat16())
