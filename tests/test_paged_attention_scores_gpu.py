"""Paged attention where scores pass float32's largest number."""
import pytest
import torch

from megalodon_amd import fused_ops
from paged import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dv", [64, 1040])
@pytest.mark.parametrize("news,olds,bad", [([1], [40], 17), ([5], [300], 301), ([100], [20], 5), ([100], [20], 70), ([100], [700], 500)])
def test_scores_that_overflow(news, olds, bad, dv, bits):
    """q . k = 2^126 stands in float32, scale q . k = 2^130 does not: an infinity, whose row is NaN, as where the sum itself overflows; from
    the other side the key has no weight.  Rows in front of the key are as without."""
    for exponent, scale, sign in ((63, 16.0, 1), (63, 16.0, -1), (64, 2.0, 1), (64, 2.0, -1)):
        x = Batch(news, olds, 1, 1, 64, dv, 16, torch.bfloat16, bits, seed=31)
        x.q[..., 0] = 2.0 ** exponent
        x.k[..., 0] = 0.0
        page, slot = int(x.table[0, bad // 16]), bad % 16
        clean = fused_ops.paged_attention(x.q.cuda(), *x.pools(), x.ints(x.lengths), x.ints(x.cu), scale, 0, **x.exponents()).cpu()
        assert bool(torch.isfinite(clean).all())
        codes = torch.zeros(64)
        codes[0] = sign * (1.0 if bits == 8 else 2.0 ** exponent)
        x.k[page, slot, 0] = codes.to(x.k.dtype)
        if bits == 8:
            x.ke[page, slot] = 127 + exponent
        got = fused_ops.paged_attention(x.q.cuda(), *x.pools(), x.ints(x.lengths), x.ints(x.cu), scale, 0, **x.exponents()).cpu()
        blind = max(0, bad - olds[0])
        assert torch.equal(got[:blind], clean[:blind])
        if sign > 0:
            assert bool(torch.isnan(got[blind:]).all())
        else:
            assert bool(torch.isfinite(got[blind:]).all()) and bool((got[blind:] != 0).any())


def test_scores_that_overflow_in_another_piece():
    """The key with the infinite score is one workgroup's, the rows' other keys others'."""
    x = Batch([100], [9000], 1, 1, 64, 64, 16, torch.bfloat16, seed=32)
    x.q[..., 0], x.k[..., 0] = 2.0 ** 63, 0.0
    for bad in (3, 4500, 8999):
        y = x.k.clone()
        x.k[int(x.table[0, bad // 16]), bad % 16, 0] = 0
        x.k[int(x.table[0, bad // 16]), bad % 16, 0, 0] = 2.0 ** 63
        got = fused_ops.paged_attention(x.q.cuda(), *x.pools(), x.ints(x.lengths), x.ints(x.cu), 16.0, 0)
        assert bool(torch.isnan(got).all())
        x.k = y


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("news,heads,dv", [([512, 512], 64, 1024), ([200, 312, 512], 130, 128), ([1] * 16, 64, 1024), ([20] * 40, 30, 1024)])
def test_scores_that_overflow_where_a_workgroup_has_a_block(news, heads, dv, bits):
    x = Batch(news, [40] * len(news), heads, 1, 64, dv, 16, torch.bfloat16, bits, seed=33)
    x.q[..., 0], x.k[..., 0] = 2.0 ** 63, 0.0
    codes = torch.zeros(64)
    codes[0] = 1.0 if bits == 8 else 2.0 ** 63
    x.k[int(x.table[0, 1]), 4] = codes.to(x.k.dtype)  # position 20 of the first sequence
    if bits == 8:
        x.ke[int(x.table[0, 1]), 4] = 127 + 63
    got = fused_ops.paged_attention(x.q.cuda(), *x.pools(), x.ints(x.lengths), x.ints(x.cu), 16.0, 0, **x.exponents()).cpu()
    assert bool(torch.isnan(got[:news[0]]).all()) and bool(torch.isfinite(got[news[0]:]).all())
