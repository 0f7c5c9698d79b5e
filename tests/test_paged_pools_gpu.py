"""Keys and values written to pools that lie between each other, and pools that are one another's memory."""
import pytest
import torch

from megalodon_amd import fused_ops
from paged import Batch

pytestmark = pytest.mark.gpu

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def write(x, k, v, rows, **ex):
    fused_ops.paged_cache_write(*rows, k, v, x.table.cuda(), x.ints(x.lengths), x.ints(x.cu), **ex)
    return fused_ops.paged_cache_read(k, v, x.table.cuda(), x.ints(x.olds), x.ints(x.cu), x.cu[-1], **ex)


def test_pools_between_each_other():
    x = Batch([5, 20], [3, 10], 2, 1, 32, 48, 16, BF16, seed=2)
    pages, rows = x.k.shape[0], [torch.randn(25, 2, w).to(BF16).cuda() for w in (32, 48)]
    row = torch.zeros(pages, 16, 2, 80, dtype=BF16, device="cuda")
    slot = torch.zeros(pages, 16, 160, dtype=BF16, device="cuda")
    page = torch.zeros(pages, 16 * 160, dtype=BF16, device="cuda")
    for k, v in ((row[..., :32], row[..., 32:]), (slot[..., :64].unflatten(2, (2, 32)), slot[..., 64:].unflatten(2, (2, 48))),
                 (page[:, :1024].view(pages, 16, 2, 32), page[:, 1024:].view(pages, 2, 16, 48).transpose(1, 2))):
        assert all(torch.equal(a, b) for a, b in zip(write(x, k, v, rows), rows))


def test_pools_of_the_same_memory_are_refused():
    x = Batch([2], [5], 2, 1, 64, 64, 16, BF16, 8, seed=1)
    rows = [torch.zeros(2, 2, 64, dtype=BF16, device="cuda") for _ in range(2)]
    k, v, _ = x.pools()
    e, f = x.exponents().values()
    write(x, k, v, rows, k_exponents=e, v_exponents=f)
    before = k.clone().view(torch.uint8), e.clone()
    for pools, ex in (((k, k), (e, f)), ((k, v), (e, e)), ((k, k[...]), (e, f)), ((k, v), (e, k.view(torch.uint8)[..., 5]))):
        with pytest.raises(RuntimeError, match="share memory"):
            write(x, *pools, rows, k_exponents=ex[0], v_exponents=ex[1])
    inside = torch.zeros(4, 16, 2, 64, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="share memory"):
        write(x, inside, inside, rows)
    room = torch.full((4096,), 127, dtype=torch.uint8, device="cuda")  # exponents, and new rows on them
    with pytest.raises(RuntimeError, match="new rows"):
        write(x, k, v, [room[:512].view(BF16).view(2, 2, 64), rows[1]], k_exponents=room[:e.numel()].view(e.shape), v_exponents=f)
    assert torch.equal(k.view(torch.uint8), before[0]) and torch.equal(e, before[1])
    with pytest.raises(RuntimeError, match="overlap"):
        fused_ops.paged_attention(x.q.cuda(), k, v, x.table.cuda(), x.ints(x.lengths), x.ints(x.cu), k_exponents=room[:e.numel()].view(e.shape), v_exponents=f,
                                  out=room[:512].view(BF16).view(2, 2, 64))
    # reading them is nobody's harm
    a, b = fused_ops.paged_cache_read(k, k, x.table.cuda(), x.ints(x.olds), x.ints(x.cu), 2, e, e)
    assert torch.equal(a, b)
