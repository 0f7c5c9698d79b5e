"""More rows in a call than a launch has threads for along one axis."""
import pytest
import torch

from megalodon_amd import fused_ops

pytestmark = pytest.mark.gpu


def test_rows_behind_two_to_the_26():
    n = 2 ** 26 + 3
    pages = -(-n // 65536)
    table = torch.randperm(pages, device="cuda").to(torch.int32).view(1, pages)
    k, v = (torch.randint(-2 ** 14, 2 ** 14, (n, 1, 16), dtype=torch.int16, device="cuda").view(torch.bfloat16) for _ in range(2))
    k_pages, v_pages = (torch.zeros(pages, 65536, 1, 16, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ints = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([n], [0, n], [0])]
    fused_ops.paged_cache_write(k, v, k_pages, v_pages, table, ints[0], ints[1])
    got = fused_ops.paged_cache_read(k_pages, v_pages, table, ints[2], ints[1], n)
    for pool, rows, back in ((k_pages, k, got[0]), (v_pages, v, got[1])):
        assert torch.equal(back.view(torch.int16), rows.view(torch.int16))
        line = pool.view(torch.int16)[table[0].long()].flatten(0, 1)
        assert torch.equal(line[:n], rows.view(torch.int16)) and not bool(line[n:].any())


@pytest.mark.parametrize("batch,heads", [(2 ** 22 + 5, 16), (2 ** 22 + 5, 1)])
def test_attention_of_as_many_sequences(batch, heads):
    """A token each at position 0, which has weight 1 whatever the score: the value itself.  Sequences share pages."""
    pages = 1021
    q = torch.ones(batch, heads, 16, dtype=torch.bfloat16, device="cuda")
    k = torch.randn(pages, 16, heads, 16, device="cuda").to(torch.bfloat16)
    v = torch.randn(pages, 16, heads, 16, device="cuda").to(torch.bfloat16)
    table = (torch.arange(batch, device="cuda") % pages).to(torch.int32).view(batch, 1)
    cu = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    fused_ops.paged_attention(q, k, v, table, torch.ones(batch, dtype=torch.int32, device="cuda"), cu, out=out)
    assert torch.equal(out, v[:, 0][table[:, 0].long()])
