"""`_InnerAttention.forward_paged` against `_InnerAttention.forward` on its own contiguous cache."""
import pytest
import torch

from megalodon_amd.modules import PagedCache, _InnerAttention
from paged import UNIT

pytestmark = pytest.mark.gpu

HEADS, DK, DV, CHUNK, PAGE = 2, 64, 128, 48, 16


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_like_the_contiguous_cache(dtype):
    """Two sequences, a prompt (of whole chunks, or short of one) and then tokens one by one across a chunk's end.  Each side is off from the
    exact result by half a step of it and half a step of the probabilities: u (|o| + A) with A = sum_j p_j |v_j| <= max |v|, what float32 adds is
    below 2^-16 A; the two together by twice that.  (Float16's probabilities below 2^-14: another 2^-25 sum |v| each.)"""
    attn = _InnerAttention(DK, DV, HEADS, CHUNK, 0.0, "fused").eval()
    prompts, tokens = [2 * CHUNK, 41], 20
    gen = torch.Generator().manual_seed(3)
    whole = [[torch.randn(n + tokens, HEADS * w, generator=gen).mul(s).to(dtype).cuda() for w, s in ((DK, DK ** -0.5), (DK, 1.0), (DV, 1.0))] for n in prompts]
    cache = PagedCache(24, PAGE, HEADS, DK, DV, dtype=dtype, device="cuda")
    table = ints(torch.randperm(24, generator=gen)[:16].view(2, 8).tolist())
    own = [(torch.empty(1, 0, HEADS, DK, dtype=dtype, device="cuda"), torch.empty(1, 0, HEADS, DV, dtype=dtype, device="cuda"), 0) for _ in prompts]
    done = [0, 0]
    for step in range(tokens + 1):
        n = prompts if step == 0 else [1, 1]
        parts = [[t[d:d + m] for t in x] for x, d, m in zip(whole, done, n)]
        done = [d + m for d, m in zip(done, n)]
        got = attn.forward_paged(*(torch.cat(t) for t in zip(*parts)), cache, table, ints(done), ints([0, n[0], n[0] + n[1]]))
        at = 0
        for b in range(2):
            want, own[b] = attn(*(t[None] for t in parts[b]), None, None, own[b])
            top = whole[b][2][:done[b]].float().abs().max()
            bound = 2.02 * UNIT[dtype] * (want[0].float().abs() + top) + 2.0 ** -15 * top + 2.0 ** -24 * (1 + CHUNK * top)
            assert bool(((got[at:at + n[b]].float() - want[0].float()).abs() <= bound).all())
            at += n[b]


def test_a_refused_call_writes_nothing():
    attn = _InnerAttention(DK, DV, HEADS, CHUNK, 0.0, "fused").eval()
    cache = PagedCache(2, PAGE, HEADS, DK, DV, device="cuda")
    q, k, v = (torch.ones(3, HEADS * w, dtype=torch.bfloat16, device="cuda") for w in (DK, DK, DV))
    args = cache, ints([[0, 1]]), ints([3]), ints([0, 3])
    with pytest.raises(RuntimeError, match="gradient"):
        attn.forward_paged(q.clone().requires_grad_(True), k, v, *args)
    assert bool((cache.k_pages == 0).all())
    with torch.no_grad():
        out = attn.forward_paged(q.clone().requires_grad_(True), k, v, *args)
    assert bool((out == 1).all()) and not out.requires_grad
