"""Attention of new tokens over the paged cache against its definition in 64 bits."""
import math

import pytest
import torch

from megalodon_amd import fused_ops
from paged import Batch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def attend(x, scale, chunk, **more):
    return fused_ops.paged_attention(x.q.cuda(), *x.pools(), x.ints(x.lengths), x.ints(x.cu), scale, chunk, **x.exponents(), **more)


def check(got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound.clamp(min=1e-300)).max())} of what is allowed"


CASES = [
    # news, olds, heads, shared, dk, dv, page, chunk
    ([1], [0], 1, 1, 64, 64, 16, 0),
    ([1, 1, 1], [100, 0, 255], 2, 1, 256, 2048, 64, 256),
    ([3, 7, 0, 1], [100, 0, 5, 33], 2, 4, 128, 128, 16, 0),
    ([20, 31], [77, 3], 1, 1, 256, 512, 32, 0),
    ([70, 129, 1], [50, 0, 300], 1, 1, 256, 2048, 16, 64),
    ([9], [1000], 1, 2, 80, 48, 16, 100),
    ([2, 40], [31, 32], 1, 1, 512, 1040, 128, 0),
    ([5], [11], 1, 1, 272, 4096, 16, 0),
    ([1, 1], [9000, 63], 1, 1, 16, 16, 256, 0),
    ([0, 1, 2] * 25, [k * 7 % 50 for k in range(75)], 1, 1, 64, 128, 16, 0),
    ([200], [37], 3, 5, 64, 256, 32, 96),
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[2:]))
def test_against_the_definition(case, dtype, bits):
    news, olds, heads, shared, dk, dv, page, chunk = case
    x = Batch(news, olds, heads, shared, dk, dv, page, dtype, bits, seed=dk + dv, extra_rows=3)
    scale = dk ** -0.5
    want, bound = x.attention(scale, chunk)
    got = attend(x, scale, chunk)
    check(got, want, bound)
    assert bool((got[x.cu[-1]:] == 0).all())
    again = attend(x, scale, chunk)
    assert torch.equal(got, again)
    own = torch.full_like(got, 7.0)
    assert attend(x, scale, chunk, out=own) is not None
    assert torch.equal(own[:x.cu[-1]], got[:x.cu[-1]]) and bool((own[x.cu[-1]:] == 7).all())


@pytest.mark.parametrize("scale", [0.0, -0.7, 40.0])
def test_scales(scale):
    x = Batch([4, 50], [60, 0], 2, 1, 64, 64, 16, BF16, seed=5)
    want, bound = x.attention(scale, 0)
    check(attend(x, scale, 0), want, bound)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("news,olds", [([40, 3], [20, 0]), ([6, 2], [300, 7])])
@pytest.mark.parametrize("dv", [64, 1040, 2048])
def test_values_that_a_row_does_not_see_do_not_reach_it(news, olds, dv, bits):
    """Infinities and NaN in the key and the value of a later token: the rows before it are as without, those from it on are not."""
    x = Batch(news, olds, 1, 1, 64, dv, 16, F16, bits, seed=3)
    clean = attend(x, 0.2, 0).cpu()
    b, bad = 0, olds[0] + news[0] // 2
    page, slot = int(x.table[b, bad // 16]), bad % 16
    for spoil_k, value in ((True, math.nan), (False, math.inf), (False, math.nan)):
        y = Batch(news, olds, 1, 1, 64, dv, 16, F16, bits, seed=3)
        if bits == 8:
            value = math.nan
        (y.k if spoil_k else y.v)[page, slot] = torch.full((), value).to(y.k.dtype)
        got = attend(y, 0.2, 0).cpu()
        at = bad - olds[0]
        assert torch.equal(got[:at], clean[:at])
        assert not bool(torch.isfinite(got[at:news[0]]).any())
        assert torch.equal(got[news[0]:], clean[news[0]:])


def test_one_infinite_value_reaches_its_column_only():
    x = Batch([24], [8], 1, 1, 64, 256, 16, BF16, seed=9)
    clean = attend(x, 0.2, 0).cpu()
    x.v[int(x.table[0, 1]), 4, 0, 77] = math.inf  # position 20, row 12
    got = attend(x, 0.2, 0).cpu()
    keep = torch.ones_like(clean, dtype=torch.bool)
    keep[12:, 0, 77] = False
    assert torch.equal(got[keep], clean[keep]) and bool(torch.isposinf(got[12:, 0, 77]).all())


def test_rows_without_keys_are_zero():
    """More new rows than the sequence has positions, an empty sequence, a table that is too short."""
    x = Batch([5, 2], [3, 14], 1, 2, 64, 64, 16, BF16, seed=1)
    lengths = x.ints([2, 16])  # the first three rows of sequence 0 have no position
    got = fused_ops.paged_attention(x.q.cuda(), *x.pools(), lengths, x.ints(x.cu), 1.0, 0)
    assert bool((got[:3] == 0).all()) and bool((got[3:] != 0).any())
    assert bool((fused_ops.paged_attention(x.q.cuda(), *x.pools(), x.ints([0, -5]), x.ints(x.cu), 1.0, 0) == 0).all())
    k, v, table = x.pools()
    assert bool((fused_ops.paged_attention(x.q.cuda(), k, v, table[:, :0], x.ints(x.lengths), x.ints(x.cu), 1.0, 0) == 0).all())
    # positions behind the table have no keys: with chunks of 16, row 17 sees none of the 16 that there are
    beyond = fused_ops.paged_attention(x.q.cuda(), k, v, table[:, :1].contiguous(), x.ints([8, 18]), x.ints(x.cu), 1.0, 16)
    assert bool((beyond[5:] == 0).all()) and bool((beyond[:5] != 0).any())


def test_scores_of_minus_infinity_everywhere_give_zeros():
    x = Batch([1], [40], 1, 1, 64, 64, 16, BF16, seed=2)
    x.q[:] = 1
    for p in range(41):
        x.k[int(x.table[0, p // 16]), p % 16] = -math.inf
    assert bool((attend(x, 1.0, 0) == 0).all())


@pytest.mark.parametrize("bits", [16, 8])
def test_a_number_that_is_no_page_has_no_keys(bits):
    x = Batch([3], [61], 1, 1, 64, 64, 16, BF16, bits, seed=4)
    whole, _ = x.attention(0.3, 0)
    k, v = x.stored(0, 0, 64)
    seen = [p for p in range(64) if not 16 <= p < 32]
    for number in (-1, x.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        y = Batch([3], [61], 1, 1, 64, 64, 16, BF16, bits, seed=4)
        y.table[0, 1] = number
        got = attend(y, 0.3, 0).double().cpu()
        for t in range(3):
            keys = [p for p in seen if p <= 61 + t]
            want = torch.softmax(k[keys, 0] @ y.q[t, 0].double() * 0.3, 0) @ v[keys, 0]
            assert (got[t, 0] - want).abs().max() < 0.03 and (got[t, 0] - whole[t, 0]).abs().max() > 0.03


def test_layouts():
    """Pools whose heads lie outside their positions, keys and values side by side, strided rows of q, a strided table."""
    x = Batch([3, 18], [70, 5], 2, 2, 64, 128, 16, BF16, seed=6)
    want = attend(x, 0.2, 0)
    k, v, table = x.pools()
    lengths, cu, q = x.ints(x.lengths), x.ints(x.cu), x.q.cuda()
    outside = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]
    assert torch.equal(fused_ops.paged_attention(q, *outside, table, lengths, cu, 0.2, 0), want)
    both = torch.cat((k, v), -1)
    assert torch.equal(fused_ops.paged_attention(q, both[..., :64], both[..., 64:], table, lengths, cu, 0.2, 0), want)
    wide = torch.full((q.shape[0], q.shape[1], 96), math.nan, dtype=BF16, device="cuda")
    wide[..., 8:72] = q
    assert torch.equal(fused_ops.paged_attention(wide[..., 8:72], k, v, table, lengths, cu, 0.2, 0), want)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view_as(q).copy_(q)  # not on a 16-byte boundary
    assert torch.equal(fused_ops.paged_attention(odd, k, v, table, lengths, cu, 0.2, 0), want)
    every = torch.full((4, table.shape[1] + 3), -7, dtype=torch.int32, device="cuda")
    every[::2, :table.shape[1]] = table
    assert torch.equal(fused_ops.paged_attention(q, k, v, every[::2, :table.shape[1]], lengths, cu, 0.2, 0), want)
    assert torch.equal(fused_ops.paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, table, lengths, cu, 0.2, 0), want)


def test_pages_behind_two_to_the_31_elements():
    heads, page, dk, dv = 1, 16, 64, 2048
    pages = 2 ** 31 // (page * dv) + 100
    k = torch.zeros(pages, page, heads, dk, dtype=BF16, device="cuda")
    v = torch.zeros(pages, page, heads, dv, dtype=BF16, device="cuda")
    x = Batch([2], [30], heads, 1, dk, dv, page, BF16, seed=8)
    want, bound = x.attention(0.2, 0)
    far = torch.tensor([[pages - 1, pages - 50]], dtype=torch.int32)
    for i in range(2):
        k[far[0, i]], v[far[0, i]] = x.k[x.table[0, i]].cuda(), x.v[x.table[0, i]].cuda()
    got = fused_ops.paged_attention(x.q.cuda(), k, v, far.cuda(), x.ints(x.lengths), x.ints(x.cu), 0.2, 0)
    check(got, want, bound)


def test_streams_and_graphs():
    """Captured once, replayed with other lengths, tables and queries; two graphs in turn, an eager call between."""
    xs = [Batch([1, 1, 1], olds, 2, 1, 64, 256, 16, BF16, seed=10 + i, spare=20 - sum(-(-(o + 1) // 16) for o in olds))
          for i, olds in enumerate(([5, 90, 17], [100, 1, 33], [63, 64, 15]))]
    width = max(x.table.shape[1] for x in xs)
    for x in xs:
        x.table = torch.nn.functional.pad(x.table, (0, width - x.table.shape[1]), value=-1)
    k, v, table = xs[0].pools()
    q, lengths, cu = xs[0].q.cuda(), xs[0].ints(xs[0].lengths), xs[0].ints(xs[0].cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            fused_ops.paged_attention(q, k, v, table, lengths, cu, 0.2, 64)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(fused_ops.paged_attention(q, k, v, table, lengths, cu, 0.2, 64))
    for turn in range(6):
        x = xs[turn % 3]
        for to, new in zip((k, v, table), x.pools()):
            to.copy_(new)
        q.copy_(x.q)
        lengths.copy_(x.ints(x.lengths))
        graphs[turn % 2].replay()
        want, bound = x.attention(0.2, 64)
        check(outs[turn % 2], want, bound)
        assert torch.equal(outs[turn % 2], fused_ops.paged_attention(q, k, v, table, lengths, cu, 0.2, 64))
        torch.cuda.synchronize()


def test_refusals():
    x = Batch([2], [5], 2, 2, 64, 64, 16, BF16, seed=1)
    k, v, table = x.pools()
    q, lengths, cu = x.q.cuda(), x.ints(x.lengths), x.ints(x.cu)

    def call(q=q, k=k, v=v, table=table, lengths=lengths, cu=cu, scale=1.0, chunk=0, **more):
        return fused_ops.paged_attention(q, k, v, table, lengths, cu, scale, chunk, **more)

    call()
    out = torch.empty(2, 4, 64, dtype=BF16, device="cuda")
    codes, e = k.to(torch.float8_e4m3fn), torch.full(k.shape[:3], 127, dtype=torch.uint8, device="cuda")
    for bad in [dict(q=q.cpu()), dict(k=k.cpu()), dict(table=table.cpu()), dict(lengths=lengths.cpu()), dict(cu=cu.cpu()),
                dict(q=q.float()), dict(q=q.half()), dict(q=q[0]), dict(q=q[:, :3]), dict(q=q[..., :48]), dict(k=k.float(), v=v.float()),
                dict(v=v.half()), dict(v=v[:1]), dict(k=k[..., ::2]), dict(table=table.long()), dict(table=table[0]),
                dict(lengths=lengths.long()), dict(lengths=x.ints([1, 2])), dict(cu=x.ints([0])), dict(chunk=-1),
                dict(k=k[:, :8], v=v[:, :8]), dict(k=k[..., :40], q=q[..., :40]), dict(v=v[..., 8:]), dict(k=codes, v=codes),
                dict(k_exponents=e, v_exponents=e), dict(k=codes, v=codes, k_exponents=e), dict(k=codes, v=codes, k_exponents=e, v_exponents=e[:1]),
                dict(k=codes, v=codes, k_exponents=e.int(), v_exponents=e.int()), dict(k=k[:1].expand(4, -1, -1, -1), v=v[:1].expand(4, -1, -1, -1)),
                dict(out=out.float()), dict(out=out[:1]), dict(out=out.transpose(0, 1).contiguous().transpose(0, 1)), dict(out=q),
                dict(q=q.clone().requires_grad_(True))]:
        with pytest.raises(RuntimeError):
            call(**bad)
    with pytest.raises(RuntimeError):
        call(k=torch.zeros(1, 16, 2, 528, dtype=BF16, device="cuda"), v=v[:1], q=torch.zeros(2, 4, 528, dtype=BF16, device="cuda"))
    with torch.no_grad():
        call(q=q.clone().requires_grad_(True))
    empty = call(q=q[:0], cu=x.ints([0, 0]))
    assert empty.shape == (0, 4, 64)
    nobody = call(table=table[:0], lengths=lengths[:0], cu=x.ints([0]))
    assert bool((nobody == 0).all())
    kept = torch.full_like(out, 3)
    call(table=table[:0], lengths=lengths[:0], cu=x.ints([0]), out=kept)
    assert bool((kept == 3).all())
