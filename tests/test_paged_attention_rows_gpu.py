"""Paged attention in blocks of many rows and in mixed batches, the ways a call is cut, and what may not touch it."""
import math

import pytest
import torch

from megalodon_amd import fused_ops
from paged import Batch, to_8_bits

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def attend(x, scale, chunk, **more):
    return fused_ops.paged_attention(x.q.cuda(), *x.pools(), x.ints(x.lengths), x.ints(x.cu), scale, chunk, **x.exponents(), **more)


def check(got, want, bound, heads=slice(None)):
    off = (got.double().cpu() - want)[:, heads].abs()
    assert bool((off <= bound[:, heads]).all()), f"off by {float((off / bound[:, heads].clamp(min=1e-300)).max())} of what is allowed"


CASES = [
    # news, olds, heads, shared, dk, dv, page, chunk
    ([150], [300], 2, 1, 128, 128, 16, 0),               # one sequence, blocks that see much the same
    ([150], [300], 1, 1, 256, 256, 32, 0),
    ([130], [400], 2, 1, 128, 1024, 64, 0),
    ([65], [1], 1, 1, 128, 384, 16, 0),                  # ... that do not: three waves, a block of one row
    ([300], [0], 1, 2, 256, 2048, 64, 128),              # two slabs of columns, chunks
    ([33, 64, 63], [4000, 0, 17], 1, 1, 64, 112, 128, 0),
    ([200, 1, 1, 33, 0, 64], [10, 500, 3, 100, 9, 64], 1, 1, 128, 128, 16, 0),
    ([200, 1, 1, 33, 0, 64], [10, 500, 3, 100, 9, 64], 1, 3, 160, 640, 16, 48),
    ([90 if i % 3 else 1 for i in range(70)], [i * 13 % 200 for i in range(70)], 1, 1, 64, 64, 16, 64),
    ([700], [5000], 1, 1, 32, 32, 64, 4096),             # a chunk ends inside the new rows
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-" + "-".join(str(x) for x in c[2:]))
def test_against_the_definition(case, dtype, bits):
    news, olds, heads, shared, dk, dv, page, chunk = case
    x = Batch(news, olds, heads, shared, dk, dv, page, dtype, bits, seed=dk + dv, extra_rows=2)
    scale = dk ** -0.5
    want, bound = x.attention(scale, chunk)
    got = attend(x, scale, chunk)
    check(got, want, bound)
    assert bool((got[x.cu[-1]:] == 0).all())
    own = torch.full_like(got, 7.0)
    attend(x, scale, chunk, out=own)
    assert torch.equal(own[:x.cu[-1]], got[:x.cu[-1]]) and bool((own[x.cu[-1]:] == 7).all())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("news,olds,heads", [([512, 512], [0, 77], 64), ([1] * 16, [k * 9 for k in range(16)], 64), ([20] * 40, [5] * 40, 30)])
def test_as_many_blocks_as_there_is_room_for(news, olds, heads, bits):
    """Workgroups enough without cutting a block: a workgroup a block, no workspace."""
    x = Batch(news, olds, heads, 1, 64, 1024, 16, BF16, bits, seed=heads, extra_rows=3)
    some = [0, heads // 3, heads - 1]
    want, bound = x.attention(0.125, 64, some)
    got = attend(x, 0.125, 64)
    check(got, want, bound, some)
    assert bool((got[x.cu[-1]:] == 0).all())
    own = torch.full_like(got, 7.0)
    attend(x, 0.125, 64, out=own)
    assert torch.equal(own[:x.cu[-1]], got[:x.cu[-1]]) and bool((own[x.cu[-1]:] == 7).all())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(scale, bits):
    x = Batch([100], [200], 1, 1, 256, 128, 16, F16, bits, seed=5)
    want, bound = x.attention(scale, 0)
    check(attend(x, scale, 0), want, bound)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dv", [64, 128, 1040])
@pytest.mark.parametrize("news,olds", [([100], [20]), ([80, 40], [300, 7])])
def test_values_that_a_row_does_not_see_do_not_reach_it(news, olds, dv, bits):
    clean = attend(Batch(news, olds, 1, 1, 64, dv, 16, BF16, bits, seed=3), 0.2, 0).cpu()
    bad = olds[0] + news[0] // 2
    for spoil_k, value in ((True, math.nan), (False, math.inf), (False, math.nan)):
        y = Batch(news, olds, 1, 1, 64, dv, 16, BF16, bits, seed=3)
        pool = y.k if spoil_k else y.v
        pool[int(y.table[0, bad // 16]), bad % 16] = torch.full((), math.nan if bits == 8 else value).to(pool.dtype)
        got, at = attend(y, 0.2, 0).cpu(), bad - olds[0]
        assert torch.equal(got[:at], clean[:at])
        assert not bool(torch.isfinite(got[at:news[0]]).any())
        assert torch.equal(got[news[0]:], clean[news[0]:])


def test_small_8_bit_numbers_in_float16():
    """Below 2^-14 float16's numbers are 2^-24 apart: a stored key or value that is read as one is off by 2^-25 at most, a
    score then by scale 2^-25 sum |q|, which moves a probability by a factor within 1 +- 2.1 times that."""
    for news, olds in (([100], [60]), ([3], [200])):
        x = Batch(news, olds, 1, 1, 128, 128, 16, F16, 8, seed=11)
        x.ke -= 16
        x.ve -= 16
        scale = 300.0
        want, bound = x.attention(scale, 0)
        moved = 2.1 * scale * 2.0 ** -25 * x.q.double().abs().sum(-1).max()
        top = max(float(x.stored(0, 0, x.lengths[0])[1].abs().max()), 0.0)
        check(attend(x, scale, 0), want, bound + moved * top + 2.0 ** -25)


@pytest.mark.parametrize("news", [1, 100])
def test_many_small_probabilities_keep_their_weight(news):
    """One key with a score of zero, 16384 with p = 2^-20.4 of its own, which float16 holds to 2^-4.6 of itself only: lifted, each is off
    by 2^-11, the result's rounding by 2^-11, the sums by 16400 2^-23, the scores (one product each) by 14.2 2^-22."""
    n, x = 16384, Batch([news], [16384], 1, 1, 16, 16, 256, F16, seed=12)
    x.q.zero_(), x.k.zero_(), x.v.zero_()
    x.q[:, 0, 0] = 1
    low = float(torch.tensor(-20.4 * math.log(2)).half())
    for p in range(n):
        page, slot = int(x.table[0, p // 256]), p % 256
        x.k[page, slot, 0, 0], x.v[page, slot] = low, 1
    x.v[int(x.table[0, n // 256]), n % 256] = 0
    got = attend(x, 1.0, 0)[0].double().cpu()
    tail = n * math.exp(low)
    want = tail / (1 + tail)
    assert bool(((got - want).abs() <= (2.0 ** -10 + 16400 * 2.0 ** -23 + 14.2 * 2.0 ** -22) * 1.01 * want).all())


def test_pages_of_several_sequences():
    x = Batch([3, 70, 2], [60, 64, 40], 2, 1, 64, 128, 16, BF16, seed=13)
    x.table[1, :3], x.table[2, :2] = x.table[0, :3].clone(), x.table[0, :2].clone()
    want, bound = x.attention(0.2, 0)
    check(attend(x, 0.2, 0), want, bound)


@pytest.mark.parametrize("rows", [6, 130])
def test_two_calls_at_once(rows):
    xs = [Batch([rows, rows // 2], [700 + 50 * i, 33], 2, 1, 128, 512, 16, BF16, seed=14 + i) for i in range(2)]
    alone = [attend(x, 0.1, 0) for x in xs]
    args = [(x.q.cuda(), *x.pools(), x.ints(x.lengths), x.ints(x.cu), 0.1, 0) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(fused_ops.paged_attention(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])


def test_a_graph_follows_the_batch():
    """The same rows dealt to sequences in other ways and lengths from replay to replay, eager calls between."""
    deals = [([200, 0, 10], [100, 900, 30]), ([1, 208, 1], [640, 3, 77]), ([70, 70, 70], [0, 1, 2]), ([0, 0, 210], [5, 5, 500])]
    xs = [Batch(a, b, 2, 1, 128, 256, 16, BF16, seed=20 + i, spare=80 - sum(-(-(p + q) // 16) for p, q in zip(a, b))) for i, (a, b) in enumerate(deals)]
    width = max(x.table.shape[1] for x in xs)
    for x in xs:
        x.table = torch.nn.functional.pad(x.table, (0, width - x.table.shape[1]), value=-1)
    now = [*xs[0].pools(), xs[0].ints(xs[0].lengths), xs[0].ints(xs[0].cu), xs[0].q.cuda()]

    def call():
        k, v, table, lengths, cu, q = now
        return fused_ops.paged_attention(q, k, v, table, lengths, cu, 0.1, 512)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for turn in (0, 1, 2, 3, 1, 0):
        x = xs[turn]
        for to, new in zip(now, (*x.pools(), x.ints(x.lengths), x.ints(x.cu), x.q)):
            to.copy_(new)
        graph.replay()
        want, bound = x.attention(0.1, 512)
        check(out, want, bound)
        assert torch.equal(out, call())
        torch.cuda.synchronize()


@pytest.mark.parametrize("news,olds", [([60, 80], [200, 5]), ([2, 4], [200, 5])])
def test_rows_in_front_of_the_first_sequence_are_left(news, olds):
    x = Batch(news, olds, 2, 1, 64, 128, 16, BF16, seed=15)
    want = attend(x, 0.2, 0)
    q = torch.cat((torch.full_like(x.q[:5], math.nan), x.q)).cuda()
    out = torch.full((q.shape[0], 2, 128), 7.0, dtype=BF16, device="cuda")
    fused_ops.paged_attention(q, *x.pools(), x.ints(x.lengths), x.ints([5 + c for c in x.cu]), 0.2, 0, out=out)
    assert bool((out[:5] == 7).all()) and torch.equal(out[5:], want)


@pytest.mark.parametrize("cu", [[0, 130, 20, 150], [0, 150, 0, 150], [0, 200, 300, 1 << 30], [-7, 150, -9, 90]])
def test_bounds_that_make_no_sense_stay_inside(cu):
    """Nothing is said of the rows; the call ends, and what lies beside out and the next call are as they were."""
    x = Batch([50, 50, 50], [100, 0, 30], 2, 1, 64, 128, 16, BF16, seed=16)
    want = attend(x, 0.2, 0)
    room = torch.full((170, 2, 128), 7.0, dtype=BF16, device="cuda")
    fused_ops.paged_attention(x.q.cuda(), *x.pools(), x.ints(x.lengths), x.ints(cu), 0.2, 0, out=room[10:160])
    torch.cuda.synchronize()
    assert bool((room[:10] == 7).all()) and bool((room[160:] == 7).all())
    assert torch.equal(attend(x, 0.2, 0), want)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dv", [128, 272, 1040])
@pytest.mark.parametrize("news,olds", [([1], [900]), ([100], [900]), ([70, 40], [300, 650])])
@pytest.mark.parametrize("rising", [True, False])
def test_maxima_that_rise_all_the_way_or_never(news, olds, dv, bits, rising):
    """Keys along one direction whose scores rise by some 2^9 a tile of 32 keys, or fall by that: m follows at every tile, or never."""
    x = Batch(news, olds, 1, 1, 64, dv, 16, BF16, 16, seed=17)
    x.q[..., 0] = 8.0
    for b in range(len(news)):
        for p in range(x.lengths[b]):
            x.k[int(x.table[b, p // 16]), p % 16, 0, 0] = (p if rising else -p) / 32
    if bits == 8:
        whole = x
        x = Batch(news, olds, 1, 1, 64, dv, 16, BF16, 8, seed=17)
        x.q = whole.q
        codes, e = to_8_bits(whole.k)
        x.k, x.ke = codes.to(torch.float8_e4m3fn), e
    want, bound = x.attention(0.8, 0)
    check(attend(x, 0.8, 0), want, bound)
