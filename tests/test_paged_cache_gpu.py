"""Writing to the paged cache and reading it back: bit for bit."""
import math

import pytest
import torch

from megalodon_amd import fused_ops
from megalodon_amd.modules import PagedCache, _InnerAttention
from paged import UNIT, Batch, powers, to_8_bits

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
SHAPES = [
    # news, olds, heads, dk, dv, page
    ([1], [0], 1, 16, 16, 16),
    ([1, 1, 1], [15, 16, 17], 4, 256, 2048, 16),
    ([40, 0, 3], [5, 9, 63], 2, 64, 128, 64),
    ([7, 130], [0, 1], 3, 80, 4096, 32),
    ([1, 0, 2] * 30, [k * 5 % 40 for k in range(90)], 1, 512, 144, 16),
]


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x) for x in s[2:]))
def test_write_and_read(shape, dtype, bits):
    news, olds, heads, dk, dv, page = shape
    x = Batch(news, olds, heads, 1, dk, dv, page, dtype, bits, seed=dk)
    gen = torch.Generator().manual_seed(dv)
    rows = {"k": dk, "v": dv}
    new = {what: (torch.randn(x.cu[-1] + 2, heads, w, generator=gen) * 2.0 ** torch.randint(-9, 9, (x.cu[-1] + 2, heads, 1), generator=gen)).to(dtype)
           for what, w in rows.items()}
    k, v, table = x.pools()
    ex = x.exponents()
    fused_ops.paged_cache_write(new["k"].cuda(), new["v"].cuda(), k, v, table, x.ints(x.lengths), x.ints(x.cu), **ex)
    got = fused_ops.paged_cache_read(k, v, table, x.ints(x.olds), x.ints(x.cu), x.cu[-1] + 2, dtype=dtype, **ex)
    for what, pool, old_pool, back in (("k", k, x.k, got[0]), ("v", v, x.v, got[1])):
        want = old_pool.clone()
        codes, e = to_8_bits(new[what]) if bits == 8 else (new[what], None)
        exps = {"k": x.ke, "v": x.ve}[what]
        exps = None if exps is None else exps.clone()
        for b, n in enumerate(news):
            for i in range(n):
                p = olds[b] + i
                where = (int(x.table[b, p // page]), p % page)
                want[where] = codes[x.cu[b] + i].to(want.dtype)
                if exps is not None:
                    exps[where] = e[x.cu[b] + i]
        assert same_bits(pool.cpu(), want)  # what is not written is as it was
        stood_for = new[what].double() if bits == 16 else codes * powers(e)[..., None]
        assert torch.equal(back[:x.cu[-1]].double().cpu(), stood_for[:x.cu[-1]].to(dtype).double())
        assert bool((back[x.cu[-1]:] == 0).all())
        if exps is not None:
            assert torch.equal(ex[what + "_exponents"].cpu(), exps)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rounding_at_the_edges(dtype):
    """Ties, subnormal numbers of both types, the largest numbers, zeros, infinities and NaN."""
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = [[0.0] * 16, [-0.0] + [0.0] * 15, [top, -top] + [0.0] * 14, [top * 0.97, top / 3, top / 5, -top / 7] * 4,
            [tiny / 4, tiny / 2, -tiny, tiny * 0.75] * 4, [448.0, 447.0, 432.0, 416.0, 17.0, 18.0, 19.0, 21.0, 23.0, 25.0, 27.0, 29.0, 31.0, 33.0, 34.0, 38.0],
            [449.0, 448.0, 2.0 ** -6, 2.0 ** -7, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 5 * 2.0 ** -10, 2.0 ** -11, 7 * 2.0 ** -11, -2.0 ** -9, 1.0, 1.125, 1.0625, 1.1875, 0.0],
            [math.inf, 1.0, -math.inf, 2.0] * 4, [math.nan, 5.0, -3.0, 0.1] * 4, [math.nan, math.inf] * 8,
            [0.875, 0.876953125, 1.75, 1.7578125] * 4, [2.0 ** -14, 2.0 ** -15, 2.0 ** -20, 2.0 ** -24] * 4]
    x = torch.tensor(rows).to(dtype).unsqueeze(1)
    n = len(rows)
    k, v = (torch.zeros(1, 16, 1, 16, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    ke, ve = (torch.zeros(1, 16, 1, dtype=torch.uint8, device="cuda") for _ in range(2))
    ints = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([[0]], [n], [0, n], [0])]
    fused_ops.paged_cache_write(x.cuda(), x.flip(0).contiguous().cuda(), k, v, ints[0], ints[1], ints[2], ke, ve)
    codes, e = to_8_bits(x)
    got = k[0, :n].float().double().cpu()
    assert torch.equal(ke[0, :n].cpu(), e)
    assert torch.equal(got.nan_to_num(-9e9), codes.nan_to_num(-9e9)) and torch.equal(v[0, :n].float().double().cpu().nan_to_num(-9e9), codes.flip(0).nan_to_num(-9e9))
    back, _ = fused_ops.paged_cache_read(k, v, ints[0], ints[3], ints[2], n, ke, ve, dtype)
    finite = torch.isfinite(x)
    assert torch.equal(torch.isfinite(back.cpu()), finite)  # a finite number stays finite
    # to nearest: half a step of e4m3, relative for normal codes and 2^-10 codes below, and never past the type's largest
    unit = powers(e)[..., None]
    off = (back.double().cpu() - x.double())[finite]
    room = torch.maximum(x.double().abs() * 2.0 ** -4, unit * 2.0 ** -10)
    room = torch.where(x.double().abs() > 240 * unit, torch.maximum(room, (x.double().abs() - 240 * unit)), room)
    assert bool((off.abs() <= (room + torch.finfo(dtype).smallest_normal * UNIT[dtype])[finite]).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_every_code_and_exponent(dtype):
    """What is read is code * 2^(exponent - 127) rounded to the type, subnormal results and overflow included."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    exps = torch.arange(1, 255, dtype=torch.uint8)
    k = codes.view(1, 1, 1, 256).expand(16, 16, 1, 256).contiguous().cuda()
    e = torch.full((256,), 127, dtype=torch.uint8)
    e[:254] = exps
    e = e.view(16, 16, 1).cuda()
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(1, 16)
    zero, cu = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([0, 254], dtype=torch.int32, device="cuda")
    got, _ = fused_ops.paged_cache_read(k, k.clone(), table, zero, cu, 254, e, e, dtype)
    want = (codes.float().double().view(1, 1, 256) * powers(exps).view(254, 1, 1)).to(dtype)
    assert torch.equal(got.cpu().float().nan_to_num(nan=-1e30), want.float().nan_to_num(nan=-1e30))


def test_places_that_do_not_exist():
    """Positions in front of the first, behind the table, on no page: dropped, or zeros, and nothing else is touched."""
    x = Batch([6], [40], 1, 1, 16, 32, 16, BF16, seed=1)
    k, v, table = x.pools()
    new_k, new_v = torch.randn(6, 1, 16).to(BF16).cuda(), torch.randn(6, 1, 32).to(BF16).cuda()
    for length, entry in ((2, None), (-3, None), (16 * table.shape[1] + 6, None), (2 ** 31 - 1, None), (38, -1), (38, x.k.shape[0]), (38, -2 ** 31)):
        t = table.clone()
        if entry is not None:
            t[0, 2] = entry
        a, b = k.clone(), v.clone()
        fused_ops.paged_cache_write(new_k, new_v, a, b, t, x.ints([length]), x.ints([0, 6]))
        placed = [p for p in range(length - 6, length) if 0 <= p < 16 * t.shape[1] and 0 <= int(t[0, p // 16]) < k.shape[0]]
        for p in placed:
            i = p - (length - 6)
            assert same_bits(a[int(t[0, p // 16]), p % 16], new_k[i]) and same_bits(b[int(t[0, p // 16]), p % 16], new_v[i])
        changed = (a.view(torch.int16) != k.view(torch.int16)).any(-1).sum()
        assert int(changed) <= len(placed)
        got, _ = fused_ops.paged_cache_read(a, b, t, x.ints([length - 6]), x.ints([0, 6]), 6)
        for i in range(6):
            if length - 6 + i not in placed:
                assert bool((got[i] == 0).all())
    got, _ = fused_ops.paged_cache_read(k, v, table, x.ints([2 ** 31 - 4]), x.ints([0, 6]), 6)
    assert bool((got == 0).all())


def test_layouts_of_rows_and_pools():
    x = Batch([5, 20], [3, 10], 2, 1, 64, 128, 16, BF16, 8, seed=2)
    k, v, table = x.pools()
    ex = x.exponents()
    lengths, cu = x.ints(x.lengths), x.ints(x.cu)
    wide = torch.randn(25, 2, 64 + 128 + 16).to(BF16).cuda()
    plain = wide[..., :64].contiguous(), wide[..., 64:192].contiguous()
    fused_ops.paged_cache_write(*plain, k, v, table, lengths, cu, **ex)
    want = fused_ops.paged_cache_read(k, v, table, x.ints([0, 0]), x.ints([0, 8, 38]), 38, **ex)
    k2, v2 = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in x.pools()[:2])
    ex2 = {name: t.transpose(1, 2).contiguous().transpose(1, 2) for name, t in x.exponents().items()}
    fused_ops.paged_cache_write(wide[..., :64], wide[..., 64:192], k2, v2, table, lengths, cu, **ex2)
    got = fused_ops.paged_cache_read(k2, v2, table, x.ints([0, 0]), x.ints([0, 8, 38]), 38, **ex2)
    assert all(same_bits(a, b) for a, b in zip(got, want))
    odd = torch.empty(25 * 2 * 64 + 1, dtype=BF16, device="cuda")[1:].view(25, 2, 64).copy_(plain[0])
    fused_ops.paged_cache_write(odd, plain[1].transpose(0, 1).contiguous().transpose(0, 1), k2, v2, table, lengths, cu, **ex2)
    got = fused_ops.paged_cache_read(k2, v2, table, x.ints([0, 0]), x.ints([0, 8, 38]), 38, **ex2)
    assert all(same_bits(a, b) for a, b in zip(got, want))


def test_refusals():
    x = Batch([2], [5], 2, 1, 64, 64, 16, BF16, seed=1)
    k, v, table = x.pools()
    rows, lengths, cu = torch.zeros(2, 2, 64, dtype=BF16, device="cuda"), x.ints(x.lengths), x.ints(x.cu)
    codes, e = k.to(torch.float8_e4m3fn), torch.full(k.shape[:3], 127, dtype=torch.uint8, device="cuda")

    def write(a=rows, b=rows, k=k, v=v, table=table, lengths=lengths, cu=cu, **more):
        fused_ops.paged_cache_write(a, b, k, v, table, lengths, cu, **more)

    write()
    for bad in [dict(a=rows.cpu()), dict(a=rows.float()), dict(a=rows.half()), dict(a=rows[:1]), dict(a=rows[:, :1]), dict(a=rows[..., :32]),
                dict(a=rows[0]), dict(a=k[0, :2]), dict(k=codes, v=codes), dict(k=codes, v=codes, k_exponents=e, v_exponents=e, a=rows.half()),
                dict(lengths=lengths.long()), dict(cu=cu[:1]), dict(table=table.long()), dict(a=rows.clone().requires_grad_(True)),
                dict(k=k[:, :8], v=v[:, :8]), dict(k=k.cpu(), v=v.cpu())]:
        with pytest.raises(RuntimeError):
            write(**bad)

    def read(begins=lengths, cu=cu, rows=2, **more):
        return fused_ops.paged_cache_read(k, v, table, begins, cu, rows, **more)

    read()
    for bad in [dict(rows=-1), dict(dtype=torch.float32), dict(dtype=F16), dict(begins=lengths.cpu()), dict(begins=x.ints([1, 1])), dict(cu=x.ints([0])),
                dict(k_exponents=e)]:
        with pytest.raises(RuntimeError):
            read(**bad)
    assert read(rows=0, cu=x.ints([0, 0]))[0].shape == (0, 2, 64)
    before = k._version
    write()
    assert k._version > before
    for dtype in (torch.float32, torch.float8_e4m3fn):
        with pytest.raises(RuntimeError):
            PagedCache(1, 16, 1, 16, 16, dtype=dtype, device="cuda")


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_sequences_in_pieces(dtype, quantized):
    """Ragged prompts in pieces, then tokens one by one, chunks crossed on the way, pages taken as they are needed:
    each call's rows are the chunk attention of the whole sequences."""
    heads, dk, dv, chunk, page = 2, 64, 128, 48, 16
    attn = _InnerAttention(dk, dv, heads, chunk, 0.0, "fused").eval()
    cache = PagedCache(40, page, heads, dk, dv, dtype=dtype, quantized=quantized, device="cuda")
    pieces = [[30, 1, 0], [17, 40, 5], [1, 1, 1], [4, 0, 90], [1, 1, 1], [1, 1, 1]]
    total = [sum(p[b] for p in pieces) for b in range(3)]
    gen = torch.Generator().manual_seed(0)
    q, k, v = ([torch.randn(n, heads, w, generator=gen).to(dtype) for n in total] for w in (dk, dk, dv))
    q = [t * dk ** -0.5 for t in q]
    table = torch.full((3, 8), -1, dtype=torch.int32)
    free, done = list(range(40)), [0, 0, 0]
    for piece in pieces:
        for b in range(3):
            for i in range(-(-done[b] // page), -(-(done[b] + piece[b]) // page)):
                table[b, i] = free.pop(len(free) // 2)
        part = [[t[b][done[b]:done[b] + piece[b]] for b in range(3)] for t in (q, k, v)]
        xq, xk, xv = (torch.cat(t).flatten(1).cuda() for t in part)
        done = [d + n for d, n in zip(done, piece)]
        cu = torch.tensor([0, *torch.tensor(piece).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
        got = attn.forward_paged(xq, xk, xv, cache, table.cuda(), torch.tensor(done, dtype=torch.int32, device="cuda"), cu)
        at = 0
        for b in range(3):
            for i in range(piece[b]):
                p = done[b] - piece[b] + i
                low = p // chunk * chunk
                ks, vs = k[b][low:p + 1], v[b][low:p + 1]
                if quantized:
                    ks, vs = (c * powers(e)[..., None] for c, e in (to_8_bits(ks), to_8_bits(vs)))
                for h in range(heads):
                    w = torch.softmax(ks[:, h].double() @ q[b][p, h].double(), 0)
                    want, A = w @ vs[:, h].double(), w @ vs[:, h].double().abs()
                    # (as in paged.Batch.attention: the result's and the probabilities' rounding; what float32 adds is below 2^-16 A)
                    bound = 1.01 * UNIT[dtype] * (want.abs() + A) + 2.0 ** -16 * A + 2.0 ** -25 * (1 + vs[:, h].double().abs().sum(0))
                    off = (got[at, h * dv:(h + 1) * dv].double().cpu() - want).abs()
                    assert bool((off <= bound).all())
                at += 1
    back, _ = cache.read(table.cuda(), torch.zeros(3, dtype=torch.int32, device="cuda"),
                         torch.tensor([0, *torch.tensor(total).cumsum(0).tolist()], dtype=torch.int32, device="cuda"), sum(total))
    want = torch.cat(k)
    if quantized:
        codes, e = to_8_bits(want)
        want = (codes * powers(e)[..., None]).to(dtype)
    assert torch.equal(back.cpu(), want)


@pytest.mark.parametrize("bits", [16, 8])
def test_write_read_captured(bits):
    x = Batch([1, 1], [3, 30], 1, 1, 64, 64, 16, BF16, bits, seed=3)
    k, v, table = x.pools()
    ex = x.exponents()
    rows, lengths, cu = torch.zeros(2, 1, 64, dtype=BF16, device="cuda"), x.ints(x.lengths), x.ints(x.cu)
    begins = lengths - 1
    graph = torch.cuda.CUDAGraph()
    fused_ops.paged_cache_write(rows, rows, k, v, table, lengths, cu, **ex)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        fused_ops.paged_cache_write(rows, rows, k, v, table, lengths, cu, **ex)
        got = fused_ops.paged_cache_read(k, v, table, begins, cu, 2, **ex)
    for turn in range(5):
        rows.copy_(torch.randn(2, 1, 64))
        lengths.copy_(x.ints([turn + 1, 32 - turn]))
        begins.copy_(lengths - 1)
        graph.replay()
        want = rows.cpu()
        if bits == 8:
            codes, e = to_8_bits(want)
            want = (codes * powers(e)[..., None]).to(BF16)
        assert torch.equal(got[0].cpu(), want) and torch.equal(got[1].cpu(), want)
        torch.cuda.synchronize()
