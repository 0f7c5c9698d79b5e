"""Paged attention over 8-bit rows whose numbers the call's type does not hold, and behind exponents that nobody wrote."""
import math

import pytest
import torch

from megalodon_amd import fused_ops
from paged import SMALL, UNIT, Batch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def attend(x, scale, chunk):
    return fused_ops.paged_attention(x.q.cuda(), *x.pools(), x.ints(x.lengths), x.ints(x.cu), scale, chunk, **x.exponents()).cpu()


def definition(x, scale, chunk):
    """As Batch.attention, over the stored numbers rounded to the rows' type (infinite where that does not hold them)."""
    out = torch.zeros(x.rows, x.heads * x.shared, x.v.shape[3], dtype=torch.float64)
    bound = torch.zeros_like(out)
    u, small = UNIT[x.dtype], SMALL[x.dtype]
    for b, n in enumerate(x.news):
        k, v = (t.to(x.dtype).double() for t in x.stored(b, 0, x.lengths[b]))
        for t in range(n):
            p = x.olds[b] + t
            low = p // chunk * chunk if chunk else 0
            for g in range(x.heads * x.shared):
                kh, vh, q = k[low:p + 1, g // x.shared], v[low:p + 1, g // x.shared], x.q[x.cu[b] + t, g].double()
                w = torch.softmax((kh * q).sum(-1) * scale, 0)
                o, A = (w[:, None] * vh).sum(0), (w[:, None] * vh.abs()).sum(0)
                sizes = (kh.abs() * q.abs()).sum(-1)
                d = (len(q) + 4) * 2.0 ** -23 * scale * sizes[sizes < math.inf].max()
                out[x.cu[b] + t, g] = o
                bound[x.cu[b] + t, g] = 1.01 * u * (o.abs() + A) + (2 * d + 2.0 ** -20 + (p + 9 - low) * 2.0 ** -23) * A + small * (1 + vh.abs().sum(0))
    return out, bound


def check(got, want, bound):
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), finite)
    assert torch.equal(got[~finite].double().nan_to_num(nan=7.0), want[~finite].nan_to_num(nan=7.0))  # (infinities of their sign)
    assert bool(((got.double() - want)[finite].abs() <= bound[finite]).all())


def place(x, position):
    return int(x.table[0, position // x.page]), position % x.page


# few rows of a sequence and many; the position in keys that all rows see (whole groups of 32, or the last few), that later rows see, of
# the chunk before
WHERE = [([1], [40], 10, 0), ([1], [40], 35, 0), ([1], [40], 40, 0), ([5], [300], 5, 0), ([5], [300], 299, 0), ([5], [300], 302, 0), ([5], [62], 63, 64),
         ([100], [20], 5, 0), ([100], [20], 70, 0), ([100], [20], 63, 64), ([80, 40], [300, 7], 340, 0)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dv", [64, 1040])
@pytest.mark.parametrize("where", WHERE, ids=lambda w: f"{w[0][0]}-{w[1][0]}-{w[2]}-{w[3]}")
def test_values_past_the_type_are_infinite_to_the_rows_that_see_them(where, dv, dtype):
    """A stored value of 448 2^9 (2^127) is an infinity in float16 (bfloat16), as it is where the cache is read; small codes beside
    it are numbers."""
    news, olds, bad, chunk = where
    x = Batch(news, olds, 1, 1, 64, dv, 16, dtype, 8, seed=21)
    clean = attend(x, 0.1, chunk)
    codes = torch.full((dv,), 2.0 ** -6)
    codes[1::3], codes[2::7] = 448.0, -448.0
    x.v[place(x, bad)] = codes.to(x.v.dtype)
    x.ve[place(x, bad)] = 136 if dtype == F16 else 254
    want, bound = definition(x, 0.1, chunk)
    got = attend(x, 0.1, chunk)
    check(got, want, bound)
    position = torch.tensor([o + i for n, o in zip(news, olds) for i in range(n)])
    blind = (position < bad) | (position // (chunk or 10 ** 9) != bad // (chunk or 10 ** 9))
    blind[news[0]:] = True  # (other sequences)
    assert torch.equal(got[blind], clean[blind]) and not bool(torch.isfinite(got[~blind]).all(-1).any())


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("where", WHERE, ids=lambda w: f"{w[0][0]}-{w[1][0]}-{w[2]}-{w[3]}")
def test_keys_past_the_type_are_infinite(where, sign):
    """A score of infinity makes a row NaN, one of minus infinity takes the key out, in few rows as in many."""
    news, olds, bad, chunk = where
    x = Batch(news, olds, 1, 1, 64, 64, 16, F16, 8, seed=22)
    x.q[..., 0] = sign
    codes = torch.zeros(64)
    codes[0] = 448.0
    x.k[place(x, bad)] = codes.to(x.k.dtype)
    x.ke[place(x, bad)] = 136
    want, bound = definition(x, 0.1, chunk)
    check(attend(x, 0.1, chunk), want, bound)


@pytest.mark.parametrize("dv", [64, 1040])
@pytest.mark.parametrize("byte", [255, 254, 0])
@pytest.mark.parametrize("news,olds", [([1], [40]), ([5, 1], [300, 7]), ([100], [20]), ([80, 40], [300, 7])])
def test_exponents_that_nobody_wrote_do_not_matter(news, olds, byte, dv):
    """Behind a sequence's end, on pages of nobody, and on the page whose numbers stand in for those of a number that is no page."""
    for dtype in (BF16, F16):
        x = Batch(news, olds, 1, 1, 64, dv, 16, dtype, 8, seed=23)
        pages = x.k.shape[0]
        spare = next(i for i in range(pages) if i not in x.table.flatten().tolist())
        turn = [(i + spare) % pages for i in range(pages)]  # the spare page is number 0
        x.k, x.v, x.ke, x.ve = x.k[turn], x.v[turn], x.ke[turn], x.ve[turn]
        x.table = torch.where(x.table >= 0, (x.table - spare) % pages, x.table)
        x.table[0, 1] = -1
        clean = attend(x, 0.2, 0)
        owned = torch.zeros(x.ke.shape, dtype=torch.bool)
        for b, length in enumerate(x.lengths):
            for p in range(length):
                if x.table[b, p // 16] >= 0:
                    owned[x.table[b, p // 16], p % 16] = True
        x.ke[~owned], x.ve[~owned] = byte, byte
        assert bool(torch.isfinite(clean).all()) and torch.equal(attend(x, 0.2, 0), clean)


@pytest.mark.parametrize("dv", [64, 1040])
@pytest.mark.parametrize("news,olds", [([6], [300]), ([100], [20])])
def test_an_exponent_that_is_none_stays_with_the_rows_that_see_it(news, olds, dv):
    """Byte 255 stands for no number; the rows in front of it are as without."""
    x = Batch(news, olds, 1, 1, 64, dv, 16, BF16, 8, seed=24)
    clean = attend(x, 0.2, 0)
    bad = olds[0] + news[0] // 2
    x.ve[place(x, bad)] = 255
    assert torch.equal(attend(x, 0.2, 0)[:news[0] // 2], clean[:news[0] // 2])
