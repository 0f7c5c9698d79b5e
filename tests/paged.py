"""Ragged batches on a paged cache, and the operators' definitions in 64 bits, sequence by sequence."""
import math
import random

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative
SMALL = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half a step below the normal numbers


def powers(e):
    """2 ** (e - 127), exact."""
    return torch.ldexp(torch.ones((), dtype=torch.float64), e.to(torch.int64).cpu() - 127)


def to_8_bits(x):
    """(codes as float64 numbers, exponents): the definition, number by number."""
    top_of_type = {torch.bfloat16: 120, torch.float16: 8}[x.dtype]
    x = x.double()
    finite = torch.isfinite(x)
    top = torch.where(finite, x.abs(), 0.0).amax(-1)
    e = torch.zeros(top.shape, dtype=torch.int64)
    flat = e.view(-1)
    for i, t in enumerate(top.reshape(-1).tolist()):
        if t > 0:
            n = -126
            while t > 448.0 * 2.0 ** n:
                n += 1
            flat[i] = n
    y = x * torch.ldexp(torch.ones((), dtype=torch.float64), -e)[..., None]
    step = 2.0 ** (torch.floor(torch.log2(y.abs().nan_to_num(1.0, 1.0).clamp(min=2.0 ** -6))) - 3)
    codes = torch.round(y / step) * step  # (half to even)
    codes = torch.where((e == top_of_type)[..., None], codes.clamp(-240, 240), codes)
    return torch.where(finite, codes, math.nan), (e + 127).to(torch.uint8)


class Batch:
    """News and olds: new and old positions of each sequence.  Everything that no sequence owns is NaN."""

    def __init__(self, news, olds, heads, shared, dk, dv, page, dtype, bits=16, seed=0, spare=2, extra_rows=0, device="cuda"):
        gen = torch.Generator().manual_seed(seed)
        self.news, self.olds, self.heads, self.shared, self.page, self.dtype, self.bits = news, olds, heads, shared, page, dtype, bits
        n = len(news)
        self.lengths = [a + b for a, b in zip(news, olds)]
        counts = [-(-length // page) for length in self.lengths]
        pages = sum(counts) + spare
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        self.table = torch.full((n, max(counts + [1]) + 1), -1, dtype=torch.int32)
        for b, c in enumerate(counts):
            for i in range(c):
                self.table[b, i] = order.pop()
        self.cu = [0]
        for a in news:
            self.cu.append(self.cu[-1] + a)
        self.rows = self.cu[-1] + extra_rows
        self.k, self.v = (torch.randn(pages, page, heads, w, generator=gen).to(dtype) for w in (dk, dv))
        self.q = torch.randn(self.rows, heads * shared, dk, generator=gen).to(dtype)
        owned = torch.zeros(pages, page, dtype=torch.bool)
        for b in range(n):
            for p in range(self.lengths[b]):
                owned[self.table[b, p // page], p % page] = True
        self.k[~owned], self.v[~owned] = math.nan, math.nan
        self.ke = self.ve = None
        if bits == 8:
            self.k, self.ke = (t.to(torch.float8_e4m3fn) if i == 0 else t for i, t in enumerate(to_8_bits(self.k)))
            self.v, self.ve = (t.to(torch.float8_e4m3fn) if i == 0 else t for i, t in enumerate(to_8_bits(self.v)))
        self.device = device

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def pools(self):
        return self.k.to(self.device), self.v.to(self.device), self.table.to(self.device)

    def exponents(self):
        return {} if self.bits == 16 else {"k_exponents": self.ke.to(self.device), "v_exponents": self.ve.to(self.device)}

    def stored(self, b, first, last):
        """Keys and values of positions first .. last - 1 of sequence b in float64."""
        out = []
        for pool, e in ((self.k, self.ke), (self.v, self.ve)):
            page = torch.tensor([int(self.table[b, p // self.page]) for p in range(first, last)], dtype=torch.long)
            slot = torch.tensor([p % self.page for p in range(first, last)], dtype=torch.long)
            x = pool.float().double()[page, slot] if pool.dtype == torch.float8_e4m3fn else pool.double()[page, slot]
            out.append(x if e is None else x * powers(e[page, slot])[..., None])
        return out

    def attention(self, scale, chunk, heads=None):
        """(out, bound) of the query heads in `heads` (None: all): float64, and what 16-bit probabilities and results and 32-bit arithmetic may be off by.

        With u half a step of the type, A = sum_j p_j |v_j|, N keys of width W: rounding the result costs u |o|, rounding
        the probabilities u A (below float16's normal numbers 2^-25 sum |v| instead), the float32 sums (N + 8) 2^-23 A.
        A score is off by at most d = (W + 4) 2^-23 scale sum |q k| (products, their sum, the factor scale log2 e) and
        its power by 2^-21 of itself, which moves p by a factor within 1 +- (2 d + 2^-20): (2 d + 2^-20) A."""
        u, small = UNIT[self.dtype], SMALL[self.dtype]
        dv = self.v.shape[3]
        out = torch.zeros(self.rows, self.heads * self.shared, dv, dtype=torch.float64)
        bound = torch.zeros_like(out)
        for b, n in enumerate(self.news):
            if n == 0:
                continue
            k, v = self.stored(b, 0, self.lengths[b])
            for t in range(n):
                p = self.olds[b] + t
                low = p // chunk * chunk if chunk else 0
                for g in heads or range(self.heads * self.shared):
                    kh, vh, q = k[low:p + 1, g // self.shared], v[low:p + 1, g // self.shared], self.q[self.cu[b] + t, g].double()
                    w = torch.softmax(kh @ q * scale, 0)
                    o, A = w @ vh, w @ vh.abs()
                    d = (len(q) + 4) * 2.0 ** -23 * abs(scale) * (kh.abs() @ q.abs()).max()
                    out[self.cu[b] + t, g] = o
                    bound[self.cu[b] + t, g] = 1.01 * u * (o.abs() + A) + (2 * d + 2.0 ** -20 + (p + 1 - low + 8) * 2.0 ** -23) * A + small * (1 + vh.abs().sum(0))
        return out, bound
