"""The paged key / value cache and the attention that reads it, as cases to be timed.

Sequences of different lengths share one pool of pages.  A page holds ``page`` consecutive
positions of one sequence: keys (pages, page, heads, qk_width) and values (pages, page, heads,
v_width), in 16 bits or as e4m3 numbers with one power of two for each position and head.
``table[b]`` names the pages of sequence b in their order, ``lengths[b]`` how many positions it
has, the new ones included, and rows ``cu[b] .. cu[b + 1]`` of the packed operands are its new
tokens.  Four kinds:

* ``write``  new keys and values go to their places in the pool (16 bits);
* ``store8``  the same into an 8-bit pool, and back from it;
* ``read``  stored positions of many sequences into contiguous rows;
* ``attend``  every new token attends over the stored positions of its sequence: from the start of
  its own chunk of ``chunk`` positions (0: from the first) to itself.  ``shared`` query heads read one
  key / value head.

Heads are those of the block of BASELINE's configuration 4 (256 query / key and 2048 value features)
or generic ones of 128 and 64; lengths are inside or across its chunks of 4096, or generic.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    mega = {"heads": 4, "shared": 1, "qk_width": 256, "v_width": 2048, "page": 64, "chunk": 4096}
    lean = {"heads": 8, "shared": 4, "qk_width": 128, "v_width": 128, "chunk": 0}
    return [
        # Serving, every step: one token each of sixteen sequences enters the cache.
        {"name": "write_step", "kind": "write", "dtype": "bf16", "batch": 16,
         "new_low": 1, "new_high": 1, "old_low": 90, "old_high": 390, **mega},
        # Serving with drafts: a few tokens each enter an 8-bit cache and are looked at again.
        {"name": "store8_drafts", "kind": "store8", "dtype": "f16", "batch": 16,
         "new_low": 2, "new_high": 7, "old_low": 0, "old_high": 301, **mega},
        # A prompt of a whole chunk enters an 8-bit cache, its stored form is handed on.
        {"name": "store8_prompt", "kind": "store8", "dtype": "bf16", "batch": 1,
         "new_low": 4096, "new_high": 4096, "old_low": 0, "old_high": 0, **mega},
        # The open chunks of sixteen sequences leave an 8-bit cache for contiguous 16-bit rows.
        {"name": "read_chunks", "kind": "read", "dtype": "bf16", "bits": 8, "batch": 16,
         "new_low": 1, "new_high": 3999, "old_low": 0, "old_high": 97, **mega},
        # Two sequences move out of a 16-bit cache: the smallest transfer.
        {"name": "read_pair", "kind": "read", "dtype": "f16", "bits": 16, "batch": 2,
         "new_low": 33, "new_high": 61, "old_low": 100, "old_high": 100,
         **{**mega, "heads": 1}},
        # Interactive generation: one sequence, one token, behind a prompt of ordinary, odd length.
        {"name": "attend_token", "kind": "attend", "dtype": "bf16", "bits": 16, "batch": 1,
         "new_low": 1, "new_high": 1, "old_low": 1531, "old_high": 1531, **mega},
        # Serving: sixteen sequences of different lengths, one token each, 8-bit cache.
        {"name": "attend_step8", "kind": "attend", "dtype": "bf16", "bits": 8, "batch": 16,
         "new_low": 1, "new_high": 1, "old_low": 1000, "old_high": 4000, **mega},
        # Drafted tokens of eight sequences looked at in one call.
        {"name": "attend_drafts", "kind": "attend", "dtype": "f16", "bits": 16, "batch": 8,
         "new_low": 3, "new_high": 7, "old_low": 777, "old_high": 3500, **mega},
        # A long prompt arrives in pieces of 512 tokens: one of the later pieces.
        {"name": "attend_piece", "kind": "attend", "dtype": "bf16", "bits": 16, "batch": 1,
         "new_low": 512, "new_high": 512, "old_low": 1531, "old_high": 1531, **mega},
        # A prompt of two whole chunks at once: the largest call.
        {"name": "attend_prompt", "kind": "attend", "dtype": "bf16", "bits": 16, "batch": 1,
         "new_low": 8192, "new_high": 8192, "old_low": 0, "old_high": 0, **mega},
        # Long contexts of thirty-two sequences on shared heads, one token each, small pages.
        {"name": "attend_long", "kind": "attend", "dtype": "bf16", "bits": 16, "batch": 32,
         "new_low": 1, "new_high": 1, "old_low": 500, "old_high": 16000,
         "page": 16, **lean},
        # Pieces of four prompts of different lengths on shared heads, 8-bit cache.
        {"name": "attend_pieces8", "kind": "attend", "dtype": "f16", "bits": 8, "batch": 4,
         "new_low": 255, "new_high": 1023, "old_low": 0, "old_high": 7001,
         "page": 128, **lean},
    ]


def _spread(rng, low, high):
    """A whole number of low .. high, even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["write", "store8", "read", "attend", "attend", "attend"])
    case = {"kind": kind, "dtype": rng.choice(["bf16", "f16"]), "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "read" or kind == "attend":
        case["bits"] = rng.choice([8, 16])
    if rng.random() < 0.6:  # the block's heads
        case.update(heads=rng.choice([1, 2, 4]), shared=1, qk_width=256, v_width=2048, chunk=rng.choice([1024, 2048, 4096]))
        reach = case["chunk"]
    else:
        width = rng.choice([64, 128])
        case.update(heads=_spread(rng, 1, 8), shared=rng.choice([1, 2, 4, 8]), qk_width=width, v_width=rng.choice([width, 2 * width]),
                    chunk=rng.choice([0, 0, 2048]))
        reach = 8192
    if kind == "attend" and rng.random() < 0.5:  # single tokens and drafts
        case["batch"] = _spread(rng, 1, 32)
        top = rng.choice([1, 1, 9])
    else:
        case["batch"] = _spread(rng, 1, 8)
        top = _spread(rng, 1, 4096 // case["batch"])
    case["new_low"], case["new_high"] = _spread(rng, 1, top), top
    old = _spread(rng, 1, 512 if kind in ("write", "store8") else reach)
    case["old_low"], case["old_high"] = rng.randint(0, old), old
    while True:  # no dearer than the listed ones
        cost = work(case)
        if cost["flops"] <= 3e11 and cost["bytes"] <= 8e8:
            return case
        which = "new" if cost["flops"] > 3e11 or case["new_high"] >= case["old_high"] else "old"
        for end in ("_low", "_high"):
            case[which + end] = max(1, case[which + end] // 2)


def _sequences(case):
    """New and old tokens of every sequence: even over the case's ranges, in an order of no meaning."""
    n, mixed = case["batch"], random.Random(case["batch"])
    new, old = (([low + (high - low) * b // max(1, n - 1) for b in range(n)]) 
                for low, high in ((case[what + "_low"], case[what + "_high"]) for what in ("new", "old")))
    mixed.shuffle(new)
    mixed.shuffle(old)
    return new, old


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, page, heads = DTYPES[case["dtype"]], case["page"], case["heads"]
    new, old = _sequences(case)
    lengths = [a + b for a, b in zip(new, old)]
    per_sequence = [-(-length // page) for length in lengths]
    pages = sum(per_sequence) + 3  # (some pages of the pool are nobody's)
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    table = torch.full((len(new), max(per_sequence)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, count in enumerate(per_sequence):
        table[b, :count] = order[at:at + count]
        at += count
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    state = {"case": case, "dtype": dtype, "table": table, "lengths": ints(lengths), "cu": ints(cu), "host": (new, old, cu),
             "rows": cu[-1], "begins": ints(old)}
    bits = {"write": 16, "store8": 8}.get(case["kind"], case.get("bits"))
    for what, width in (("k", case["qk_width"]), ("v", case["v_width"])):
        values = _normal(gen, pages, page, heads, width).to(dtype)
        if what == "v":
            values = torch.nn.functional.silu(values)  # (as the block makes them)
        state[what + "_exp"] = None
        if bits == 8:
            values, state[what + "_exp"] = _to_8_bits(values)
        state[what + "_pages"] = values
        if case["kind"] in ("write", "store8"):
            rows = _normal(gen, cu[-1], heads, width)
            # magnitudes differ from token to token, as they do behind a projection
            rows *= torch.exp2(torch.randint(-3, 4, (cu[-1], heads, 1), device="cuda", generator=gen).float())
            state[what] = rows.to(dtype)
    if case["kind"] == "attend":
        state["q"] = (1.5 * _normal(gen, cu[-1], heads * case["shared"], case["qk_width"])).to(dtype)
        state["scale"] = case["qk_width"] ** -0.5
    return state


# ---- plain forms ------------------------------------------------------------------------------

def _power(biased):
    """2 ^ (biased - 127), exact: the number's own exponent field."""
    return (biased.int() << 23).view(torch.float32)


def _to_8_bits(x):
    """(codes, exponents): each row over the last axis as e4m3 numbers times 2 ^ (exponent - 127), the
    smallest power that keeps the row's largest magnitude at or below 448."""
    top = x.abs().amax(-1).float()
    fraction, power = torch.frexp(top)
    exponent = torch.where(fraction > 0.875, power - 8, power - 9).clamp(-126, 120)
    exponent = torch.where(top > 0, exponent, torch.zeros_like(exponent))
    codes = (x.float() * _power(127 - exponent)[..., None]).to(torch.float8_e4m3fn)
    return codes, (exponent + 127).to(torch.uint8)


def _places(state, b, first, last):
    """Where positions first .. last - 1 of sequence b are: their pages and their places inside them."""
    page = state["case"]["page"]
    position = torch.arange(first, last, device="cuda")
    return state["table"][b].long()[position // page], position % page


def _stored(state, what, b, first, last):
    """Stored rows of sequence b in float32."""
    where = _places(state, b, first, last)
    rows = state[what + "_pages"][where].float()
    if state[what + "_exp"] is not None:
        rows = rows * _power(state[what + "_exp"][where])[..., None]
    return rows


def _write(state):
    new, old, cu = state["host"]
    for what in ("k", "v"):
        rows, exponents = state[what], None
        if state[what + "_exp"] is not None:
            rows, exponents = _to_8_bits(rows)
        for b in range(len(new)):
            where = _places(state, b, old[b], old[b] + new[b])
            state[what + "_pages"][where] = rows[cu[b]:cu[b + 1]]
            if exponents is not None:
                state[what + "_exp"][where] = exponents[cu[b]:cu[b + 1]]


def _read(state):
    new, old, cu = state["host"]
    return tuple(torch.cat([_stored(state, what, b, old[b], old[b] + new[b]) for b in range(len(new))]).to(state["dtype"])
                 for what in ("k", "v"))


def _chunk_start(position, chunk):
    return position // chunk * chunk if chunk else position * 0


def _attend(state):
    case = state["case"]
    new, old, cu = state["host"]
    heads, shared, chunk = case["heads"], case["shared"], case["chunk"]
    outs = []
    for b in range(len(new)):
        for at in range(0, new[b], 2048):  # (rows at a time, for the scores' size)
            n = min(2048, new[b] - at)
            row = torch.arange(old[b] + at, old[b] + at + n, device="cuda")
            first = int(_chunk_start(old[b] + at, chunk))
            key = torch.arange(first, old[b] + at + n, device="cuda")
            k = _stored(state, "k", b, first, old[b] + at + n).permute(1, 2, 0)   # (heads, width, keys)
            v = _stored(state, "v", b, first, old[b] + at + n).transpose(0, 1)    # (heads, keys, width)
            q = state["q"][cu[b] + at:cu[b] + at + n].float().view(n, heads, shared, -1).permute(1, 0, 2, 3).reshape(heads, n * shared, -1)
            seen = (key <= row[:, None]) & (key >= _chunk_start(row, chunk)[:, None])
            s = torch.matmul(q, k.contiguous()) * state["scale"]
            s = s.view(heads, n, shared, -1).masked_fill(~seen[None, :, None], float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p = (p / p.sum(-1, keepdim=True)).view(heads, n * shared, -1)
            out = torch.matmul(p, v.contiguous()).view(heads, n, shared, -1)
            outs.append(out.permute(1, 0, 2, 3).reshape(n, heads * shared, -1).to(state["dtype"]))
    return torch.cat(outs)


# ---- one pass -----------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        from megalodon_amd import fused_ops
        pool = (state["k_pages"], state["v_pages"], state["table"])
        exps = {"k_exponents": state["k_exp"], "v_exponents": state["v_exp"]}
        if kind == "attend":
            return fused_ops.paged_attention(state["q"], *pool, state["lengths"], state["cu"], scale=state["scale"],
                                             chunk_size=state["case"]["chunk"], **exps)
        if kind != "read":
            fused_ops.paged_cache_write(state["k"], state["v"], *pool, state["lengths"], state["cu"], **exps)
            if kind == "write":
                return state["k_pages"], state["v_pages"]
        return fused_ops.paged_cache_read(*pool, state["begins"], state["cu"], state["rows"], dtype=state["dtype"], **exps)
    if kind == "attend":
        return _attend(state)
    if kind != "read":
        _write(state)
        if kind == "write":
            return state["k_pages"], state["v_pages"]
    return _read(state)


def work(case):
    new, old = _sequences(case)
    heads, wide = case["heads"], case["qk_width"] + case["v_width"]
    rows = sum(new)
    row16, row8 = 2 * wide * heads, (wide + 2) * heads
    meta = 4 * (3 * case["batch"] + sum(-(-(a + b) // case["page"]) for a, b in zip(new, old)))
    if case["kind"] == "write":
        return {"bytes": 2 * rows * row16 + meta, "flops": 0}
    if case["kind"] == "store8":  # in, codes out; codes in, rows out
        return {"bytes": 2 * rows * (row16 + row8) + meta, "flops": 4 * rows * wide * heads}
    stored = row8 if case["bits"] == 8 else row16
    if case["kind"] == "read":
        return {"bytes": rows * (stored + row16) + meta, "flops": (2 * rows * wide * heads if case["bits"] == 8 else 0)}
    keys = pairs = 0
    for n, o in zip(new, old):
        keys += o + n - _chunk_start(o, case["chunk"])
        pairs += sum(p + 1 - _chunk_start(p, case["chunk"]) for p in range(o, o + n))
    return {"bytes": keys * stored + rows * heads * case["shared"] * wide * 2 + meta, "flops": 2 * pairs * heads * case["shared"] * wide}


# ---- the definition in 64 bits, sequence by sequence and head by head --------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    new, old = _sequences(case)
    page, table = case["page"], state["table"].tolist()

    def two_to(n):  # (a power function need not be exact, and a tie would fall to the wrong side)
        return (n + 1023 << 52).view(torch.float64)

    def slots(b, first, last):
        return [table[b][p // page] * page + p % page for p in range(first, last)]

    def values(what, index, head=slice(None)):
        rows = state[what + "_pages"].flatten(0, 1)[:, head][index].double()
        if state[what + "_exp"] is None:
            return rows
        return rows * two_to(state[what + "_exp"].flatten(0, 1)[:, head][index].long() - 127)[..., None]

    def eight(x):
        """x as the nearest e4m3 numbers (ties to even) times the row's power of two."""
        x = x.double()
        top = x.abs().amax(-1, keepdim=True)
        n = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0)).long()
        n += (top > 448.0 * two_to(n)).long() - (top <= 224.0 * two_to(n)).long()  # (where the logarithm is off by a digit)
        unit = two_to(n)
        y = x / unit
        step = two_to(torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent.long() - 4)
        return torch.round(y / step) * step * unit

    if case["kind"] == "write":
        where = torch.tensor([s for b in range(len(new)) for s in slots(b, old[b], old[b] + new[b])], device="cuda")
        out = []
        for what in ("k", "v"):
            pool = state[what + "_pages"].double()
            pool.flatten(0, 1)[where] = state[what].double()
            out.append(pool)
        return tuple(out)
    if case["kind"] == "store8":
        return tuple(eight(state[what]) for what in ("k", "v"))
    if case["kind"] == "read":
        index = torch.tensor([s for b in range(len(new)) for s in slots(b, old[b], old[b] + new[b])], device="cuda")
        return tuple(values(what, index) for what in ("k", "v"))

    out = torch.zeros(sum(new), case["heads"] * case["shared"], case["v_width"], dtype=torch.float64, device="cuda")
    at, span = 0, case["chunk"] or 10 ** 9
    for b in range(len(new)):
        index = torch.tensor(slots(b, 0, old[b] + new[b]), device="cuda")
        for first in range(0, new[b], 1024):
            last = min(new[b], first + 1024)
            low, high = (old[b] + first) // span * span, old[b] + last
            row = torch.arange(old[b] + first, high, device="cuda")[:, None]
            key = torch.arange(low, high, device="cuda")[None, :]
            hidden = (key > row) | (torch.div(key, span, rounding_mode="floor") != torch.div(row, span, rounding_mode="floor"))
            for h in range(case["heads"]):
                kt, v = values("k", index[low:high], h).t().contiguous(), values("v", index[low:high], h)
                for g in range(case["shared"]):
                    qh = h * case["shared"] + g
                    s = state["q"][at + first:at + last, qh].double() @ kt * state["scale"]
                    s[hidden] = -math.inf
                    out[at + first:at + last, qh] = torch.softmax(s, -1) @ v
        at += new[b]
    return out
