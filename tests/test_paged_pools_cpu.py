"""Writing to the paged cache wants pools whose places do not share memory; which do is told by addresses and strides alone."""
import ctypes

import pytest
import torch

from megalodon_amd import _lib
from test_paged_cache_cpu import Cache, i64

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def answer(k, v, ke=None, ve=None):
    """The C entry's answer to a write of no rows: 0 or a refusal.  The tensors lend their addresses and strides."""
    fields = {"k_stride": k.stride()[:3], "v_stride": v.stride()[:3]}
    if ke is not None:
        fields.update(ke_stride=ke.stride(), ve_stride=ve.stride())
    c = Cache(k=k.data_ptr(), v=v.data_ptr(), pages=k.shape[0], page_size=k.shape[1], heads=k.shape[2], k_width=k.shape[3], v_width=v.shape[3],
              table=1 << 22, table_stride=4, table_width=4, batch=3, **{n: (i64 * 3)(*s) for n, s in fields.items()})
    if ke is not None:
        c.k_exponents, c.v_exponents = ke.data_ptr(), ve.data_ptr()
    fn = _lib.load().mega_paged_cache_write
    fn.restype = ctypes.c_int
    none = ctypes.c_void_p(None)
    code = fn(ctypes.byref(c), ctypes.c_int(1), none, i64(0), i64(0), none, i64(0), i64(0), none, none, i64(0), none)
    assert code == 0 or b"share memory" in _lib.load().mega_last_error()
    return code



def share(k, v):
    """Whether two tensors have a byte in common, byte by byte."""
    def bytes_of(t):
        at = torch.zeros((), dtype=torch.int64)
        for size, stride in zip(t.shape, t.stride()):
            at = at[..., None] + torch.arange(size) * stride
        at = at.flatten() * t.element_size() + t.data_ptr()
        return set((at[:, None] + torch.arange(t.element_size())).flatten().tolist())
    return bool(bytes_of(k) & bytes_of(v))


def layouts():
    P, S, H, A, B = 3, 16, 2, 32, 48
    row = torch.empty(P, S, H, A + B, dtype=BF16)
    yield "halves of a row", row[..., :A], row[..., A:]
    yield "halves of a row, values first", row[..., B:], row[..., :B]
    yield "a piece in common", row[..., :A], row[..., 16:16 + B]
    slot = torch.empty(P, S, H * (A + B), dtype=BF16)
    yield "halves of a position", slot[..., :H * A].unflatten(2, (H, A)), slot[..., H * A:].unflatten(2, (H, B))
    page = torch.empty(P, S * H * (A + B), dtype=BF16)
    yield "halves of a page", page[:, :S * H * A].view(P, S, H, A), page[:, S * H * A:].view(P, S, H, B)
    yield "heads outside, positions outside", page[:, :S * H * A].view(P, H, S, A).transpose(1, 2), page[:, S * H * A:].view(P, S, H, B)
    yield "pages that reach into the next half", page[:, :S * H * A].view(P, S, H, A), page[:, S * H * A - 16:-16].view(P, S, H, B)
    two = torch.empty(P, 2, S, H, A, dtype=BF16)
    yield "keys and values of a page in turn", two[:, 0], two[:, 1]
    yield "the same", two[:, 0], two[:, 0]
    inner = torch.empty(P, S, 2, H, A, dtype=BF16)
    yield "in turn for a position", inner[:, :, 0], inner[:, :, 1]
    heads = torch.empty(P, S, H, 2, A, dtype=BF16)
    yield "in turn for a head", heads[:, :, :, 0], heads[:, :, :, 1]
    many = torch.empty(P + 1, S, H, A, dtype=BF16)
    yield "a page further", many[:P], many[1:]
    flat = torch.empty(2 * P, S, H, A, dtype=BF16)
    yield "pages in turn", flat[::2], flat[1::2]
    yield "pages behind", flat[:P], flat[P:]
    one = torch.empty(P, S, 1, 2 * A, dtype=BF16)
    yield "one head", one[..., :A], one[..., A:]
    yield "apart", torch.empty(P, S, H, A, dtype=BF16), torch.empty(P, S, H, B, dtype=BF16)


@pytest.mark.parametrize("name,k,v", list(layouts()), ids=lambda x: x if isinstance(x, str) else "")
def test_layouts(name, k, v):
    assert answer(k, v) == answer(v, k) == int(share(k, v))


def test_rows_of_a_pool_that_share_memory():
    flat, v = torch.empty(4096, dtype=BF16), torch.empty(3, 16, 2, 32, dtype=BF16)
    for stride, meets in (((1024, 64, 32, 1), False), ((1024, 32, 512, 1), False), ((512, 64, 32, 1), True), ((1024, 48, 32, 1), True), ((1024, 64, 16, 1), True)):
        k = flat.as_strided((3, 16, 2, 32), stride)
        assert answer(k, v) == int(meets) and answer(v, k) == int(meets)


def test_exponents():
    k, v = (torch.empty(3, 16, 2, w, dtype=E4M3) for w in (32, 48))
    both = torch.empty(3, 16, 2, 2, dtype=torch.uint8)
    assert answer(k, v, both[..., 0], both[..., 1]) == 0
    assert answer(k, v, both[..., 0], both[..., 0]) == 1
    # exponents behind the codes of a row, and on them
    rows = torch.empty(3, 16, 2, 48, dtype=torch.uint8)
    assert answer(rows[..., :32].view(E4M3), v, rows[..., 32], both[..., 1]) == 0
    assert answer(rows[..., :32].view(E4M3), v, rows[..., 31], both[..., 1]) == 1


def test_random_layouts_are_never_taken_for_apart():
    """Pools cut at random out of one tensor of nested axes: where memory is shared the call is refused; equal strides leave nothing open."""
    gen = torch.Generator().manual_seed(0)

    def pick(n):
        return int(torch.randint(n, (), generator=gen))
    met = apart = 0
    for _ in range(400):
        whole = torch.empty(6, 20, 4, 96, dtype=BF16)
        cuts = []
        for _ in range(2):
            at = [pick(4), pick(5), pick(3), 16 * pick(5)]
            step = 1 + pick(2)
            cuts.append(whole[at[0]:at[0] + 3:step][:2, at[1]:at[1] + 16, at[2]:at[2] + 2, at[3]:at[3] + 16])
        k, v = cuts
        if k.shape[:3] != v.shape[:3] or k.shape[1:3] != (16, 2):
            continue
        meets = share(k, v)
        met, apart = met + meets, apart + (not meets)
        assert answer(k, v) >= int(meets)
        if k.stride() == v.stride():
            assert answer(k, v) == int(meets)
    assert met > 20 and apart > 20
