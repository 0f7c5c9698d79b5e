"""What the embedding, the gated product and clipping write, and what they do not: outputs and workspaces are pieces of larger buffers, at odd elements where that
is allowed, whose other elements have to stay as they were.  The values are those of the Python entry points, bit for bit (they run the same kernels)."""
import pytest
import torch

from megalodon_amd import _lib, fused_ops

pytestmark = pytest.mark.gpu

MARK, GUARD = 0x5a, 4096  # bytes


class Piece:
    """`shape` elements at `at` bytes behind a guard of marked bytes, marked themselves."""

    def __init__(self, shape, dtype, at=0):
        size = torch.Size(shape).numel() * torch.empty((), dtype=dtype).element_size()
        self.bytes = torch.full((GUARD + at + size + GUARD,), MARK, dtype=torch.uint8, device="cuda")
        self.front, self.behind = GUARD + at, GUARD + at + size
        self.tensor = self.bytes[self.front:self.behind].view(dtype).view(shape) if at % 8 == 0 else None
        self.shape, self.dtype = shape, dtype
        self.pointer = _lib.ctypes.c_void_p(self.bytes.data_ptr() + self.front)

    def value(self):
        return self.bytes[self.front:self.behind].clone().view(self.dtype).view(self.shape)

    def kept(self):
        return bool((self.bytes[:self.front] == MARK).all()) and bool((self.bytes[self.behind:] == MARK).all())


def size_of(name, *args):
    fn = getattr(_lib.load(), name)
    fn.restype = _lib.ctypes.c_int64
    return fn(*args)


def same(a, b):
    return torch.equal(a.reshape(-1).view(torch.int32 if a.element_size() == 4 else torch.int16), b.contiguous().reshape(-1).view(torch.int32 if b.element_size() == 4 else torch.int16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (3, 17, 1), (5, 33, 3), (40, 100, 7), (64, 50, 8), (65, 200, 129), (700, 90, 1001), (3, 1000, 24), (9000, 31, 9), (9000, 3000, 260), (300, 40, 2049)])
@pytest.mark.parametrize("at", [0, 1])
def test_embedding(n, V, D, dtype, at):
    lib, size = _lib, torch.empty((), dtype=dtype).element_size()
    g = torch.Generator("cuda").manual_seed(n + V + D)
    table = torch.randn(V, D, generator=g, device="cuda").to(dtype)
    tokens = torch.randint(-1, V + 1, (n,), generator=g, device="cuda")
    dy = torch.randn(n, D, generator=g, device="cuda").to(dtype)
    leaf = table.clone().requires_grad_(True)
    y = fused_ops.embedding(tokens, leaf, 2.0, 0)
    dw, = torch.autograd.grad(y, leaf, dy)
    code, sizes, none = lib.i32(lib.dtype_code(dtype)), (lib.i64(n), lib.i64(V), lib.i64(D)), lib.stream_ptr()
    out, to = Piece((n, D), dtype, at * size), Piece((V, D), dtype, at * size)
    ws = Piece((size_of("mega_embedding_workspace_bytes", code, *sizes),), torch.uint8)
    lib.call("mega_embedding_fwd", lib.ptr(tokens), lib.i32(64), lib.ptr(table), code, *sizes, lib.i64(D), lib.f64(2), out.pointer, none)
    lib.call("mega_embedding_bwd", lib.ptr(dy), code, lib.ptr(tokens), lib.i32(64), *sizes, lib.f64(2), lib.i64(0), to.pointer, ws.pointer, none)
    assert out.kept() and to.kept() and ws.kept()
    assert same(out.value(), y.detach()) and same(to.value(), dw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("tokens,n_in,n_out", [
    (1, 1, 1), (3, 7, 5), (1, 64, 17), (8, 1024, 33), (13, 1032, 9), (16, 2048, 100), (16, 3000, 31), (17, 24, 8), (33, 1001, 63), (64, 520, 192),
    (65, 64, 8), (65, 1, 1), (129, 1001, 63), (200, 128, 130), (257, 1000, 300), (300, 1024, 333), (700, 24, 9000), (2100, 264, 72), (1300, 2048, 1409),
])
@pytest.mark.parametrize("at", [0, 1])
def test_gated_linear(tokens, n_in, n_out, wide, dtype, at):
    lib = _lib
    g = torch.Generator("cuda").manual_seed(tokens + n_in + n_out)
    rows = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w1, w3, dh = rows(tokens, n_in).to(dtype), (rows(n_out, n_in) / n_in ** 0.5).to(dtype), (rows(n_out, n_in) / n_in ** 0.5).to(dtype), rows(tokens, n_out).to(dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
    h = fused_ops.gated_linear(*leaves, None if wide else dtype)
    want = torch.autograd.grad(h, leaves, dh)
    kept = torch.float32 if wide else dtype
    code, kind, sizes, none = lib.i32(lib.dtype_code(dtype)), lib.i32(lib.dtype_code(kept)), (lib.i64(tokens), lib.i64(n_in), lib.i64(n_out)), lib.stream_ptr()
    pitch = -(-n_out // 8) * 8
    out, a, b = Piece((tokens, n_out), dtype, 2 * at), Piece((tokens, pitch), kept), Piece((tokens, pitch), kept)
    ws = Piece((size_of("mega_gated_linear_workspace_bytes", *sizes, lib.i32(0)),), torch.uint8)
    lib.call("mega_gated_linear_fwd", lib.ptr(x), lib.ptr(w1), lib.ptr(w3), code, *sizes, out.pointer, a.pointer, b.pointer, kind, ws.pointer, none)
    assert out.kept() and a.kept() and b.kept() and ws.kept() and same(out.value(), h.detach())
    alone = Piece((tokens, n_out), dtype, 2 * at)
    lib.call("mega_gated_linear_fwd", lib.ptr(x), lib.ptr(w1), lib.ptr(w3), code, *sizes, alone.pointer, lib.ptr(None), lib.ptr(None), kind, ws.pointer, none)
    assert alone.kept() and ws.kept() and same(alone.value(), h.detach())
    grads = [Piece(t.shape, dtype, 2 * at) for t in (x, w1, w3)]
    ws = Piece((size_of("mega_gated_linear_workspace_bytes", *sizes, lib.i32(7)),), torch.uint8)
    lib.call("mega_gated_linear_bwd", lib.ptr(dh), lib.ptr(x), lib.ptr(w1), lib.ptr(w3), a.pointer, b.pointer, kind, code, *sizes, *(p.pointer for p in grads), ws.pointer, none)
    assert ws.kept() and a.kept() and b.kept()
    for p, w in zip(grads, want):
        assert p.kept() and same(p.value(), w)


@pytest.mark.parametrize("at", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_clipping(dtype, at):
    """Views between guards of one buffer, read and written on any element's boundary."""
    g = torch.Generator("cuda").manual_seed(9)
    sizes = [1, 2, 7, 8, 9, 1000, 8191, 8192, 8193, 16385, 100003]
    buffers = [Piece((n + 1,), dtype) for n in sizes]
    out = [p.tensor[at:at + n] for p, n in zip(buffers, sizes)]
    ts = [torch.randn(n + 1, generator=g, device="cuda").to(dtype)[1 - at:][:n] for n in sizes]
    norm, new = fused_ops.clip_grads(ts, 1.0, out=out)
    _, want = fused_ops.clip_grads([t.clone() for t in ts], 1.0)
    for p, o, w in zip(buffers, new, want):
        assert p.kept() and same(o.clone(), w)
        rest = p.value()[-1:] if at == 0 else p.value()[:1]
        assert (rest.view(torch.uint8) == MARK).all()
