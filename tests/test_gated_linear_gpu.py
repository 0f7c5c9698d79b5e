"""The gated half of a feed-forward network, silu(x w1^T) * (x w3^T), against its formula in 64 bits.

Bars are sums of what can go wrong, element by element: a rounding to the element type is off by at most eps / 2 of the
value (or half of the smallest number), a float32 sum of n products by n 2^-24 of their magnitudes, exp by a few 2^-22 times
its argument.  silu has |silu'| <= 1.1 and |silu''| <= 0.5.  What the backward feeds the matrix cores (da, db) is rounded once (up to 64 tokens: to
two terms), and so is what it keeps (a, b) where that is in the operands' type."""
import pytest
import torch

from megalodon_amd import fused_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def half(t, dtype):
    """How far rounding t to dtype can be off."""
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def product(a, ea, b, eb, n):
    """A float32 sum of n products of a (off by ea) and b (off by eb): how far it can be off."""
    return (n + 2) * U * ((a.abs() + ea) @ (b.abs() + eb)) + ea @ b.abs() + a.abs() @ eb + ea @ eb


def formula(x, w1, w3, dh, dtype, kept=None):
    """((value, bar), ...) of h, dx, dw1, dw3."""
    x, w1, w3, dh = (t.detach().double() for t in (x, w1, w3, dh))
    none = lambda t: torch.zeros_like(t)
    K, H, T = x.shape[1], w1.shape[0], x.shape[0]
    a, b = x @ w1.t(), x @ w3.t()
    ea, eb = (product(x, none(x), w.t(), none(w.t()), K) for w in (w1, w3))
    s = torch.sigmoid(a)
    g = a * s
    h = g * b
    exp = 2.0 ** -20 * (2 + a.abs())
    eh = 1.1 * ea * (b.abs() + eb) + g.abs() * eb + exp * h.abs()
    out = [(h, eh + half(h.abs() + eh, dtype))]
    if kept == dtype:
        ea, eb = ea + half(a.abs() + ea, dtype), eb + half(b.abs() + eb, dtype)
    slope = s * (1 + a * (1 - s))
    da, db = dh * b * slope, dh * g
    eda = dh.abs() * ((slope.abs() + 0.5 * ea) * eb + 0.5 * ea * b.abs() + exp * b.abs() * 2)
    edb = dh.abs() * (1.1 * ea + exp * (g.abs() + ea))
    rounding = lambda t: half(half(t, dtype), dtype) if T <= 64 else half(t, dtype)  # (up to 64 tokens: what rounding left is rounded itself)
    eda, edb = eda + rounding(da.abs() + eda), edb + rounding(db.abs() + edb)
    dx = da @ w1 + db @ w3
    edx = product(da, eda, w1, none(w1), 2 * H) + product(db, edb, w3, none(w3), 2 * H)
    out.append((dx, edx + half(dx.abs() + edx, dtype)))
    for d, e in ((da, eda), (db, edb)):
        w, ew = d.t() @ x, product(d.t(), e.t(), x, none(x), T)
        out.append((w, ew + half(w.abs() + ew, dtype)))
    return out


def close(got, want):
    value, bar = want
    assert got.shape == value.shape
    off = (got.double() - value).abs()
    assert bool((off <= bar).all()), f"{(off / bar).max().item():.3g} times the bar"
    # ... and on the whole, where the signs of roundings differ: a correct result is off by eps / sqrt(12) at most for each of
    # the four roundings on its way
    if value.numel() > 1000:
        assert off.norm() <= 4 * torch.finfo(got.dtype).eps / 12 ** 0.5 * value.norm() + 1e-12


def operands(tokens, n_in, n_out, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + tokens + 7 * n_in + 11 * n_out)
    rows = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return (rows(tokens, n_in).to(dtype), (rows(n_out, n_in) / n_in ** 0.5).to(dtype), (rows(n_out, n_in) / n_in ** 0.5).to(dtype), rows(tokens, n_out).to(dtype))


def check(x, w1, w3, dh):
    with torch.no_grad():
        alone = fused_ops.gated_linear(x, w1, w3)
    for kept in (None, x.dtype):
        want = formula(x, w1, w3, dh, x.dtype, kept)
        close(alone, want[0])
        leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
        h = fused_ops.gated_linear(*leaves, kept)
        assert torch.equal(h, alone)
        for got, w in zip(torch.autograd.grad(h, leaves, dh), want[1:]):
            close(got, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 32, 33, 63, 64])
@pytest.mark.parametrize("n_in,n_out", [(64, 16), (1024, 2752), (8, 1), (1, 17), (7, 5), (1001, 31), (520, 192)])
def test_few_tokens(tokens, n_in, n_out, dtype):
    check(*operands(tokens, n_in, n_out, dtype))


@pytest.mark.parametrize("tokens", [8, 9, 13, 16])
@pytest.mark.parametrize("n_in,n_out,dtype", [(2048, 5504, torch.float16), (4096, 333, torch.bfloat16), (1544, 4100, torch.float16), (1032, 8, torch.bfloat16), (3000, 17, torch.bfloat16)])
def test_tokens_in_lds(tokens, n_in, n_out, dtype):
    """Rows of whole and part-filled steps, last groups of features that are not whole, workgroups without a second group."""
    check(*operands(tokens, n_in, n_out, dtype))


@pytest.mark.parametrize("tokens,n_in,n_out,dtype", [
    (65, 64, 8, torch.bfloat16),           # part of a tile
    (65, 1, 1, torch.float16),             # rows and columns laid out anew
    (129, 1001, 63, torch.bfloat16),
    (300, 1024, 2752, torch.bfloat16),     # tiles of 128, at most one for a CU
    (100, 2048, 640, torch.float16),       # cut along k
    (1021, 1024, 2752, torch.float16),     # more than one for a CU
    (2000, 1000, 2731, torch.bfloat16),    # the same, odd
    (4084, 2048, 5504, torch.bfloat16),    # tiles of 256
    (1531, 4096, 11008, torch.bfloat16),   # the last round's cut along k
    (257, 4095, 300, torch.float16),
    (2500, 512, 4100, torch.float16),
    (30000, 64, 2000, torch.bfloat16),     # several tiles of 256 for a workgroup, of one slab,
    (30011, 128, 1999, torch.float16),     # two,
    (30000, 192, 2000, torch.bfloat16),    # three
    (20000, 320, 2100, torch.bfloat16),    # and five
    (200, 4096, 2048, torch.bfloat16),
    (5000, 520, 1032, torch.bfloat16),     # both gradients' sums in pieces
    (20000, 264, 72, torch.float16),       # dw of two tiles, many pieces
    (700, 24, 130000, torch.bfloat16),     # dx of three
    (66000, 40, 40, torch.float16),        # a tile more than the chip has units
    (300, 1000, 2736, torch.bfloat16),     # a last slab of 40 k
    (1500, 3064, 1000, torch.float16),     # of 56, in pieces
])
def test_tiles(tokens, n_in, n_out, dtype):
    check(*operands(tokens, n_in, n_out, dtype))


@pytest.mark.parametrize("n_in", [1024, 1001])
def test_tokens_of_several_launches(n_in):
    """An operand of 2^30 elements and more: launch by launch, the weights' gradients added to."""
    one = ((1 << 30) - 1) // (-(-n_in // 8) * 8) // 256 * 256  # tokens of a launch
    tokens, n_out = one + 300, 8
    x, w1, w3, dh = operands(tokens, n_in, n_out, torch.bfloat16)
    want = formula(x, w1, w3, dh, x.dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
    h = fused_ops.gated_linear(*leaves)
    close(h, want[0])
    dx, *dw = torch.autograd.grad(h, leaves, dh)
    close(dx, want[1])
    del dx, h
    first = formula(x[:one], w1, w3, dh[:one], x.dtype)
    for got, (value, bar), (part, off) in zip(dw, want[2:], first[2:]):
        close(got, (value, bar + half(part.abs() + off, x.dtype)))  # (the first launch's sum was rounded)


@pytest.mark.parametrize("tokens", [5, 200])
def test_layouts(tokens):
    """Leading axes, transposed and misaligned operands, an output gradient of another layout."""
    x, w1, w3, dh = operands(tokens * 2, 136, 72, torch.bfloat16)
    want = formula(x, w1, w3, dh, x.dtype)
    with torch.no_grad():
        assert torch.equal(fused_ops.gated_linear(x.view(2, tokens, 136), w1, w3).view(2 * tokens, 72), fused_ops.gated_linear(x, w1, w3))
        close(fused_ops.gated_linear(x.t().contiguous().t(), w1, w3), want[0])
        shifted = [torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (x, w1, w3)]
        close(fused_ops.gated_linear(*shifted), want[0])
        close(fused_ops.gated_linear(x, torch.cat([w1, w3], 1)[:, :136], torch.cat([w1, w3], 1)[:, 136:]), want[0])
        close(fused_ops.gated_linear(x[:1].expand(7, 136), w1, w3), tuple(t[:1].expand(7, 72) for t in want[0]))
        vector = fused_ops.gated_linear(x[3], w1, w3)
        close(vector, tuple(t[3] for t in want[0]))
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
    h = fused_ops.gated_linear(*leaves)
    for got, w in zip(torch.autograd.grad(h, leaves, dh.t().contiguous().t()), want[1:]):
        close(got, w)


@pytest.mark.parametrize("tokens", [3, 128])
def test_some_gradients(tokens):
    x, w1, w3, dh = operands(tokens, 192, 128, torch.bfloat16)
    want = formula(x, w1, w3, dh, x.dtype)[1:]
    for asked in ([0], [1], [2], [1, 2], [0, 2]):
        leaves = [t.clone().requires_grad_(i in asked) for i, t in enumerate((x, w1, w3))]
        got = torch.autograd.grad(fused_ops.gated_linear(*leaves), [leaves[i] for i in asked], dh)
        for i, g in zip(asked, got):
            close(g, want[i])


def test_gradients_are_tensors_of_their_own():
    x, w1, w3, dh = operands(70, 72, 40, torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
    grads = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
    assert all(g.untyped_storage().nbytes() == 2 * g.numel() and g.is_contiguous() for g in grads)


@pytest.mark.parametrize("tokens", [9, 130])
def test_output_gradient_negated_on_reading(tokens):
    x, w1, w3, dh = operands(tokens, 72, 40, torch.float16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
    h = fused_ops.gated_linear(*leaves)
    want = torch.autograd.grad(h, leaves, dh, retain_graph=True)
    for got, w in zip(torch.autograd.grad(h, leaves, torch._neg_view(-dh)), want):
        assert torch.equal(got, w)


def test_saved_tensors_through_hooks():
    """What is saved may travel (host memory, another boundary); of another shape it is refused."""
    x, w1, w3, dh = operands(70, 72, 36, torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
    want = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
    shifted = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), shifted):
        h = fused_ops.gated_linear(*leaves)
    for got, w in zip(torch.autograd.grad(h, leaves, dh), want):
        assert torch.equal(got, w)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[: t.shape[0] // 2]):
        h = fused_ops.gated_linear(*leaves)
    with pytest.raises(RuntimeError, match="saved tensor"):
        torch.autograd.grad(h, leaves, dh)


def test_no_tokens():
    _, w1, w3, _ = operands(1, 64, 32, torch.float16)
    x = torch.empty(0, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    w1.requires_grad_(True)
    h = fused_ops.gated_linear(x, w1, w3)
    assert h.shape == (0, 32)
    dx, dw = torch.autograd.grad(h, (x, w1), torch.empty_like(h))
    assert dx.shape == x.shape and not dw.any()


@pytest.mark.parametrize("tokens,n_in", [(4, 64), (130, 64), (130, 60), (11, 1288)])
def test_rows_do_not_touch_each_other(tokens, n_in):
    """An infinity or a NaN in one token's row, or in a feature's weights, stays there."""
    x, w1, w3, _ = operands(tokens, n_in, 40, torch.bfloat16)
    clean = fused_ops.gated_linear(x, w1, w3)
    x2, w2 = x.clone(), w1.clone()
    x2[1, 5], x2[2, 0], w2[7, 3] = float("nan"), float("inf"), float("inf")
    got = fused_ops.gated_linear(x2, w2, w3)
    rows = [i for i in range(tokens) if i not in (1, 2)]
    columns = [i for i in range(40) if i != 7]
    assert torch.equal(got[rows][:, columns], clean[rows][:, columns])
    assert got[1].isnan().all() and not got[2].isfinite().all()
    dh = torch.ones_like(clean)
    grads = []
    for t in (x, x2):
        leaf = t.clone().requires_grad_(True)
        grads.append(torch.autograd.grad(fused_ops.gated_linear(leaf, w1, w3), leaf, dh)[0])
    assert torch.equal(grads[1][rows], grads[0][rows]) and grads[1][1].isnan().all()


def test_large_arguments():
    """Gates far on either side: exp overflows and the gate is zero, or the argument itself."""
    x = torch.tensor([[400.0], [-400.0], [90.0], [-90.0], [0.0]], device="cuda").bfloat16()
    for rows in (x, x.repeat(20, 1)):
        w = torch.ones(8, 1, device="cuda").bfloat16()
        got = fused_ops.gated_linear(rows, w, w).double()
        v = rows.double().expand(-1, 8)
        assert ((got - v * v * torch.sigmoid(v)).abs() <= 2.0 ** -8 * v * v * torch.sigmoid(v) + 1e-30).all()


def test_differentiated_twice():
    x, w1, w3, _ = (t.float().cpu().double() for t in operands(6, 16, 8, torch.bfloat16))
    a, b = (torch.randn(6, 8, dtype=torch.float64), torch.randn(6, 16, dtype=torch.float64))

    def second(fn, cast):
        leaves = [cast(t).requires_grad_(True) for t in (x, w1, w3)]
        dx, = torch.autograd.grad(fn(*leaves), leaves[:1], cast(a), create_graph=True)
        return torch.autograd.grad(dx, leaves, cast(b))

    got = second(fused_ops.gated_linear, lambda t: t.cuda().bfloat16())
    want = second(lambda x, w1, w3: torch.nn.functional.silu(x @ w1.t()) * (x @ w3.t()), lambda t: t.bfloat16().double())
    for g, w in zip(got, want):
        assert (g.double().cpu() - w).norm() <= 0.05 * w.norm()


@pytest.mark.parametrize("sizes", [(96, 256, 160), (7, 250, 90), (4500, 500, 1410)])
def test_captured(sizes):
    """Forward and backward in a graph whose replays follow new operands, the program's own work between them."""
    x, w1, w3, dh = operands(*sizes, torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        h = fused_ops.gated_linear(*leaves)
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for seed in range(3):
        new = operands(*sizes, torch.bfloat16, seed)
        with torch.no_grad():
            for t, v in zip((*leaves, dh), new):
                t.copy_(v)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_two_streams():
    """Calls on two streams at once have workspaces of their own."""
    many = [operands(2500, 500, 1410, torch.bfloat16, seed) for seed in range(4)]

    def one(x, w1, w3, dh):
        leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
        h = fused_ops.gated_linear(*leaves)
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))

    want = [one(*m) for m in many]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None] * 4
    for i, m in enumerate(many):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = one(*m)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_against_differences():
    """The gradients against differences of the operator's own outputs (steps that the types hold exactly)."""
    x, w1, w3, _ = operands(3, 8, 4, torch.float16)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w3)]
    grads = torch.autograd.grad(fused_ops.gated_linear(*leaves).sum(), leaves)
    step = 2.0 ** -5
    for i in range(3):
        for at in ((0, 0), (2, 3)):
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in (x, w1, w3)]
                moved[i][at] = torch.round(moved[i][at] / 2 ** -8) * 2 ** -8 + sign * step
                ends.append(fused_ops.gated_linear(*moved).double().sum())
            slope = ((ends[0] - ends[1]) / (2 * step)).item()
            # rounding of 12 outputs at either end over the distance; third derivatives times step^2
            assert abs(slope - grads[i][at].item()) <= 0.15 + 0.05 * abs(slope)


@pytest.mark.parametrize("bad", ["dtype", "float32", "shapes", "n_in", "cpu", "empty", "kept"])
def test_refusals(bad):
    x, w1, w3, _ = operands(4, 16, 8, torch.bfloat16)
    if bad == "dtype": w3 = w3.half()
    if bad == "float32": x, w1, w3 = x.float(), w1.float(), w3.float()
    if bad == "shapes": w3 = w3[:4]
    if bad == "n_in": x = x[:, :8]
    if bad == "cpu": x = x.cpu()
    if bad == "empty": w1, w3 = w1[:0], w3[:0]
    with pytest.raises(RuntimeError):
        fused_ops.gated_linear(x, w1, w3, torch.float16 if bad == "kept" else None)
