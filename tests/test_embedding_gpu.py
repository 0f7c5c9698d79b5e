"""Embedding and its gradient against the formulas in 64 bits.

A value is off by at most the rounding of its product in float32 and half a step of its type; a gradient by that and by
(n + 2) 2^-24 of the magnitudes that its n summands have together."""
import pytest
import torch

from megalodon_amd import fused_ops
from megalodon_amd.modules import Embedding

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(t, dtype):
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def formula(tokens, weight, dy, scale, padding):
    """(y, bar), (dw, bar)"""
    V, D = weight.shape
    t = tokens.reshape(-1).long()
    there = (t >= 0) & (t < V)
    w = weight.detach().double()
    y = torch.where(there[:, None], w[t.clamp(0, V - 1)] * scale, 0.0)
    kept = there if padding is None else there & (t != padding % V)
    rows = dy.reshape(-1, D).double()[kept]
    dw, mag, n = torch.zeros_like(w), torch.zeros_like(w), torch.zeros(V, dtype=torch.float64, device=w.device)
    dw.index_add_(0, t[kept], rows)
    mag.index_add_(0, t[kept], rows.abs())
    n.index_add_(0, t[kept], torch.ones_like(t[kept], dtype=torch.float64))
    dw, mag = dw * scale, mag * abs(scale)
    off = (n[:, None] + 3) * U * mag
    return (y, half(y, weight.dtype) + 3 * U * y.abs()), (dw, off + half(dw.abs() + off, weight.dtype))


def close(got, want):
    value, bar = want
    off = (got.detach().double().reshape(value.shape) - value).abs()
    assert bool((off <= bar).all()), f"{(off - bar).max().item():.3g} over the bar"


def check(tokens, weight, scale=1.0, padding=None, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    dy = torch.randn(*tokens.shape, weight.shape[1], generator=g, device="cuda").to(weight.dtype)
    want_y, want_dw = formula(tokens, weight, dy, scale, padding)
    with torch.no_grad():
        close(fused_ops.embedding(tokens, weight, scale, padding), want_y)
    leaf = weight.clone().requires_grad_(True)
    y = fused_ops.embedding(tokens, leaf, scale, padding)
    assert y.shape == (*tokens.shape, weight.shape[1]) and y.dtype == weight.dtype
    close(y, want_y)
    dw, = torch.autograd.grad(y, leaf, dy)
    close(dw, want_dw)
    again, = torch.autograd.grad(fused_ops.embedding(tokens, leaf, scale, padding), leaf, dy)
    assert torch.equal(dw, again)
    return dw


def table(V, D, dtype, seed=0):
    return torch.randn(V, D, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def text(n, V, seed=0):
    """Tokens as frequent as in text: the r-th about 1 / r."""
    g = torch.Generator("cuda").manual_seed(seed)
    rank = ((V + 1.0) ** torch.rand(n, generator=g, device="cuda", dtype=torch.float64)).long().sub(1).clamp(0, V - 1)
    return torch.randperm(V, generator=g, device="cuda")[rank]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V,D", [(1, 1), (2, 3), (100, 8), (37, 129), (1000, 1001), (50, 2048), (33, 2056), (500, 4100)])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 257, 2000])
def test_sizes(n, V, D, dtype):
    check(text(n, V, n), table(V, D, dtype), D ** 0.5)


@pytest.mark.parametrize("n", [4084, 8191, 8192, 8193, 12345, 40000])
@pytest.mark.parametrize("V", [1, 3, 2047, 2048, 50001])
def test_many_tokens(n, V):
    """Both ways to sort; digits of one pass and of two."""
    check(text(n, V, n + V), table(V, 72, torch.bfloat16), 0.5)


@pytest.mark.parametrize("V", [900, 70001])
def test_several_lines_of_positions_for_a_workgroup(V):
    g = torch.Generator("cuda").manual_seed(V)  # (no frequent ones: the oracle adds up in 64 bits one by one)
    check(torch.randint(V, (2048 * 1024 * 2 + 12345,), generator=g, device="cuda", dtype=torch.int32), table(V, 4, torch.bfloat16))


def test_three_passes():
    V = (1 << 22) + 77
    n = 9000
    tokens = torch.randint(0, V, (n,), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    tokens[::7] = V - 1
    tokens[::11] = 0
    check(tokens, table(V, 8, torch.bfloat16), 2.0)


@pytest.mark.parametrize("n", [5000, 20000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_runs_over_many_pieces(n, dtype):
    """One token at every position; two that share them; one at both ends of the line."""
    weight = table(9, 520, dtype)
    check(torch.full((n,), 4, device="cuda"), weight)
    check(torch.arange(n, device="cuda") % 2 * 8, weight)
    check((torch.arange(n, device="cuda") >= n - 3).long() * 8, weight)


@pytest.mark.parametrize("D", [1, 9, 64, 500, 1100, 1030])
@pytest.mark.parametrize("n", [3000, 100001])
def test_narrow_rows(n, D):
    """Several pieces to a workgroup; one token has most of the positions, one the last of each hundred, the others few."""
    tokens = torch.full((n,), 5, device="cuda")
    tokens[99::100] = 2
    tokens[7::10000] = torch.arange(len(tokens[7::10000]), device="cuda") % 6
    check(tokens, table(7, D, torch.bfloat16))


@pytest.mark.parametrize("n", [700, 9001])
def test_sums_run_in_order(n):
    """The sums are those of one order, whatever the other tokens are: small numbers behind a large one come out the same."""
    weight = torch.zeros(5, 64, device="cuda")
    tokens = torch.full((n,), 2, device="cuda")
    dy = torch.randn(n, 64, device="cuda") * 10.0 ** torch.randint(-3, 4, (n, 1), device="cuda")
    leaf = weight.requires_grad_(True)
    first, = torch.autograd.grad(fused_ops.embedding(tokens, leaf), leaf, dy)
    for other in (0, 1, 3, 4):
        got, = torch.autograd.grad(fused_ops.embedding(torch.full_like(tokens, other), leaf), leaf, dy)
        assert torch.equal(got[other], first[2]) and not got[[i for i in range(5) if i != other]].any()


@pytest.mark.parametrize("bits", [torch.int32, torch.int64])
@pytest.mark.parametrize("n", [100, 10000])
def test_padding_and_foreign_tokens(n, bits):
    V = 300
    tokens = torch.randint(0, V, (n,), device="cuda", generator=torch.Generator("cuda").manual_seed(n)).to(bits)
    tokens[::3] = 7
    tokens[1::10] = -1
    tokens[2::10] = V
    tokens[3::10] = torch.iinfo(bits).min
    tokens[4::10] = torch.iinfo(bits).max
    weight = table(V, 136, torch.bfloat16)
    dw = check(tokens.view(2, -1), weight, 3.0, padding=7)
    assert not dw[7].any()
    dw = check(tokens, weight, 3.0, padding=7 - V)
    assert not dw[7].any()
    dw = check(torch.full((n,), 7, device="cuda", dtype=bits), weight, padding=7)
    assert not dw.any()


def test_every_row_is_written():
    """Rows without a token come out as zeros whatever the memory held, rows in front of and behind the gradient's stay."""
    weight = table(1000, 24, torch.float32).requires_grad_(True)
    tokens = torch.tensor([999, 0, 500], device="cuda")
    for _ in range(3):
        junk = torch.full((1000, 24), float("nan"), device="cuda")
        del junk
        dw, = torch.autograd.grad(fused_ops.embedding(tokens, weight).sum(), weight)
        assert dw[[0, 500, 999]].eq(1).all() and dw.sum() == 72


@pytest.mark.parametrize("V,D,dtype", [(40001, 1001, torch.float32), (70003, 1003, torch.bfloat16), (33, 3, torch.bfloat16)])
def test_rows_without_tokens(V, D, dtype):
    """Lines of rows of any width and boundary, in tables that a cache holds and in larger ones."""
    tokens = torch.tensor([0, V - 1, 17, 18, 5, 5, V // 2], device="cuda")
    leaf = table(V, D, dtype).requires_grad_(True)
    junk = torch.full((V * D + 16,), 7.0, dtype=dtype, device="cuda")  # (what the gradient's memory held)
    del junk
    dy = torch.ones(len(tokens), D, dtype=dtype, device="cuda")
    dw, = torch.autograd.grad(fused_ops.embedding(tokens, leaf), leaf, dy)
    want = torch.bincount(tokens, minlength=V).to(dtype)
    assert torch.equal(dw, want[:, None].expand(V, D))


def test_no_tokens():
    weight = table(10, 16, torch.float16).requires_grad_(True)
    for shape in ((0,), (3, 0)):
        y = fused_ops.embedding(torch.empty(shape, dtype=torch.long, device="cuda"), weight)
        assert y.shape == (*shape, 16)
        dw, = torch.autograd.grad(y, weight, torch.empty_like(y))
        assert dw.shape == weight.shape and not dw.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Tables that are slices or transposed, rows off 16 bytes, a scalar token, tokens and gradients of other strides."""
    whole = table(64, 41, dtype)
    tokens = text(60, 30, 5).view(6, 10)
    for weight in (whole[:30, :33], whole[5:35, 3:40], whole.t()[:30], whole[::2][:30], whole[:1].expand(30, 41)):
        with torch.no_grad():
            close(fused_ops.embedding(tokens.t(), weight, 2.0), formula(tokens.t(), weight, torch.zeros(10, 6, weight.shape[1], device="cuda"), 2.0, None)[0])
    assert torch.equal(fused_ops.embedding(torch.tensor(3, device="cuda"), whole), whole[3])
    leaf = whole[:30].clone().requires_grad_(True)
    dy = torch.randn(41, 10, 6, device="cuda").to(dtype).permute(2, 1, 0)
    dw, = torch.autograd.grad(fused_ops.embedding(tokens, leaf), leaf, dy)
    close(dw, formula(tokens, leaf, dy, 1.0, None)[1])
    dw, = torch.autograd.grad(fused_ops.embedding(tokens, leaf), leaf, torch.ones(1, 1, 1, device="cuda", dtype=dtype).expand(6, 10, 41))
    close(dw, formula(tokens, leaf, torch.ones(6, 10, 41, device="cuda"), 1.0, None)[1])


def test_values_that_are_not_finite():
    """They stay in their rows."""
    weight = table(20, 40, torch.bfloat16)
    weight[3, 5], weight[4, 6] = float("nan"), float("inf")
    tokens = torch.tensor([1, 3, 4, 2, -5, 3], device="cuda")
    y = fused_ops.embedding(tokens, weight, 2.0)
    assert y[[0, 3, 4]].isfinite().all() and y[1, 5].isnan() and y[2, 6].isinf() and not y[4].any()
    leaf = weight.clone().requires_grad_(True)
    dy = torch.ones(6, 40, device="cuda", dtype=torch.bfloat16)
    dy[4], dy[0, 0] = float("nan"), float("inf")
    dw, = torch.autograd.grad(fused_ops.embedding(tokens, leaf), leaf, dy)
    assert dw[1, 0].isinf() and dw[[i for i in range(20) if i != 1]].isfinite().all() and dw[3].eq(2).all()


def test_differentiated_twice():
    tokens = torch.tensor([[1, 2, 2], [9, -1, 0]], device="cuda")
    weight = table(9, 5, torch.float32).requires_grad_(True)
    dy = torch.randn(2, 3, 5, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(fused_ops.embedding(tokens, weight, 3.0, 2), weight, dy, create_graph=True)
    v = torch.randn_like(dw)
    back, = torch.autograd.grad(dw, dy, v)
    want = torch.zeros_like(dy)
    want[0, 0], want[1, 2] = 3.0 * v[1], 3.0 * v[0]
    assert torch.allclose(back, want, rtol=1e-6)


def test_captured():
    """Forward and backward in a graph whose replays follow new tokens and gradients, eager calls between them."""
    V, n = 500, 9000
    weight = table(V, 64, torch.bfloat16).requires_grad_(True)
    tokens, dy = text(n, V), torch.randn(n, 64, device="cuda").bfloat16()
    step = lambda: (lambda y: (y.detach(), *torch.autograd.grad(y, weight, dy)))(fused_ops.embedding(tokens, weight, 2.0, 3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for seed in range(4):
        tokens.copy_(text(n, V, seed + 10))
        dy.normal_()
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_two_streams():
    """Calls side by side do not share their workspaces."""
    weight = table(400, 256, torch.float32).requires_grad_(True)
    work = [(text(6000 + 3000 * i, 400, i), torch.randn(6000 + 3000 * i, 256, device="cuda")) for i in range(2)]
    alone = [torch.autograd.grad(fused_ops.embedding(t, weight), weight, dy)[0] for t, dy in work]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in work], [[], []]
    for _ in range(5):
        for i, (t, dy) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                y = fused_ops.embedding(t, weight)
                got[i].append(torch.autograd.grad(y, weight, dy)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(g, alone[i]) for i in range(2) for g in got[i])


def test_module():
    torch.manual_seed(0)
    layer = Embedding(50, 32, padding_idx=4, scale=2.0, device="cuda", dtype=torch.bfloat16)
    assert not layer.weight[4].any() and set(layer.state_dict()) == {"weight"}
    tokens = torch.tensor([[4, 5, 5]], device="cuda")
    y = layer(tokens)
    assert torch.equal(y, 2 * layer.weight[tokens])
    y.sum().backward()
    assert layer.weight.grad[5].eq(4).all() and layer.weight.grad.sum() == 128


@pytest.mark.parametrize("bad", ["tokens", "weight", "dims", "empty", "padding", "cpu", "double"])
def test_refusals(bad):
    tokens, weight, padding = torch.zeros(3, dtype=torch.long, device="cuda"), table(5, 8, torch.float32), None
    if bad == "tokens": tokens = tokens.short()
    if bad == "weight": weight = weight.long()
    if bad == "dims": weight = weight[0]
    if bad == "empty": weight = weight[:0]
    if bad == "padding": padding = 5
    if bad == "cpu": weight = weight.cpu()
    if bad == "double": weight = weight.double()
    with pytest.raises(RuntimeError):
        fused_ops.embedding(tokens, weight, 1.0, padding)
