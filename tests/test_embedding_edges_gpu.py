"""Embedding's gradient at the ends of its ranges.

Where gradients are small whole numbers, every sum of them below 2^24 is exact in float32, in any order, and a result is that sum rounded once."""
import pytest
import torch

from megalodon_amd import fused_ops
from megalodon_amd.modules import Embedding

pytestmark = pytest.mark.gpu


def test_more_pieces_than_a_launch_has_threads_for():
    """Rows of 8 columns have pieces of 4 positions: from 2^26 tokens on a workgroup for each, of 256 threads, would be 2^32 threads and more."""
    n, V, D = (1 << 26) + 12345, 1009, 8
    g = torch.Generator("cuda").manual_seed(1)
    tokens = torch.randint(0, V, (n,), generator=g, device="cuda", dtype=torch.int32)
    tokens[::5] = 77  # one that has a fifth of the positions
    dy = torch.randint(-1, 3, (n, D), generator=g, device="cuda", dtype=torch.int8).bfloat16()
    weight = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    junk = torch.full((V, D), 7.0, dtype=torch.bfloat16, device="cuda")  # (what the gradient's memory held)
    y = fused_ops.embedding(tokens, weight)
    del junk
    dw, = torch.autograd.grad(y, weight, dy)
    del y
    want = torch.stack([torch.bincount(tokens, dy[:, d].double(), minlength=V) for d in range(D)], 1)
    assert want.abs().max() < 1 << 24
    assert torch.equal(dw, want.to(torch.float32).bfloat16())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradient_that_is_differentiated_again(dtype):
    """The gradient is the one without `create_graph`, bit for bit: frequent tokens are summed in float32, in one order, and scaled once.  Its own gradients are
    the formula's: dW[v] = s sum dy[r], so that a table u of ones' gradients gives s u[t_r] where r counts."""
    n, V, D, scale, padding = 6000, 50, 24, 3.0, 7
    g = torch.Generator("cuda").manual_seed(5)
    tokens = torch.randint(-2, V + 2, (2, n // 2), generator=g, device="cuda")
    tokens[:, ::2], tokens[:, 1::8] = 11, padding
    weight = torch.randn(V, D, generator=g, device="cuda").to(dtype).requires_grad_(True)
    dy = torch.randn(2, n // 2, D, generator=g, device="cuda").abs().to(dtype).requires_grad_(True)
    y = fused_ops.embedding(tokens, weight, scale, padding)
    once, = torch.autograd.grad(y, weight, dy.detach(), retain_graph=True)
    for _ in range(2):
        again, = torch.autograd.grad(y, weight, dy, create_graph=True)
        assert torch.equal(again, once) and again.requires_grad
    kept = (tokens >= 0) & (tokens < V) & (tokens != padding)
    rows = dy.detach().double()[kept]
    want = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, tokens[kept], rows) * scale
    # 6000 positive float32 summands, the scale's product, one rounding; whole in float16 (11 has 3000 of |N(0, 1)|, 7200 or so)
    assert ((again.detach().double() - want).abs() <= (6002 * 2.0 ** -24 + 1.01 * torch.finfo(dtype).eps / 2) * want).all()
    u = torch.randn(V, D, generator=g, device="cuda").to(dtype).requires_grad_(True)
    back, = torch.autograd.grad(again, dy, u, create_graph=True)
    assert torch.equal(back.detach(), torch.where(kept[..., None], (u.detach().float() * scale)[tokens.clamp(0, V - 1)], 0.0).to(dtype))
    # ... and once more: u's gradient is dW of the gradients of `back`
    v = torch.randn(2, n // 2, D, generator=g, device="cuda").abs().to(dtype)
    third, = torch.autograd.grad(back, u, v)
    want = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, tokens[kept], v.double()[kept]) * scale
    assert ((third.double() - want).abs() <= (6002 * 2.0 ** -24 + 1.01 * torch.finfo(dtype).eps / 2) * want).all()


class Rows(torch.nn.Module):
    """Two tables, one scaled and with a padding row."""

    def __init__(self, dtype):
        super().__init__()
        self.first = Embedding(40, 16, padding_idx=3, scale=0.5, device="cuda", dtype=dtype)
        self.second = Embedding(40, 8, device="cuda", dtype=dtype)

    def forward(self, tokens):
        return self.first(tokens), self.second(tokens)


def foreign(seed, shape=(4, 25), V=40, bits=torch.long):
    """Tokens with some that are no row."""
    return torch.randint(-3, V + 3, shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(bits)


@pytest.mark.parametrize("gradients", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_traced(dtype, gradients):
    """A trace holds operations: called with other tokens it gives what the layer gives, and the layer's gradients."""
    layers = Rows(dtype)
    with torch.set_grad_enabled(gradients):
        traced = torch.jit.trace(layers, (foreign(1),), check_trace=False)
        for seed in (2, 3):
            tokens = foreign(seed)
            got, want = traced(tokens), layers(tokens)
            assert all(torch.equal(a, b) and a.requires_grad == gradients for a, b in zip(got, want))
    if gradients:
        dy = [torch.randint(-2, 3, y.shape, device="cuda").to(dtype) for y in want]
        for a, b in zip(torch.autograd.grad(got, layers.parameters(), dy), torch.autograd.grad(want, layers.parameters(), dy)):
            assert torch.equal(a, b)  # (whole numbers and halves: exact)


def test_fake_tensors():
    from torch._subclasses import FakeTensorMode
    with FakeTensorMode():
        fake = Embedding(40, 16, scale=2.0, device="cuda", dtype=torch.bfloat16)
        y = fake(torch.zeros(5, 3, device="cuda", dtype=torch.long))
        assert y.shape == (5, 3, 16) and y.dtype == torch.bfloat16
        dw, = torch.autograd.grad(y, fake.weight, torch.empty_like(y))
        assert dw.shape == (40, 16)


def test_functions_of_functions():
    """vmap over tokens and over tables, functionalize, several gradients at once, gradients that are zeros without memory."""
    layer = Embedding(40, 16, padding_idx=3, scale=0.5, device="cuda", dtype=torch.bfloat16)
    tokens = foreign(4, (6, 9))
    with torch.no_grad():
        want = layer(tokens)
        assert torch.equal(torch.func.vmap(layer)(tokens), want)
        tables = torch.stack([layer.weight, -layer.weight])
        both = torch.func.vmap(lambda w: fused_ops.embedding(tokens, w, 0.5, 3))(tables)
        assert torch.equal(both, torch.stack([want, -want]))
        assert torch.equal(torch.func.functionalize(layer)(tokens), want)
    for bits in (torch.int32, torch.long):
        y = layer(tokens.to(bits))
        many = torch.randint(-2, 3, (3, *y.shape), device="cuda").bfloat16()
        got, = torch.autograd.grad(y, layer.weight, many, is_grads_batched=True, retain_graph=True)
        assert torch.equal(got, torch.stack([torch.autograd.grad(y, layer.weight, g, retain_graph=True)[0] for g in many]))
        dw, = torch.autograd.grad(y, layer.weight, torch._efficientzerotensor(tuple(y.shape), dtype=y.dtype, device="cuda"))
        assert not dw.any()
    grads = torch.func.grad(lambda w: fused_ops.embedding(tokens, w, 0.5, 3).float().sum())(layer.weight.detach())
    y = layer(tokens)
    assert torch.equal(grads, torch.autograd.grad(y, layer.weight, torch.ones_like(y))[0])


def test_tokens_and_tables_negated_on_reading():
    table, tokens = torch.randn(40, 16, device="cuda"), foreign(6)
    want = fused_ops.embedding(tokens, table, 3.0)
    assert torch.equal(fused_ops.embedding(torch._neg_view(-tokens), table, 3.0), want)
    assert torch.equal(fused_ops.embedding(tokens, torch._neg_view(-table), 3.0), want)
    leaf, dy = table.requires_grad_(True), torch.randn_like(want)
    y = fused_ops.embedding(tokens, leaf, 3.0)
    grads = [torch.autograd.grad(y, leaf, g, retain_graph=True)[0] for g in (dy, torch._neg_view(-dy))]
    assert torch.equal(*grads)


@pytest.mark.parametrize("back", [lambda t: t.short(), lambda t: t.double(), lambda t: t.cpu(), lambda t: t[:-1], lambda t: torch.cat([t, t])])
def test_saved_tokens_that_came_back_as_something_else(back):
    """What hooks hand back is refused where it is not the tokens any more, before anything is launched."""
    weight = torch.randn(40, 16, device="cuda", requires_grad=True)
    tokens = foreign(7, (50,))
    dy = torch.randn(50, 16, device="cuda")
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
        y = fused_ops.embedding(tokens, weight)
        with pytest.raises(RuntimeError, match="saved tokens"):
            torch.autograd.grad(y, weight, dy)


def test_saved_tokens_in_other_places_and_types():
    weight = torch.randn(40, 16, device="cuda", requires_grad=True)
    tokens = foreign(8, (50,))
    dy = torch.randn(50, 16, device="cuda")
    want, = torch.autograd.grad(fused_ops.embedding(tokens, weight), weight, dy)
    for pack, back in ((lambda t: t.cpu(), lambda t: t.cuda()), (lambda t: t.int(), lambda t: t), (lambda t: t.view(5, 10).t().contiguous(), lambda t: t.t()), (lambda t: -t, torch._neg_view)):
        with torch.autograd.graph.saved_tensors_hooks(pack, back):
            got, = torch.autograd.grad(fused_ops.embedding(tokens, weight), weight, dy)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_under_autocast(dtype):
    """Autocast has nothing to cast: the same kernels, bit for bit, in the table's type."""
    n, V, D = 9000, 40, 72
    g = torch.Generator("cuda").manual_seed(2)
    tokens = foreign(9, (n,))
    weight = torch.randn(V, D, generator=g, device="cuda").to(dtype).requires_grad_(True)
    dy = torch.randn(n, D, generator=g, device="cuda").to(dtype)
    want = fused_ops.embedding(tokens, weight, 3.0)
    grad, = torch.autograd.grad(want, weight, dy)
    for cast in (torch.bfloat16, torch.float16):
        with torch.autocast("cuda", cast):
            y = fused_ops.embedding(tokens, weight, 3.0)
            inside, = torch.autograd.grad(y, weight, dy, retain_graph=True)
        assert y.dtype == dtype and torch.equal(y, want) and type(y.grad_fn) is type(want.grad_fn)
        assert torch.equal(inside, grad) and torch.equal(torch.autograd.grad(y, weight, dy)[0], grad)


def test_offsets_beyond_32_bits():
    """A table, rows and a gradient of more than 2^32 elements each: the last rows of all three."""
    V, D, n = 550_007, 8200, 530_000
    weight = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    last = torch.arange(V - 50, V, device="cuda")
    weight[last] = torch.randn(50, D, device="cuda").bfloat16()
    weight.requires_grad_(True)
    tokens = torch.arange(n, device="cuda") % (V - 50)  # (each but once; the last 200 positions: the last 50 rows, four times each)
    tokens[-200:] = last.repeat(4)
    y = fused_ops.embedding(tokens, weight, 2.0)
    assert y.numel() > 1 << 32 and torch.equal(y[-200:], 2 * weight.detach()[last].repeat(4, 1)) and not y[:-200][:: 4099].any()
    dy = torch.ones_like(y)
    dy[-200:] = torch.randint(-3, 4, (200, D), device="cuda").bfloat16()
    dw, = torch.autograd.grad(y, weight, dy)
    assert torch.equal(dw[last], 2 * dy[-200:].view(4, 50, D).float().sum(0).bfloat16())
    assert dw[: n - 200 : 4099].eq(2).all() and not dw[n - 200 : V - 50].any()
