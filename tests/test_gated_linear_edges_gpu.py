"""The gated product at the ends of what its callers may do."""
import pytest
import torch

from megalodon_amd import fused_ops

pytestmark = pytest.mark.gpu


def operands(tokens, n_in, n_out, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + tokens + 7 * n_in + 11 * n_out)
    rows = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return (rows(tokens, n_in).to(dtype), (rows(n_out, n_in) / n_in ** 0.5).to(dtype), (rows(n_out, n_in) / n_in ** 0.5).to(dtype), rows(tokens, n_out).to(dtype))


def leaves_of(*tensors):
    return [t.clone().requires_grad_(True) for t in tensors]


# x (70, 72), w1 and w3 (36, 72), a and b (70, 40) float32: what a hook makes of the tensors that it recognises
SAVED = {
    "weights in another type": lambda t: t.float() if t.shape == (36, 72) else t,
    "weights in the other 16 bits": lambda t: t.half() if t.shape == (36, 72) else t,
    "rows in another type": lambda t: t.double() if t.shape == (70, 72) else t,
    "products in the other 16 bits": lambda t: t.half() if t.dtype == torch.float32 else t,
    "products in 64 bits": lambda t: t.double() if t.dtype == torch.float32 else t,
    "weights on the host": lambda t: t.cpu() if t.shape == (36, 72) else t,
    "rows on the host": lambda t: t.cpu() if t.shape == (70, 72) else t,
    "products on the host": lambda t: t.cpu() if t.dtype == torch.float32 else t,
    "fewer rows": lambda t: t[1:] if t.shape == (70, 72) else t,
    "narrower products": lambda t: t[:, :36] if t.dtype == torch.float32 else t,
}


@pytest.mark.parametrize("what", list(SAVED))
def test_saved_tensors_that_came_back_as_something_else(what):
    """What hooks hand back is refused where it is not what was saved any more, before anything is launched."""
    x, w1, w3, dh = operands(70, 72, 36, torch.bfloat16)
    leaves = leaves_of(x, w1, w3)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, SAVED[what]):
        h = fused_ops.gated_linear(*leaves)
        with pytest.raises(RuntimeError, match="saved tensor"):
            torch.autograd.grad(h, leaves, dh)


def test_saved_tensors_in_other_forms():
    """Negated on reading, in another layout: as they were."""
    x, w1, w3, dh = operands(70, 72, 36, torch.bfloat16)
    leaves = leaves_of(x, w1, w3)
    want = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
    for pack, back in ((lambda t: -t, torch._neg_view), (lambda t: t.t().contiguous(), lambda t: t.t())):
        with torch.autograd.graph.saved_tensors_hooks(pack, back):
            got = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def twice(fn, x, w1, w3, dh, us):
    """The gradients, and the gradients of (each times a u) by all four operands, once and once more."""
    grads = torch.autograd.grad(fn(x, w1, w3), (x, w1, w3), dh, create_graph=True)
    second = torch.autograd.grad(grads, (x, w1, w3, dh), us, create_graph=True)
    third = torch.autograd.grad(second, (x, w1, w3, dh), [torch.ones_like(t) for t in second])
    return grads, second, third


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [5, 100])
def test_gradients_that_are_differentiated_again(tokens, dtype):
    """The gradients are those without `create_graph`, bit for bit.  Theirs are the formula's in float32, rounded once: a rounding is off by eps / 2 of the
    value at most, float32's own part (sums of up to 100 numbers, a few steps an element) is below a 64th of that.  Those of the third order add up
    gradients of second ones that were rounded on the way: four of them."""
    x, w1, w3, dh = operands(tokens, 40, 24, dtype)
    us = [torch.randn_like(t) for t in (x, w1, w3)]
    leaves = leaves_of(x, w1, w3)
    once = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
    got = twice(fused_ops.gated_linear, *leaves_of(x, w1, w3, dh), us)
    assert all(torch.equal(g, w) for g, w in zip(got[0], once))
    wide = [t.double().cpu().requires_grad_(True) for t in (x, w1, w3, dh)]
    want = twice(lambda x, w1, w3: torch.nn.functional.silu(x @ w1.t()) * (x @ w3.t()), *wide, [u.double().cpu() for u in us])
    u = torch.finfo(dtype).eps / 2
    for order, times in ((1, 1), (2, 4)):
        for g, w in zip(got[order], want[order]):
            assert (g.double().cpu() - w).norm() <= times * u * (1 + 1 / 64) * w.norm()


def test_second_gradients_of_some_operands():
    """Only those that are asked for; operands that depend on each other; an output gradient that depends on one."""
    x, w1, w3, dh = operands(9, 16, 8, torch.bfloat16)
    us = [torch.randn_like(t) for t in (x, w1, w3)]

    def run(fn, cast, asked, tied):
        leaves = [cast(t).requires_grad_(i in asked) for i, t in enumerate((x, w1, w3))]
        w = leaves[1] * 2 if tied else leaves[2]
        h = fn(leaves[0], leaves[1], w)
        go = cast(dh) * leaves[1].detach().sum() if not tied else (leaves[1].sum() / 4) * cast(dh)
        first = torch.autograd.grad(h, [leaves[i] for i in asked], go, create_graph=True)
        loss = sum((f * cast(us[i])).sum() for f, i in zip(first, asked))
        if not loss.requires_grad:
            return []
        return torch.autograd.grad(loss, [leaves[i] for i in asked], allow_unused=True)

    for asked, tied in (([0], False), ([1], False), ([2], False), ([0, 2], False), ([0, 1], True)):
        got = run(fused_ops.gated_linear, lambda t: t.detach().clone(), asked, tied)
        want = run(lambda x, w1, w3: torch.nn.functional.silu(x @ w1.t()) * (x @ w3.t()), lambda t: t.detach().double().cpu(), asked, tied)
        for g, w in zip(got, want):
            if w is None or not w.any():
                assert g is None or not g.any()
            else:
                # (a handful of roundings of the program's own around the operator)
                assert (g.double().cpu() - w).norm() <= 8 * 2.0 ** -8 * w.norm()


def test_gradients_of_several_outputs_at_once():
    """One backward for many output gradients, and gradients that are zeros without memory."""
    x, w1, w3, _ = operands(40, 24, 16, torch.bfloat16)
    leaves = leaves_of(x, w1, w3)
    h = fused_ops.gated_linear(*leaves)
    many = torch.randn(3, 40, 16, device="cuda").bfloat16()
    got = torch.autograd.grad(h, leaves, many, is_grads_batched=True, retain_graph=True)
    wide = [t.double() for t in (x, w1, w3)]
    for i, dh in enumerate(many):
        exact = [t.clone().requires_grad_(True) for t in wide]
        want = torch.autograd.grad(torch.nn.functional.silu(exact[0] @ exact[1].t()) * (exact[0] @ exact[2].t()), exact, dh.double())
        for g, w in zip(got, want):
            assert (g[i].double() - w).norm() <= 2.0 ** -8 * (1 + 1 / 64) * w.norm()  # (one rounding of the float32 formula)
    none = torch.autograd.grad(h, leaves, torch._efficientzerotensor((40, 16), dtype=h.dtype, device="cuda"))
    assert all(g.shape == t.shape and not g.any() for g, t in zip(none, leaves))


@pytest.mark.parametrize("asked", [(1, 2), (2,)])
def test_weight_gradients_of_many_launches(asked):
    """Rows of 2^20 elements: 768 tokens to a launch.  The weights' gradients are summed in float32 through all launches and rounded once: whole numbers
    whose sums are below 2^24 come out as their sum's rounding."""
    tokens, n_in, n_out = 3 * 768 + 41, 1 << 20, 5
    g = torch.Generator("cuda").manual_seed(3)
    # a = 0 (silu = 0, silu' = 1/2), b = 2^b: da = dh 2^b / 2, db = 0 ... and with w1 of the first feature, where a is large: silu(a) = a
    x = torch.randint(0, 2, (tokens, n_in), generator=g, device="cuda", dtype=torch.int8).bfloat16()
    x[:, 0] = 1
    w1, w3 = torch.zeros(n_out, n_in, device="cuda").bfloat16(), torch.zeros(n_out, n_in, device="cuda").bfloat16()
    w1[:, 0], w3[:, 0] = 64.0, 1.0  # a = 64, silu(a) = 64 and silu'(a) = 1 in float32, b = 1
    dh = torch.randint(1, 4, (tokens, n_out), generator=g, device="cuda").bfloat16()
    leaves = [x, *(w.requires_grad_(i in asked) for i, w in ((1, w1), (2, w3)))]
    h = fused_ops.gated_linear(*leaves)
    assert torch.equal(h, torch.full_like(h, 64.0))
    grads = torch.autograd.grad(h, [leaves[i] for i in asked], dh)
    for i, got in zip(asked, grads):
        want = torch.zeros(n_out, n_in, dtype=torch.float64, device="cuda")
        for at in range(0, tokens, 256):
            want += (dh[at:at + 256].double() * (1 if i == 1 else 64)).t() @ x[at:at + 256].double()
        assert want.max() < 1 << 24 and (want.bfloat16().double() != want).any()
        assert torch.equal(got, want.float().bfloat16())


@pytest.mark.parametrize("tokens", [9, 64, 70, 300])
def test_float16_gradients_out_of_range(tokens):
    """The gradients of a and b are float16 numbers on their way: where one is beyond 65504, its token's dx and its feature's dw are not finite, as in a network of
    separate layers, never finite and wrong.  All others are the formula's."""
    n_in, n_out = 64, 40
    x, w1, w3, dh = operands(tokens, n_in, n_out, torch.float16)
    x[3], w3[5] = 1.0, 2.0  # b = 128 there, a = -64 .. 64
    w1[5] = 1 / 16  # a = 4: silu(a) = 3.93, silu' = 1.05; da = 1.05 * 128 dh, db = 3.93 dh
    dh[:, 5] = 0
    dh[3, 5] = 2000.0  # da = 2.7e5, db = 7900
    leaves = leaves_of(x, w1, w3)
    dx, d1, d3 = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
    others = [i for i in range(tokens) if i != 3]
    assert not dx[3].isfinite().any() and not d1[5].isfinite().any()
    assert dx[others].isfinite().all() and d3.isfinite().all() and d1[[i for i in range(n_out) if i != 5]].isfinite().all()
    dh[3, 5] = 400.0  # da = 54000: a float16 number
    got = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
    wide = [t.double().requires_grad_(True) for t in (x, w1, w3)]
    want = torch.autograd.grad(torch.nn.functional.silu(wide[0] @ wide[1].t()) * (wide[0] @ wide[2].t()), wide, dh.double())
    for g, w in zip(got, want):
        assert g.isfinite().all() and (g.double() - w).norm() <= 3 * 2.0 ** -11 * w.norm()  # (da, db, the result)


@pytest.mark.parametrize("tokens", [40, 200])
def test_small_float16_gradients(tokens):
    """Below 2^-14 float16 numbers lie 2^-24 apart: da and db, and with two terms what they leave, are off by 2^-25 at most, beside half a step."""
    x, w1, w3, dh = operands(tokens, 64, 40, torch.float16)
    dh = dh * 2.0 ** -13
    leaves = leaves_of(x, w1, w3)
    got = torch.autograd.grad(fused_ops.gated_linear(*leaves), leaves, dh)
    x, w1, w3, dh = (t.double() for t in (x, w1, w3, dh))
    a, b = x @ w1.t(), x @ w3.t()
    s = torch.sigmoid(a)
    da, db = dh * b * s * (1 + a * (1 - s)), dh * a * s
    u, least = 2.0 ** -11, 2.0 ** -25
    off = lambda t: t.abs() * (u + 2.0 ** -16) + least  # (2^-16: float32's part, exp among it)
    ea, eb = off(da), off(db)
    for g, w, e in ((got[0], da @ w1 + db @ w3, ea @ w1.abs() + eb @ w3.abs()), (got[1], da.t() @ x, ea.t() @ x.abs()), (got[2], db.t() @ x, eb.t() @ x.abs())):
        assert ((g.double() - w).abs() <= e * 1.01 + (w.abs() + e) * u + least).all()


def test_gradients_under_autocast():
    """Autocast has nothing to cast in them: the kernels' gradients, and their own in float32, bit for bit."""
    x, w1, w3, dh = operands(90, 40, 24, torch.bfloat16)
    us = [torch.randn_like(t) for t in (x, w1, w3)]

    def run():
        leaves = leaves_of(x, w1, w3, dh)
        h = fused_ops.gated_linear(*leaves[:3])

        def grads():
            once = torch.autograd.grad(h, leaves[:3], dh, retain_graph=True)
            again = torch.autograd.grad(h, leaves[:3], leaves[3], create_graph=True)
            many = torch.autograd.grad(h, leaves[:3], torch.stack([dh, -dh]), is_grads_batched=True, retain_graph=True)
            return [*once, *again, *many, *torch.autograd.grad(again, leaves, us)]
        return grads

    want = run()()
    grads = run()
    with torch.autocast("cuda", torch.float16):
        got = grads()
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_offsets_beyond_32_bits():
    """h, the kept products and the output gradient of more than 2^32 elements: the last tokens' rows are those of the same tokens alone."""
    tokens, n_in, n_out, part = 262_200, 72, 16_400, 300
    x, w1, w3, _ = operands(tokens, n_in, n_out, torch.bfloat16)
    leaves = leaves_of(x, w1, w3)
    h = fused_ops.gated_linear(*leaves, torch.bfloat16)
    assert h.numel() > 1 << 32
    dh = torch.zeros_like(h)
    dh[-part:] = torch.randn(part, n_out, device="cuda").bfloat16()
    dx, d1, d3 = torch.autograd.grad(h, leaves, dh)
    some = leaves_of(x[-part:], w1, w3)
    few = fused_ops.gated_linear(*some, torch.bfloat16)
    assert not dx[:-part].any()
    # the same formula, roundings that fall the other way where sums run in another order: two of them for h, four for the gradients
    for got, want, times in ((h[-part:], few, 2), *zip((dx[-part:], d1, d3), torch.autograd.grad(few, some, dh[-part:]), (4, 4, 4))):
        assert (got.double() - want.double()).norm() <= times * 2.0 ** -8 * want.double().norm()
