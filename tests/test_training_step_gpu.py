"""Embedding, a feed-forward network with the gate in its product, and clipping by the gradients' norm, as a training step has them."""
import pytest
import torch

from megalodon_amd import fused_ops
from megalodon_amd.modules import Embedding, MegaBlock, NormalizedFeedForwardNetwork

pytestmark = pytest.mark.gpu


def network(dtype, fused=True, vocab=500, dim=256, hidden=640):
    torch.manual_seed(3)
    embed = Embedding(vocab, dim, padding_idx=0, scale=dim ** 0.5, device="cuda", dtype=dtype)
    ffn = NormalizedFeedForwardNetwork(dim, hidden, swiglu=True, fused_gate=fused, init_std=dim ** -0.5).cuda().to(dtype)
    return torch.nn.ModuleList([embed, ffn])


def loss_of(net, tokens, target):
    x = net[0](tokens)
    return (net[1](x, x).float() - target.float()).square().mean()


def plain(net, tokens, target, max_norm):
    """The step in 64 bits: (loss, norm, clipped gradients by name)"""
    p = {n: t.detach().double().requires_grad_(True) for n, t in net.named_parameters()}
    w = p["0.weight"] * net[0].scale
    x = torch.where((tokens == 0)[..., None], w.detach()[tokens], w[tokens])
    mean, var = x.mean(-1, keepdim=True), x.var(-1, keepdim=True, unbiased=False)
    y = (x - mean) * (var + 1e-5).rsqrt() * (p["1.norm.weight"] + 1) + p["1.norm.bias"]
    h = torch.nn.functional.silu(y @ p["1.fc1.weight"].t()) * (y @ p["1.fc3.weight"].t())
    loss = (h @ p["1.fc2.weight"].t() + x - target.double()).square().mean()
    loss.backward()
    grads = {n: t.grad for n, t in p.items()}
    norm = sum(g.square().sum() for g in grads.values()).sqrt()
    return loss, norm, {n: g * min(1.0, max_norm / (norm + 1e-6)) for n, g in grads.items()}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 5), (3, 127), (1, 2048)])
def test_step(shape, dtype):
    net = network(dtype)
    g = torch.Generator("cuda").manual_seed(sum(shape))
    tokens = torch.randint(0, 500, shape, generator=g, device="cuda")
    tokens[:, -2:] = 0
    target = torch.randn(*shape, 256, generator=g, device="cuda").to(dtype)
    want_loss, want_norm, want = plain(net, tokens, target, 0.01)
    loss = loss_of(net, tokens, target)
    (loss * 16).backward()  # (float16's gradients are scaled, and so is the bound)
    norm = fused_ops.clip_grad_norm_(net.parameters(), 0.16)
    assert abs(loss.item() - want_loss.item()) <= 2e-2 * want_loss.item()
    assert abs(norm.item() / 16 - want_norm.item()) <= 2e-2 * want_norm.item()
    for n, t in net.named_parameters():
        assert (t.grad.double() / 16 - want[n]).norm() <= 3e-2 * want[n].norm(), n
    assert not net[0].weight.grad[0].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_network_with_and_without_the_fused_gate(dtype):
    """Both forms are within their roundings of each other, forward and gradients; layers with hooks, float32 and single rows go where they did."""
    fused, apart = network(dtype, True)[1], network(dtype, False)[1]
    for rows in (1, 40, 700):
        x = torch.randn(rows, 256, device="cuda").to(dtype)
        results = []
        for ffn in (fused, apart):
            leaf = x.clone().requires_grad_(True)
            y = ffn(leaf, leaf)
            y.backward(torch.ones_like(y))
            results.append([y.detach(), leaf.grad] + [p.grad for p in ffn.parameters()])
            ffn.zero_grad()
        for a, b in zip(*results):
            assert (a.double() - b.double()).norm() <= 6 * torch.finfo(dtype).eps * b.double().norm()
    seen = []
    handle = fused.fc1.register_forward_hook(lambda *a: seen.append(1))
    with torch.no_grad():  # (with gradients the two layers' products are one node, hooks or not)
        assert torch.equal(fused(x, x), apart(x, x)) and seen
    assert torch.equal(fused(x, x), apart(x, x))
    handle.remove()
    fused.float(), apart.float()
    assert torch.equal(fused(x.float(), x.float()), apart(x.float(), x.float()))


def test_block_with_the_fused_gate():
    """The block passes the choice on; its results are those of the block without it up to roundings."""
    blocks = []
    for fused in (True, False):
        torch.manual_seed(1)
        blocks.append(MegaBlock(256, 128, 512, 2, 16, 64, 704, 8, fused_gate=fused).cuda().bfloat16())
    assert blocks[0].nffn.fused_gate and not blocks[1].nffn.fused_gate
    x = torch.randn(2, 128, 256, device="cuda").bfloat16()
    with torch.no_grad():
        a, b = (block(x)[0].double() for block in blocks)
    assert (a - b).norm() <= 2.0 ** -7 * b.norm()


def test_captured_step():
    """A whole step in a graph, replayed on new tokens with the program's own steps between the replays."""
    net = network(torch.bfloat16)
    params = list(net.parameters())
    tokens, target = torch.randint(0, 500, (4, 200), device="cuda"), torch.randn(4, 200, 256, device="cuda").bfloat16()

    def step():
        grads = torch.autograd.grad(loss_of(net, tokens, target), params)
        norm, clipped = fused_ops.clip_grads(grads, 0.05)
        return [norm, *clipped]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for _ in range(3):
        tokens.random_(0, 500)
        target.normal_()
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert (o.double() - w.double()).norm() <= 1e-3 * w.double().norm()
