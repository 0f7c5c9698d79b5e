"""The norm of many tensors together and clipping by it, against the formulas in 64 bits.

Squares and sums are float64: n of them are off by at most n 2^-52 of the sum, the norm by half of that and its rounding to
float32 (2^-24).  A clipped value is off by the factor's rounding to float32, the product's, and half a step of its type."""
import math

import pytest
import torch

from megalodon_amd import fused_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SIZES = {
    "one": [1],
    "few": [7, 1, 64, 1000],
    "chunks": [32768, 32767, 32769, 16384, 16385, 65536, 100001],
    "empty": [0, 5, 0],
    "many": [1 + 37 * i % 4001 for i in range(333)],
    "large": [3_000_001, 8_388_608],
}
DTYPES = {"f32": [torch.float32], "bf16": [torch.bfloat16], "f16": [torch.float16], "mixed": [torch.bfloat16, torch.float32, torch.float16]}


def tensors(sizes, dtypes, seed=0, size=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return [(size * torch.randn(n, generator=g, device="cuda")).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def norm64(ts, power):
    every = torch.cat([t.double().reshape(-1) for t in ts])
    if every.numel() == 0:
        return 0.0
    return (every.abs().max() if power == math.inf else every.square().sum().sqrt()).item()


def near(got, want):
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(got.item() - want) <= (U + 1e-9) * abs(want) + 2.0 ** -149


def clipped(t, norm, max_norm):
    """(value, bar)"""
    v = t.double() * min(1.0, max_norm / (norm + 1e-6))
    info = torch.finfo(t.dtype)
    return v, v.abs() * (3 * U + info.eps / 2) + info.smallest_normal * info.eps / 2 + 2.0 ** -149


def close(got, want):
    assert bool(((got.double() - want[0]).abs() <= want[1]).all())


@pytest.mark.parametrize("power", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", list(DTYPES))
@pytest.mark.parametrize("sizes", list(SIZES))
def test_sizes(sizes, dtypes, power):
    ts = tensors(SIZES[sizes], DTYPES[dtypes], 3)
    before = [t.clone() for t in ts]
    norm = norm64(ts, power)
    near(fused_ops.grad_norm(ts, power), norm)
    for max_norm in (norm / 3, norm * 2, 0.0):
        got, new = fused_ops.clip_grads(ts, max_norm, power)
        near(got, norm)
        for t, n, b in zip(ts, new, before):
            assert torch.equal(t, b) and n.dtype == t.dtype
            close(n, clipped(b, norm, max_norm))
            if max_norm > norm + 1e-5:
                assert torch.equal(n, b)
    again, _ = fused_ops.clip_grads(ts, norm / 3, power, out=ts)
    assert torch.equal(again, got)
    for t, b in zip(ts, before):
        close(t, clipped(b, norm, norm / 3))


@pytest.mark.parametrize("count", [159, 160, 161, 320, 500])
def test_as_many_as_launches_hold(count):
    ts = tensors([3] * count, DTYPES["mixed"], count)
    norm = norm64(ts, 2.0)
    near(fused_ops.grad_norm(ts), norm)
    _, new = fused_ops.clip_grads(ts, 1.0)
    for t, n in zip(ts, new):
        close(n, clipped(t, norm, 1.0))


@pytest.mark.parametrize("size", [1e30, 1e-30, 1e-42])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_squares_that_float32_does_not_hold(size, dtype):
    ts = tensors([1000, 70000], [dtype], 5, size)
    near(fused_ops.grad_norm(ts), norm64(ts, 2.0))
    _, new = fused_ops.clip_grads(ts, 1.0)
    for t, n in zip(ts, new):
        close(n, clipped(t, norm64(ts, 2.0), 1.0))


@pytest.mark.parametrize("power", [2.0, math.inf])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_values_that_are_not_finite(dtype, power):
    for value, place in ((math.inf, 0), (-math.inf, 40000), (math.nan, 33000), (math.nan, 65999)):
        ts = tensors([10, 66000], [dtype], 6)
        ts[1][place] = value
        norm = fused_ops.grad_norm(ts, power)
        assert norm.isnan() if math.isnan(value) else norm.isinf()
        got, new = fused_ops.clip_grads(ts, 1.0, power)
        if math.isnan(value):
            assert got.isnan() and all(n.isnan().all() for n in new)
        else:  # the factor is zero: finite values vanish, the infinity itself has no value
            assert not new[0].any() and new[1][place].isnan() and new[1].isnan().sum() == 1
    assert fused_ops.clip_grads([torch.tensor([math.inf], device="cuda", dtype=dtype)], math.inf, power)[1][0].isnan()


def test_views_and_orders():
    """Views at any element of a buffer whose other elements stay as they are; axes in any order; an axis of one element."""
    for dtype in (torch.bfloat16, torch.float32):
        buffer = torch.full((200_000,), 7.0, device="cuda", dtype=dtype)
        spans = [(1, 70_000), (70_003, 90_000), (90_001, 90_002), (100_005, 199_998)]
        ts = [buffer[a:b] for a, b in spans]
        kept = torch.ones(200_000, dtype=torch.bool, device="cuda")
        for t, (a, b) in zip(ts, spans):
            t.normal_()
            kept[a:b] = False
        before = [t.clone() for t in ts]
        norm = norm64(ts, 2.0)
        near(fused_ops.clip_grads(ts, 2.0, out=ts)[0], norm)
        for t, b in zip(ts, before):
            close(t, clipped(b, norm, 2.0))
        assert buffer[kept].eq(7).all()
        turned = [torch.randn(30, 50, 7, device="cuda").to(dtype).permute(2, 0, 1), torch.randn(9, 1, 4, device="cuda").to(dtype).transpose(0, 2)]
        before, norm = [t.clone() for t in turned], norm64(turned, 2.0)
        got, new = fused_ops.clip_grads(turned, 1.0)
        near(got, norm)
        for n, b in zip(new, before):
            close(n, clipped(b, norm, 1.0))


def test_parameters():
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(30, 40), torch.nn.Linear(40, 8)).cuda()
    net(torch.randn(16, 30, device="cuda"))[:, :4].square().sum().backward()
    net[0].bias.grad = None
    grads = [p.grad.clone() for p in net.parameters() if p.grad is not None]
    versions = [p.grad._version for p in net.parameters() if p.grad is not None]
    norm = fused_ops.clip_grad_norm_(net.parameters(), 0.25)
    near(norm, norm64(grads, 2.0))
    for p, b, v in zip((p for p in net.parameters() if p.grad is not None), grads, versions):
        close(p.grad, clipped(b, norm64(grads, 2.0), 0.25))
        assert p.grad._version > v
    assert abs(norm64([p.grad for p in net.parameters() if p.grad is not None], 2.0) - 0.25) < 1e-5
    one = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert fused_ops.clip_grad_norm_(one, 1.0) == 0
    one.grad = torch.tensor([3.0, 0.0, 4.0], device="cuda")
    assert fused_ops.clip_grad_norm_(one, 1.0) == 5 and abs(one.grad.norm().item() - 1) < 1e-5
    assert fused_ops.grad_norm([]) == 0 and fused_ops.clip_grads([], 1.0)[1] == []


def test_captured():
    """In a graph whose replays follow new gradients, eager calls between them; another graph's calls in turn with it."""
    ts, others = tensors([50_000, 33, 7000] * 60, DTYPES["mixed"], 1), tensors([900_000], [torch.bfloat16], 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fused_ops.clip_grads(ts, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, results = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, what in zip(graphs, (ts, others)):
        with torch.cuda.graph(graph, stream=side):
            results.append(fused_ops.clip_grads(what, 1.0))
    for seed in range(4):
        for t in ts + others:
            t.normal_().mul_(0.5 ** seed)
        want = [fused_ops.clip_grads(what, 1.0) for what in (ts, others)]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (n, new), (m, old) in zip(results, want):
            assert torch.equal(n, m) and all(torch.equal(a, b) for a, b in zip(new, old))


def test_other_streams():
    sets = [tensors([400_000, 17], DTYPES["mixed"], i) for i in range(2)]
    alone = [fused_ops.clip_grads(s, 1.0) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(5):
        for i, s in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got.append((i, fused_ops.clip_grads(s, 1.0)))
    torch.cuda.synchronize()
    for i, (n, new) in got:
        assert torch.equal(n, alone[i][0]) and all(torch.equal(a, b) for a, b in zip(new, alone[i][1]))


@pytest.mark.parametrize("bad", ["cpu", "double", "gaps", "expanded", "power", "max_norm", "nan", "sparse", "count", "shape", "type", "overlap", "twice", "shifted", "gradient"])
def test_refusals(bad):
    buffer = torch.randn(1000, device="cuda")
    ts, out, power, max_norm = [buffer[:300], buffer[500:900]], None, 2.0, 1.0
    if bad == "cpu": ts[1] = ts[1].cpu()
    if bad == "double": ts[1] = ts[1].double()
    if bad == "gaps": ts[1] = buffer.view(10, 100)[:, :50]
    if bad == "expanded": ts[1] = buffer[:1].expand(9)
    if bad == "power": power = 1.0
    if bad == "max_norm": max_norm = -1.0
    if bad == "nan": max_norm = math.nan
    if bad == "sparse": ts[1] = torch.eye(3, device="cuda").to_sparse()
    if bad == "count": out = [torch.empty_like(ts[0])]
    if bad == "shape": out = [torch.empty_like(ts[0]), torch.empty(20, 20, device="cuda")]
    if bad == "type": out = [torch.empty_like(ts[0]), torch.empty_like(ts[1], dtype=torch.bfloat16)]
    if bad == "overlap": out = [buffer[450:750], torch.empty_like(ts[1])]
    if bad == "twice": ts = out = [ts[0], ts[0]]
    if bad == "shifted": out = [buffer[1:301], buffer[500:900]]
    if bad == "gradient": ts[0] = ts[0].clone().requires_grad_(True)
    before = buffer.clone()
    with pytest.raises(RuntimeError):
        fused_ops.clip_grads(ts, max_norm, power, out=out)
    assert torch.equal(buffer, before)


def test_the_same_tensor_twice_counts_twice():
    t = torch.randn(500, device="cuda")
    near(fused_ops.grad_norm([t, t]), norm64([t, t], 2.0))
    norm, new = fused_ops.clip_grads([t, t[100:]], 1.0)
    near(norm, norm64([t, t[100:]], 2.0))
    close(new[1], clipped(t[100:], norm64([t, t[100:]], 2.0), 1.0))
