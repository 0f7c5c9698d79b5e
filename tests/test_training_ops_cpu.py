"""What the embedding, the gated product and the gradients' norm refuse before any launch (no GPU needed)."""
import ctypes
import types

import pytest
import torch

from megalodon_amd import _lib, fused_ops
from megalodon_amd.modules import Embedding, NormalizedFeedForwardNetwork

I64, PTR, NULL = ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p(0)
SOME = PTR(4096)  # an address that is never followed


class Tensors(ctypes.Structure):
    _fields_ = [("count", I64), ("start", PTR), ("to", PTR), ("size", PTR), ("dtype", PTR)]


def tensors(sizes, dtypes, pointers=None):
    n = len(sizes)
    keep = ((PTR * n)(*(pointers or [4096] * n)), (I64 * n)(*sizes), (ctypes.c_int32 * n)(*dtypes))
    t = Tensors(n, ctypes.addressof(keep[0]), ctypes.addressof(keep[0]), ctypes.addressof(keep[1]), ctypes.addressof(keep[2]))
    t.keep = keep
    return t


def refused(name, *args):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == 1
    return lib.mega_last_error()


@pytest.mark.parametrize("dtype,tokens,n_in,n_out,word", [
    (0, 8, 64, 64, b"bfloat16"), (3, 8, 64, 64, b"bfloat16"), (1, 0, 64, 64, b"sizes"), (1, 8, 0, 64, b"sizes"), (1, 8, 64, 0, b"sizes"),
    (1, 8, 64, -1, b"sizes"), (1, 1 << 31, 64, 64, b"sizes"), (1, 8, (1 << 20) + 1, 64, b"sizes"), (1, 8, 1 << 16, 1 << 13, b"sizes"),
])
def test_gated_linear_sizes(dtype, tokens, n_in, n_out, word):
    sizes = (ctypes.c_int(dtype), I64(tokens), I64(n_in), I64(n_out))
    assert word in refused("mega_gated_linear_fwd", SOME, SOME, SOME, *sizes, SOME, NULL, NULL, ctypes.c_int(dtype), SOME, NULL)
    assert word in refused("mega_gated_linear_bwd", SOME, SOME, SOME, SOME, SOME, SOME, ctypes.c_int(dtype), *sizes, SOME, SOME, SOME, SOME, NULL)
    fn = _lib.load().mega_gated_linear_workspace_bytes
    fn.restype = I64
    if word == b"sizes":
        assert fn(*sizes[1:], 0) == 0 and fn(*sizes[1:], 7) == 0


def test_gated_linear_pointers():
    sizes = (ctypes.c_int(1), I64(8), I64(64), I64(64))
    odd = PTR(4098)
    assert b"null" in refused("mega_gated_linear_fwd", NULL, SOME, SOME, *sizes, SOME, NULL, NULL, ctypes.c_int(1), NULL, NULL)
    assert b"null" in refused("mega_gated_linear_fwd", SOME, SOME, SOME, *sizes, SOME, SOME, NULL, ctypes.c_int(1), NULL, NULL)   # one product kept
    assert b"misaligned" in refused("mega_gated_linear_fwd", odd, SOME, SOME, *sizes, SOME, NULL, NULL, ctypes.c_int(1), NULL, NULL)
    assert b"kept" in refused("mega_gated_linear_fwd", SOME, SOME, SOME, *sizes, SOME, SOME, SOME, ctypes.c_int(2), NULL, NULL)
    assert b"null" in refused("mega_gated_linear_bwd", SOME, SOME, SOME, SOME, SOME, SOME, ctypes.c_int(0), *sizes, SOME, SOME, SOME, NULL, NULL)
    assert b"kept" in refused("mega_gated_linear_bwd", SOME, SOME, SOME, SOME, SOME, SOME, ctypes.c_int(2), *sizes, SOME, SOME, SOME, SOME, NULL)
    assert b"misaligned" in refused("mega_gated_linear_bwd", SOME, SOME, SOME, SOME, odd, SOME, ctypes.c_int(0), *sizes, SOME, SOME, SOME, SOME, NULL)
    assert b"misaligned" in refused("mega_gated_linear_bwd", SOME, SOME, SOME, SOME, SOME, SOME, ctypes.c_int(0), *sizes, SOME, SOME, SOME, odd, NULL)


@pytest.mark.parametrize("dtype,bits,n,vocab,width,word", [
    (3, 64, 4, 8, 8, b"tables"), (0, 16, 4, 8, 8, b"32 or 64"), (0, 64, -1, 8, 8, b"sizes"), (0, 64, 1 << 31, 8, 8, b"sizes"),
    (0, 64, 4, 0, 8, b"sizes"), (0, 64, 4, 1 << 31, 8, b"sizes"), (0, 64, 4, 8, 0, b"sizes"), (0, 64, 4, 8, (1 << 20) + 1, b"sizes"),
])
def test_embedding_sizes(dtype, bits, n, vocab, width, word):
    assert word in refused("mega_embedding_fwd", SOME, ctypes.c_int(bits), SOME, ctypes.c_int(dtype), I64(n), I64(vocab), I64(width), I64(width), ctypes.c_double(1), SOME, NULL)
    assert word in refused("mega_embedding_bwd", SOME, ctypes.c_int(dtype), SOME, ctypes.c_int(bits), I64(n), I64(vocab), I64(width), ctypes.c_double(1), I64(-1), SOME, SOME, NULL)


def test_embedding_pointers():
    sizes = (I64(4), I64(8), I64(8))
    assert b"null" in refused("mega_embedding_fwd", NULL, ctypes.c_int(64), SOME, ctypes.c_int(0), *sizes, I64(8), ctypes.c_double(1), SOME, NULL)
    assert b"null" in refused("mega_embedding_fwd", SOME, ctypes.c_int(64), SOME, ctypes.c_int(0), *sizes, I64(-8), ctypes.c_double(1), SOME, NULL)
    assert b"null" in refused("mega_embedding_bwd", SOME, ctypes.c_int(0), SOME, ctypes.c_int(64), *sizes, ctypes.c_double(1), I64(-1), SOME, NULL, NULL)
    assert b"misaligned" in refused("mega_embedding_bwd", SOME, ctypes.c_int(0), SOME, ctypes.c_int(64), *sizes, ctypes.c_double(1), I64(-1), SOME, PTR(4100), NULL)


def test_norm_and_clipping():
    good = tensors([10, 0], [0, 1], [4096, None])
    out, ws, one = SOME, SOME, ctypes.c_double(1)
    for bad in (tensors([10], [3]), tensors([-1], [0]), tensors([1 << 44], [0]), tensors([10], [0], [None]), tensors([10], [7])):
        refused("mega_tensors_norm", ctypes.byref(bad), 0, out, ws, NULL)
        refused("mega_tensors_clip", ctypes.byref(bad), one, ws, NULL)
    refused("mega_tensors_norm", NULL, 0, out, ws, NULL)
    assert b"kind" in refused("mega_tensors_norm", ctypes.byref(good), 2, out, ws, NULL)
    assert b"null" in refused("mega_tensors_norm", ctypes.byref(good), 0, NULL, ws, NULL)
    assert b"misaligned" in refused("mega_tensors_norm", ctypes.byref(good), 0, out, PTR(4100), NULL)
    for number in (-1.0, float("nan")):
        assert b"max_norm" in refused("mega_tensors_clip", ctypes.byref(good), ctypes.c_double(number), ws, NULL)
    none = Tensors(1, None, None, None, None)
    assert b"null" in refused("mega_tensors_norm", ctypes.byref(none), 0, out, ws, NULL)


def test_workspaces_of_the_norm():
    """One number for the norm and one for each workgroup: chunks of 16 KB, of 64 KB from 128 MiB in all, 2048 workgroups to a launch of 160 tensors."""
    fn = _lib.load().mega_tensors_workspace_bytes
    fn.restype = I64
    size = lambda sizes, dtypes: fn(ctypes.byref(tensors(sizes, dtypes))) // 8 - 1
    assert size([], []) == 0
    assert size([1, 0, 8192, 8193, 4096, 4097], [1, 1, 1, 1, 0, 0]) == 1 + 1 + 2 + 1 + 2
    assert size([1] * 160, [0] * 160) == 160 and size([1] * 321, [0] * 321) == 321
    assert size([1 << 25], [1]) == 2048 and size([1 << 30], [0]) == 2048
    assert size([1 << 26] + [1] * 160, [1] * 161) == 2048 + 1


def test_operators_refuse_host_tensors():
    """There is no CPU fallback."""
    with pytest.raises(RuntimeError, match="GPU"):
        fused_ops.embedding(torch.zeros(2, dtype=torch.long), torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="GPU"):
        Embedding(4, 8)(torch.zeros(2, dtype=torch.long))
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        fused_ops.gated_linear(x, w, w)
    for call in (lambda: fused_ops.grad_norm([w]), lambda: fused_ops.clip_grads([w], 1.0)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    p = torch.nn.Parameter(torch.zeros(3))
    assert fused_ops.clip_grad_norm_([p], 1.0) == 0
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="GPU"):
        fused_ops.clip_grad_norm_([p], 1.0)


def test_network_on_the_host_goes_where_it_did():
    ffn = NormalizedFeedForwardNetwork(16, 32, swiglu=True, fused_gate=True)
    assert not ffn.takes_fused_gate(torch.zeros(2, 16))
    assert set(ffn.state_dict()) == set(NormalizedFeedForwardNetwork(16, 32, swiglu=True).state_dict())


def test_embedding_from_a_table():
    table = torch.randn(5, 3)
    layer = Embedding.from_pretrained(table, padding_idx=-1, scale=2.0)
    assert layer.weight.data_ptr() == table.data_ptr() and not layer.weight.requires_grad
    assert (layer.num_embeddings, layer.embedding_dim, layer.padding_idx, layer.scale) == (5, 3, 4, 2.0)
    assert Embedding.from_pretrained(table, freeze=False).weight.requires_grad
    assert list(layer.state_dict()) == ["weight"]


def test_which_networks_take_the_fused_gate():
    """Not those whose sizes the operator refuses, and none that was pickled without the choice."""
    net = NormalizedFeedForwardNetwork(8, 16, swiglu=True, fused_gate=True)
    assert not net.takes_fused_gate(torch.zeros(1, 8))
    x = types.SimpleNamespace(is_cuda=True, dtype=torch.bfloat16)
    weight = lambda *shape: types.SimpleNamespace(shape=shape, dtype=torch.bfloat16)
    for (n_out, n_in), takes in (((16, 8), True), ((1 << 13, (1 << 16) - 64), True), ((1 << 13, 1 << 16), False), (((1 << 20) + 1, 8), False)):
        for layer in (net.fc1, net.fc3):
            layer._parameters["weight"] = weight(n_out, n_in)
        assert net.takes_fused_gate(x) == takes
    del net.__dict__["fused_gate"]
    assert net.fused_gate is False


def test_fused_gate_beside_layers_of_other_kinds():
    """A projection that is no `Linear`, and has no weight, goes where it went without the choice."""

    class Halves(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.parts = torch.nn.ModuleList([torch.nn.Linear(8, 8), torch.nn.Linear(8, 8)])

        def forward(self, x):
            return torch.cat([p(x) for p in self.parts], -1)

    net = NormalizedFeedForwardNetwork(8, 16, swiglu=True, fused_gate=True)
    net.fc1 = Halves()
    assert not net.takes_fused_gate(torch.zeros(1, 8))
    assert not net.takes_fused_gate(types.SimpleNamespace(is_cuda=True, dtype=torch.bfloat16))
