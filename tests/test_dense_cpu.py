"""The dense operators without a GPU: argument checks of the C ABI (status codes, no
device touched), refusals of CPU tensors, module construction."""

from __future__ import annotations

import ctypes

import pytest
import torch

from ictc_o2_hp_b200 import LayerNorm, Linear, RadialTrunk, ResidualBlock, _lib, dense


def test_cpu_tensors_are_refused():
    x, w = torch.randn(3, 4), torch.randn(5, 4)
    with pytest.raises(TypeError):
        dense.linear(x, w)
    with pytest.raises(TypeError):
        dense.layer_norm(x)
    with pytest.raises(TypeError):
        Linear(4, 5)(x)


def test_modules_refuse_bad_arguments():
    with pytest.raises(ValueError):
        LayerNorm(0)
    with pytest.raises(ValueError):
        Linear(4, 5, activation="swish")
    with pytest.raises(ValueError):
        ResidualBlock(4, activation="swish")
    with pytest.raises(ValueError):
        RadialTrunk(4, 8, blocks=-1)


def test_parameters_are_those_of_the_torch_modules():
    torch.manual_seed(5)
    ours = Linear(7, 3, activation="gelu")
    torch.manual_seed(5)
    theirs = torch.nn.Linear(7, 3)
    assert {k: v.shape for k, v in ours.state_dict().items()} == \
        {k: v.shape for k, v in theirs.state_dict().items()}
    assert torch.equal(ours.weight, theirs.weight)
    norm = LayerNorm(6)
    norm.load_state_dict(torch.nn.LayerNorm(6).state_dict())
    assert LayerNorm(6, affine=False).weight is None and LayerNorm(6, bias=False).bias is None


def test_layer_norm_status_codes():
    lib = _lib.load()
    size = ctypes.c_size_t()
    some = ctypes.c_void_p(64)  # never read: every call below is refused or empty

    def forward(x=some, y=some, rows=4, width=8, eps=1e-5, dtype=0, pdtype=0, mean=None,
                stride=8):
        return lib.ictc_o2_layer_norm_forward(x, stride, None, None, y, mean, None, rows, width,
                                              eps, dtype, pdtype, None)

    assert forward(rows=0) == _lib.OK
    for bad in ({"rows": -1}, {"width": 0}, {"dtype": 7}, {"pdtype": 1}, {"dtype": 1, "pdtype": 2},
                {"x": None}, {"y": None}, {"mean": some}, {"eps": -1.0}, {"eps": float("nan")},
                {"stride": -8}):
        assert forward(**bad) == _lib.ERR_INVALID, bad
    assert lib.ictc_o2_layer_norm_workspace(4, 8, 0, 0, None) == _lib.ERR_INVALID
    assert lib.ictc_o2_layer_norm_workspace(4, 8, 0, 0, ctypes.byref(size)) == _lib.OK
    assert size.value >= 2 * 8 * 4
    args = [some, 8, None, some, some, some, 8, some, some, some]
    assert lib.ictc_o2_layer_norm_backward(*args, None, 0, 4, 8, 0, 0, None) == _lib.ERR_WORKSPACE
    assert lib.ictc_o2_layer_norm_backward(*args, None, 0, -4, 8, 0, 0, None) == _lib.ERR_INVALID
    args[3] = None
    assert lib.ictc_o2_layer_norm_backward(*args, some, 1 << 20, 4, 8, 0, 0, None) == \
        _lib.ERR_INVALID


def test_linear_status_codes():
    lib = _lib.load()
    fwd, bwd = ctypes.c_size_t(), ctypes.c_size_t()
    some = ctypes.c_void_p(256)

    def forward(x=some, w=some, y=some, rows=8, inner=16, outer=8, dtype=0, act=0, stride=16):
        return lib.ictc_o2_linear_forward(x, stride, w, 16, None, None, 0, y, None, None, 0, rows,
                                          inner, outer, dtype, act, None)

    assert forward(rows=0) == _lib.OK
    for bad in ({"rows": -1}, {"inner": 0}, {"outer": 0}, {"dtype": 3}, {"act": 5}, {"act": -1},
                {"x": None}, {"w": None}, {"y": None}, {"stride": -1}):
        assert forward(**bad) == _lib.ERR_INVALID, bad
    ws = lib.ictc_o2_linear_workspace
    assert ws(8, 16, 8, 0, 0, 3, 0, ctypes.byref(fwd), None) == _lib.ERR_INVALID
    assert ws(8, 16, 8, 0, 2, 3, 0, ctypes.byref(fwd), ctypes.byref(bwd)) == _lib.OK
    assert fwd.value == 0 and bwd.value > 0

    def backward(preact=some, g=some, x=some, w=some, dw=some, space=some, size=1 << 30, act=2,
                 rows=8):
        return lib.ictc_o2_linear_backward(x, 16, w, 16, preact, g, 8, some, dw, some, space, size,
                                           rows, 16, 8, 0, act, None)

    for bad in ({"preact": None}, {"g": None}, {"x": None}, {"w": None}, {"rows": -1}):
        assert backward(**bad) == _lib.ERR_INVALID, bad
    for bad in ({"space": None}, {"size": 16}, {"space": ctypes.c_void_p(264)}):
        assert backward(**bad) == _lib.ERR_WORKSPACE, bad


def test_radial_product_refuses_an_activation():
    """The radial product reads weight and bias of its affine layer and nothing else."""
    from ictc_o2_hp_b200 import RadialUvuTensorProduct, UvuTensorProduct
    tp = UvuTensorProduct(4, 1, 2, parity="full", parity_in2="canonical", shared_weights=False)
    with pytest.raises(ValueError, match="activation"):
        RadialUvuTensorProduct(tp, Linear(8, tp.weight_numel, activation="silu"))
    model = RadialUvuTensorProduct(tp, Linear(8, tp.weight_numel))
    args = [torch.randn(3, d) for d in (tp.input1_dimension, tp.input2_dimension, 8)]
    model.radial_out.activation = "relu"
    with pytest.raises(ValueError, match="activation"):
        model(*args)
    model.radial_out = torch.nn.Linear(8, tp.weight_numel)
    with pytest.raises(TypeError):  # accepted; CPU tensors are refused by the kernels
        model(*args)


def test_radial_messages_refuse_an_activation():
    from types import SimpleNamespace

    from ictc_o2_hp_b200 import RadialUvuTensorProduct, UvuTensorProduct, graph
    tp = UvuTensorProduct(4, 1, 2, parity="full", parity_in2="canonical", shared_weights=False)
    model = RadialUvuTensorProduct(tp, Linear(8, tp.weight_numel))
    model.radial_out.activation = "gelu"
    edges = SimpleNamespace(num_nodes=2, num_edges=3, csr=lambda which: (None, None, None))
    with pytest.raises(ValueError, match="activation"):
        graph.radial_messages(model, torch.randn(2, tp.input1_dimension), edges,
                              torch.randn(3, tp.input2_dimension), torch.randn(3, 8))


def test_fake_tensors_go_through_the_custom_operators():
    """Shapes and types propagate without memory (the forward; autograd's engine wants a
    device of the tensors' type)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 7, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.empty(24, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        scale = torch.empty(24, device="cuda", requires_grad=True)
        y = dense.layer_norm(dense.linear(x, w, activation="silu"), scale)
        assert y.shape == (3, 7, 24) and y.dtype == torch.bfloat16 and y.device.type == "cuda"
        with pytest.raises(ValueError):
            dense.linear(x, w[:, :5])
