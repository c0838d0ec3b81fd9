"""The gated linear layer without a GPU: status codes of the C ABI (no device touched),
refusals of CPU tensors, module construction, shapes of fake tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

from ictc_o2_hp_b200 import GatedBlock, GatedLinear, RadialTrunk, ResidualBlock, _lib, dense


def test_cpu_tensors_and_bad_modules_are_refused():
    with pytest.raises(TypeError):
        dense.gated_linear(torch.randn(3, 4), torch.randn(10, 4))
    with pytest.raises(TypeError):
        GatedLinear(4, 5)(torch.randn(3, 4))
    for bad in ({"activation": "swish"}, {"hidden": 0}, {"in_features": 0}):
        with pytest.raises(ValueError):
            GatedLinear(**{"in_features": 4, "hidden": 5, **bad})


def test_parameters_are_those_of_a_linear_layer():
    torch.manual_seed(5)
    ours = GatedLinear(7, 3, activation="gelu")
    torch.manual_seed(5)
    theirs = torch.nn.Linear(7, 6)
    assert torch.equal(ours.weight, theirs.weight) and torch.equal(ours.bias, theirs.bias)
    ours.load_state_dict(theirs.state_dict())
    bare = GatedLinear(7, 3, bias=False)
    assert bare.bias is None and set(bare.state_dict()) == {"weight"}
    block = GatedBlock(8, 20)
    assert block.gated.weight.shape == (40, 8) and block.down.weight.shape == (8, 20)
    assert all(isinstance(b, GatedBlock) for b in RadialTrunk(4, 8, 2, gated=True).blocks)
    assert all(isinstance(b, ResidualBlock) for b in RadialTrunk(4, 8, 2).blocks)


def test_a_gated_layer_is_no_affine_layer_of_the_radial_product():
    from ictc_o2_hp_b200 import RadialUvuTensorProduct, UvuTensorProduct
    tp = UvuTensorProduct(4, 1, 2, parity="full", parity_in2="canonical", shared_weights=False)
    with pytest.raises((TypeError, ValueError)):
        RadialUvuTensorProduct(tp, GatedLinear(8, tp.weight_numel // 2))


def test_status_codes():
    lib = _lib.load()
    fwd, bwd = ctypes.c_size_t(), ctypes.c_size_t()
    some = ctypes.c_void_p(256)  # never read: every call below is refused or empty

    def forward(x=some, w=some, y=some, rows=8, inner=16, hidden=8, dtype=0, act=2, stride=16,
                space=some, size=1 << 30):
        return lib.ictc_o2_gated_linear_forward(x, stride, w, 16, None, y, None, space, size, rows,
                                                inner, hidden, dtype, act, None)

    assert forward(rows=0) == _lib.OK
    for bad in ({"rows": -1}, {"inner": 0}, {"hidden": 0}, {"dtype": 3}, {"act": 5}, {"act": -1},
                {"x": None}, {"w": None}, {"y": None}, {"stride": -1}):
        assert forward(**bad) == _lib.ERR_INVALID, bad
    assert forward(hidden=1 << 50) == _lib.ERR_UNSUPPORTED
    ws = lib.ictc_o2_gated_linear_workspace
    assert ws(8, 16, 8, 0, 0, 3, 0, 0, ctypes.byref(fwd), None) == _lib.ERR_INVALID
    assert ws(300, 200, 80, 0, 2, 3, 1, 0, ctypes.byref(fwd), ctypes.byref(bwd)) == _lib.OK
    assert bwd.value > 0
    assert ws(0, 200, 80, 0, 2, 3, 1, 0, ctypes.byref(fwd), ctypes.byref(bwd)) == _lib.OK
    assert fwd.value == bwd.value == 0

    def backward(preact=some, g=some, x=some, w=some, dw=some, space=some, size=1 << 30, rows=300,
                 stride=80):
        return lib.ictc_o2_gated_linear_backward(x, 200, w, 200, None, preact, g, stride, some, dw, some,
                                                 space, size, rows, 200, 80, 0, 2, None)

    for bad in ({"g": None}, {"x": None}, {"w": None}, {"rows": -1}, {"stride": -1}):
        assert backward(**bad) == _lib.ERR_INVALID, bad
    for bad in ({"space": None}, {"size": 16}, {"space": ctypes.c_void_p(264)}):
        assert backward(**bad) == _lib.ERR_WORKSPACE, bad


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("rows,inner,hidden", [(40000, 64, 32), (2000000, 64, 32), (1000000, 32, 16),
                                               (40000, 96, 64)])
def test_backward_workspace_holds_either_inner_product(rows, inner, hidden, dtype, size):
    """Operands off the 16-byte boundaries are copied where they are, one by one: x may stay in
    rows of its own distance, whose product needs other room than packed rows."""
    lib = _lib.load()
    fwd, bwd, inner_bytes = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.ictc_o2_gated_linear_workspace(rows, inner, hidden, dtype, 2, 0, 1, 0,
                                              ctypes.byref(fwd), ctypes.byref(bwd)) == _lib.OK

    def padded(n):
        return -(-n // 256) * 256

    def pitch(width):
        return -(-width * size // 64) * 64

    held = padded(rows * pitch(2 * hidden)) + padded(min(rows, 296) * 2 * hidden * 4)
    held += padded(rows * pitch(inner)) + padded(2 * hidden * pitch(inner))
    for layout in (1, 3):  # aligned rows; aligned and packed
        assert lib.ictc_o2_linear_workspace(rows, inner, 2 * hidden, dtype, 0, layout, 0,
                                            ctypes.byref(fwd), ctypes.byref(inner_bytes)) == _lib.OK
        assert bwd.value >= held + inner_bytes.value, layout


def test_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 7, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.empty(24, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = dense.gated_linear(x, w)
        assert y.shape == (3, 7, 12) and y.dtype == torch.bfloat16 and y.device.type == "cuda"
        with pytest.raises(ValueError):
            dense.gated_linear(x, w[:, :5])
