"""Gradient norm and clipping without a GPU: refusals, status codes of the C ABI (no device
touched), fake tensors."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from ictc_o2_hp_b200 import _lib, gradients


def test_cpu_tensors_and_bad_arguments_are_refused():
    g = torch.ones(4)
    for call in (lambda: gradients.grad_norm([g]), lambda: gradients.grad_norm(g),
                 lambda: gradients.clip_grads([g], 1.0), lambda: gradients.clip_grads([g], 1.0, out=[g])):
        with pytest.raises(TypeError):
            call()
    p = torch.nn.Parameter(g)
    p.grad = g.clone()
    with pytest.raises(TypeError):
        gradients.clip_grad_norm_([p], 1.0)
    assert torch.equal(p.grad, g)
    for call in (lambda: gradients.grad_norm([g], 3.0), lambda: gradients.clip_grads([g], -1.0),
                 lambda: gradients.clip_grads([g], math.nan),
                 lambda: gradients.clip_grads([], 1.0, out=[g])):
        with pytest.raises(ValueError):
            call()


def test_nothing_to_clip():
    p = torch.nn.Parameter(torch.ones(3))
    assert gradients.clip_grad_norm_([p], 1.0).item() == 0
    assert gradients.grad_norm([]).item() == 0
    assert gradients.clip_grads([], 1.0)[0] == []


def test_status_codes():
    lib = _lib.load()
    size = ctypes.c_size_t()
    assert lib.ictc_o2_grad_norm_workspace(-1, 0, ctypes.byref(size)) == _lib.ERR_INVALID
    assert lib.ictc_o2_grad_norm_workspace(3, 0, None) == _lib.ERR_INVALID
    assert lib.ictc_o2_grad_norm_workspace(3, 0, ctypes.byref(size)) == _lib.OK and size.value > 0
    pointers = (ctypes.c_void_p * 2)(4096, 8192)
    some = ctypes.c_void_p(4096)  # never read: every call below is refused

    def clip(grads=pointers, out=pointers, counts=(5, 6), dtypes=(0, 1), n=2, kind=0, most=1.0,
             norm=some):
        return lib.ictc_o2_clip_grads(
            grads, out, None if counts is None else (ctypes.c_int64 * 2)(*counts),
            None if dtypes is None else (ctypes.c_int32 * 2)(*dtypes), n, kind, most, norm, some,
            1 << 30, None)

    odd = (ctypes.c_void_p * 2)(4097, 8192)
    null = (ctypes.c_void_p * 2)(4096, None)
    for bad in ({"grads": None}, {"out": None}, {"counts": None}, {"dtypes": None}, {"norm": None},
                {"n": -1}, {"kind": 2}, {"most": -1.0}, {"most": math.nan}, {"counts": (5, -1)},
                {"counts": (5, 1 << 40)}, {"dtypes": (0, 3)}, {"grads": odd}, {"out": odd},
                {"grads": null}, {"out": null}):
        assert clip(**bad) == _lib.ERR_INVALID, bad


def test_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        grads = [torch.empty(s, device="cuda", dtype=torch.bfloat16) for s in (3, 70)]
        clipped, norm = gradients.clip_grads(grads, 1.0)
        assert [t.shape for t in clipped] == [t.shape for t in grads]
        assert norm.shape == () and norm.dtype == torch.float32
        assert gradients.grad_norm(grads).shape == ()
        out, _ = gradients.clip_grads(grads, 1.0, out=grads)
        assert all(o is g for o, g in zip(out, grads))
