"""Dense operators around the tensor products: layer norm, the linear layer with bias,
activation and residual in its epilogue, and the gated linear layer, forward and backward
on the GPU.

The reference leaves the radial network and the node networks to PyTorch
(src/ictc_o2_hp/radial_uvu.py:21-66 takes only its last affine layer); these are the
pieces such networks are made of:

    y = layer_norm(x, weight, bias)                        # over the last dimension
    y = linear(x, weight, bias, activation="silu")         # act(x W^T + b)
    y = linear(h, weight, bias, residual=x)                # h W^T + b + x
    y = gated_linear(x, weight, bias, activation="silu")   # act(x Wg^T + bg) (x Wu^T + bu)

``LayerNorm`` and ``Linear`` are the modules (parameters and state_dict keys of their
``torch.nn`` namesakes), ``GatedLinear`` that of the gated layer; ``ResidualBlock``,
``GatedBlock`` and ``RadialTrunk`` run them together.
Operands are CUDA float32, bfloat16 or float16 tensors of one type (layer norm
parameters may stay float32 beside 16-bit inputs); sums, statistics and activations are
float32.  Second derivatives (force losses) are available for all of them.

Like the products, these raise for CPU tensors and other types instead of falling back.
"""

from __future__ import annotations

import ctypes
import importlib.util
import math
from pathlib import Path

import torch
from torch import Tensor

from . import _lib
from .ops import NAMESPACE

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}

# The autograd layer (argument checks, allocation, autograd nodes) is an extension module
# beside the kernel library: csrc/dense_autograd.cpp.
AUTOGRAD = Path(__file__).resolve().parent / "_lib" / "_dense_autograd.so"
_native = None


def _load():
    """Loads the extension module once and binds it to the kernel library."""
    global _native
    if _native is None:
        if not AUTOGRAD.exists():
            raise RuntimeError(f"{AUTOGRAD} is missing: build it with `python -m "
                               "ictc_o2_hp_b200.build` (the dense operators have no fallback)")
        spec = importlib.util.spec_from_file_location("_dense_autograd", AUTOGRAD)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        lib = _lib.load()
        names = ("ictc_o2_last_error", "ictc_o2_layer_norm_forward", "ictc_o2_layer_norm_workspace",
                 "ictc_o2_layer_norm_backward", "ictc_o2_linear_workspace",
                 "ictc_o2_linear_forward", "ictc_o2_linear_backward",
                 "ictc_o2_gated_linear_workspace", "ictc_o2_gated_linear_forward",
                 "ictc_o2_gated_linear_backward", "ictc_o2_gated_linear_keeps")
        module.bind(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names))
        module.bind_operators(_norm_op, _norm_grad_op, _linear_op, _linear_grad_op, _gated_op,
                              _gated_grad_op)
        _native = module
    return _native


# ------------------- custom operators, for torch.compile and whatever watches the dispatcher


@torch.library.custom_op(f"{NAMESPACE}::layer_norm_forward", mutates_args=())
def _norm_op(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float
             ) -> tuple[Tensor, Tensor, Tensor]:
    return _load().norm_forward(x, weight, bias, eps)


@_norm_op.register_fake
def _norm_op_fake(x, weight, bias, eps):
    rows = math.prod(x.shape[:-1])
    stat = x.new_empty(rows, dtype=torch.float32)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device), stat, torch.empty_like(stat)


@torch.library.custom_op(f"{NAMESPACE}::layer_norm_backward", mutates_args=())
def _norm_grad_op(x: Tensor, weight: Tensor | None, mean: Tensor, rstd: Tensor, grad: Tensor,
                  float_params: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _load().norm_backward(x, weight, mean, rstd, grad, float_params)


@_norm_grad_op.register_fake
def _norm_grad_op_fake(x, weight, mean, rstd, grad, float_params):
    dw = x.new_empty(x.shape[-1], dtype=torch.float32 if float_params else x.dtype)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device), dw, torch.empty_like(dw)


def _norm_op_setup(ctx, inputs, output):
    x, weight, bias, _ = inputs
    ctx.save_for_backward(x, weight, output[1], output[2])
    ctx.pdtype = (weight if weight is not None else bias if bias is not None else x).dtype


def _norm_op_backward(ctx, grad, _mean_grad, _rstd_grad):
    x, weight, mean, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw, db = _norm_grad_op(x, weight, mean, rstd, grad, ctx.pdtype == torch.float32)
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None)


_norm_op.register_autograd(_norm_op_backward, setup_context=_norm_op_setup)


@torch.library.custom_op(f"{NAMESPACE}::linear_forward", mutates_args=())
def _linear_op(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, code: int,
               save: bool) -> tuple[Tensor, Tensor]:
    return _load().linear_forward(x, weight, bias, residual, code, save)


@_linear_op.register_fake
def _linear_op_fake(x, weight, bias, residual, code, save):
    n = weight.shape[0]
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    shape = (math.prod(x.shape[:-1]), n) if save else (0,)
    return y, x.new_empty(shape, dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::linear_backward", mutates_args=())
def _linear_grad_op(x: Tensor, weight: Tensor, preact: Tensor, grad: Tensor, code: int
                    ) -> tuple[Tensor, Tensor, Tensor]:
    return _load().linear_backward(x, weight, preact, grad, code)


@_linear_grad_op.register_fake
def _linear_grad_op_fake(x, weight, preact, grad, code):
    return (torch.empty(x.shape, dtype=x.dtype, device=x.device),
            torch.empty(weight.shape, dtype=x.dtype, device=x.device),
            weight.new_empty(weight.shape[0]))


def _linear_op_setup(ctx, inputs, output):
    x, weight, _, _, code, _ = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.code = code


def _linear_op_backward(ctx, grad, _preact_grad):
    x, weight, preact = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw, db = _linear_grad_op(x, weight, preact, grad, ctx.code)
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None,
            grad if need[3] else None, None, None)


_linear_op.register_autograd(_linear_op_backward, setup_context=_linear_op_setup)


@torch.library.custom_op(f"{NAMESPACE}::gated_linear_forward", mutates_args=())
def _gated_op(x: Tensor, weight: Tensor, bias: Tensor | None, code: int, save: bool
              ) -> tuple[Tensor, Tensor]:
    return _load().gated_forward(x, weight, bias, code, save)


@_gated_op.register_fake
def _gated_op_fake(x, weight, bias, code, save):
    y = torch.empty((*x.shape[:-1], weight.shape[0] // 2), dtype=x.dtype, device=x.device)
    shape = (math.prod(x.shape[:-1]), weight.shape[0]) if save else (0,)
    return y, x.new_empty(shape, dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::gated_linear_backward", mutates_args=())
def _gated_grad_op(x: Tensor, weight: Tensor, bias: Tensor | None, preact: Tensor, grad: Tensor,
                   code: int) -> tuple[Tensor, Tensor, Tensor]:
    return _load().gated_backward(x, weight, bias, preact, grad, code)


@_gated_grad_op.register_fake
def _gated_grad_op_fake(x, weight, bias, preact, grad, code):
    return _linear_grad_op_fake(x, weight, preact, grad, code)


def _gated_op_setup(ctx, inputs, output):
    x, weight, bias, code, _ = inputs
    ctx.save_for_backward(x, weight, bias, output[1])
    ctx.code = code


def _gated_op_backward(ctx, grad, _preact_grad):
    x, weight, bias, preact = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw, db = _gated_grad_op(x, weight, bias, preact, grad, ctx.code)
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None, None)


_gated_op.register_autograd(_gated_op_backward, setup_context=_gated_op_setup)


# ---------------------------------------------------------------------- functions


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None,
               eps: float = 1e-5) -> Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, with the
    biased variance.  weight and bias: [x.shape[-1]], of x's type or float32."""
    if torch.compiler.is_compiling():
        return _norm_op(x, weight, bias, eps)[0]
    return (_native or _load()).layer_norm(x, weight, bias, eps)


def _cast_mixed(tensors: list) -> list:
    """What csrc/dense_autograd.cpp does under autocast, where a compiler traces."""
    given = [t for t in tensors if t is not None]
    if torch.is_autocast_enabled("cuda") and len({t.dtype for t in given}) > 1 and all(
            t.is_cuda and t.dtype in (torch.float32, torch.bfloat16, torch.float16)
            for t in given):
        dtype = torch.get_autocast_dtype("cuda")
        return [t if t is None else t.to(dtype) for t in tensors]
    return tensors


def _activation_code(activation: str) -> int:
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return code


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str = "none",
           residual: Tensor | None = None) -> Tensor:
    """act(x weight^T + bias) + residual: x [..., in], weight [out, in], bias [out],
    residual [..., out]; activation one of ACTIVATIONS.  Under ``torch.autocast`` operands
    of different types are cast to its type (equal ones are computed in their own)."""
    code = _activation_code(activation)
    if torch.compiler.is_compiling():
        x, weight, bias, residual = _cast_mixed([x, weight, bias, residual])
        save = code != 0 and torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, weight, bias, residual))
        return _linear_op(x, weight, bias, residual, code, save)[0]
    return (_native or _load()).linear(x, weight, bias, residual, code)


def gated_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None,
                 activation: str = "silu") -> Tensor:
    """act(pg) * pu with (pg | pu) = x weight^T + bias: x [..., in], weight [2 hidden, in] and
    bias [2 hidden], the gate's rows first; the result is [..., hidden].  activation and
    autocast as in ``linear``."""
    code = _activation_code(activation)
    if torch.compiler.is_compiling():
        x, weight, bias = _cast_mixed([x, weight, bias])
        save = torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, weight, bias))
        if save and weight.dim() == 2:  # as ictc_o2_gated_linear_keeps, by the sizes
            sizes, block = (weight.shape[0] // 2, weight.shape[1]), 16 // x.element_size()
            save = any(s > 64 or s % block for s in sizes)
        return _gated_op(x, weight, bias, code, save)[0]
    return (_native or _load()).gated_linear(x, weight, bias, code)


# ----------------------------------------------------------------------- modules


class LayerNorm(torch.nn.Module):
    """Layer norm over the last dimension (`width` elements)."""

    def __init__(self, width: int, eps: float = 1e-5, affine: bool = True, bias: bool = True,
                 device=None, dtype=None):
        super().__init__()
        if int(width) < 1:
            raise ValueError("width must be >= 1")
        self.width, self.eps = int(width), float(eps)
        kw = {"device": device, "dtype": dtype}
        self.weight = torch.nn.Parameter(torch.ones(self.width, **kw)) if affine else None
        self.bias = torch.nn.Parameter(torch.zeros(self.width, **kw)) if affine and bias else None

    def forward(self, x: Tensor) -> Tensor:
        if x.shape[-1] != self.width:
            raise ValueError(f"the last dimension must be {self.width}, got {x.shape[-1]}")
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self) -> str:
        return f"{self.width}, eps={self.eps}, affine={self.weight is not None}"


class Linear(torch.nn.Linear):
    """``torch.nn.Linear`` (same parameters, initialisation and state_dict) with an
    activation and an optional residual in the product's epilogue.  Being a
    ``torch.nn.Linear``, one without activation also serves as the ``radial_out`` of
    ``RadialUvuTensorProduct``."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 activation: str = "none", device=None, dtype=None):
        _activation_code(activation)
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        self.activation = activation

    def forward(self, x: Tensor, residual: Tensor | None = None) -> Tensor:
        return linear(x, self.weight, self.bias, self.activation, residual)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"


class GatedLinear(torch.nn.Module):
    """act(x Wg^T + bg) * (x Wu^T + bu).  ``weight`` [2 hidden, in] and ``bias`` [2 hidden] hold
    the gate's rows, then the other's: the parameters, initialisation and state_dict of
    ``torch.nn.Linear(in_features, 2 * hidden)``."""

    def __init__(self, in_features: int, hidden: int, bias: bool = True,
                 activation: str = "silu", device=None, dtype=None):
        super().__init__()
        _activation_code(activation)
        if int(in_features) < 1 or int(hidden) < 1:
            raise ValueError("in_features and hidden must be >= 1")
        self.in_features, self.hidden = int(in_features), int(hidden)
        self.activation = activation
        layer = torch.nn.Linear(self.in_features, 2 * self.hidden, bias, device=device, dtype=dtype)
        self.weight = layer.weight
        self.register_parameter("bias", layer.bias)

    def forward(self, x: Tensor) -> Tensor:
        return gated_linear(x, self.weight, self.bias, self.activation)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, hidden={self.hidden}, "
                f"bias={self.bias is not None}, activation={self.activation}")


class ResidualBlock(torch.nn.Module):
    """x + down(act(up(norm(x)))): a pre-norm feed-forward block of three kernels."""

    def __init__(self, width: int, hidden: int | None = None, activation: str = "silu",
                 device=None, dtype=None):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        hidden = width if hidden is None else hidden
        self.norm = LayerNorm(width, **kw)
        self.up = Linear(width, hidden, activation=activation, **kw)
        self.down = Linear(hidden, width, **kw)

    def forward(self, x: Tensor) -> Tensor:
        return self.down(self.up(self.norm(x)), residual=x)


class GatedBlock(torch.nn.Module):
    """x + down(act(gate(z)) * up(z)) with z = norm(x): a pre-norm gated feed-forward block of
    three kernels.  ``gated`` holds both projections."""

    def __init__(self, width: int, hidden: int | None = None, activation: str = "silu",
                 device=None, dtype=None):
        super().__init__()
        kw = {"device": device, "dtype": dtype}
        hidden = width if hidden is None else hidden
        self.norm = LayerNorm(width, **kw)
        self.gated = GatedLinear(width, hidden, activation=activation, **kw)
        self.down = Linear(hidden, width, **kw)

    def forward(self, x: Tensor) -> Tensor:
        return self.down(self.gated(self.norm(x)), residual=x)


class RadialTrunk(torch.nn.Module):
    """Radial basis [..., in_features] to the hidden features [..., hidden] that
    ``RadialUvuTensorProduct`` takes: an embedding layer, residual blocks (gated ones with
    ``gated=True``) and a final layer norm."""

    def __init__(self, in_features: int, hidden: int, blocks: int = 1, activation: str = "silu",
                 device=None, dtype=None, gated: bool = False):
        super().__init__()
        if int(blocks) < 0:
            raise ValueError("blocks must be >= 0")
        kw = {"device": device, "dtype": dtype}
        self.embed = Linear(in_features, hidden, activation=activation, **kw)
        block = GatedBlock if gated else ResidualBlock
        self.blocks = torch.nn.ModuleList(
            block(hidden, activation=activation, **kw) for _ in range(int(blocks)))
        self.norm = LayerNorm(hidden, **kw)

    def forward(self, basis: Tensor) -> Tensor:
        h = self.embed(basis)
        for block in self.blocks:
            h = block(h)
        return self.norm(h)
