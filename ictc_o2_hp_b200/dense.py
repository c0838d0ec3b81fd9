"""Dense operators around the tensor products: layer norm and the linear layer with
bias, activation and residual in its epilogue, forward and backward on the GPU.

The reference leaves the radial network and the node networks to PyTorch
(src/ictc_o2_hp/radial_uvu.py:21-66 takes only its last affine layer); these are the
pieces such networks are made of:

    y = layer_norm(x, weight, bias)                        # over the last dimension
    y = linear(x, weight, bias, activation="silu")         # act(x W^T + b)
    y = linear(h, weight, bias, residual=x)                # h W^T + b + x

``LayerNorm`` and ``Linear`` are the modules (parameters and state_dict keys of their
``torch.nn`` namesakes), ``ResidualBlock`` and ``RadialTrunk`` run them together.
Operands are CUDA float32, bfloat16 or float16 tensors of one type (layer norm
parameters may stay float32 beside 16-bit inputs); sums, statistics and activations are
float32.  Second derivatives (force losses) are available for both.

Like the products, these raise for CPU tensors and other types instead of falling back.
"""

from __future__ import annotations

import math
from functools import lru_cache, wraps

import torch
from torch import Tensor

from . import _lib
from .ops import NAMESPACE

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


# ------------------------------------------------------------------------ checks


def _check_input(what: str, x: Tensor) -> None:
    if x.dtype not in _DTYPES or not x.is_cuda:
        raise TypeError(f"{what} runs only on CUDA float32, bfloat16 or float16 tensors (there is "
                        f"no CPU or other-dtype fallback); got {x.dtype} on {x.device}")


def _check_like(what: str, name: str, t: Tensor, x: Tensor, float32_too: bool = False) -> None:
    if t.device != x.device:
        raise ValueError(f"{what}: {name} is on {t.device}, the input on {x.device}")
    if t.dtype != x.dtype and not (float32_too and t.dtype == torch.float32):
        raise ValueError(f"{what}: {name} is {t.dtype}, the input {x.dtype}")


def _rows(t: Tensor) -> Tensor:
    """`t` as [rows, width] with unit stride inside a row; copies only when it must."""
    width = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), width)
    return t if width == 1 or t.stride(1) == 1 else t.contiguous()


def _on_device(run):
    """`run(x, ...)` with x's device current; the guard costs nothing when it already is."""
    @wraps(run)
    def guarded(x, *args):
        if torch.cuda.current_device() == x.device.index:
            return run(x, *args)
        with torch.cuda.device(x.device):
            return run(x, *args)
    return guarded


# Workspace sizes are a function of sizes, type and device alone.
_norm_workspace = lru_cache(maxsize=4096)(_lib.layer_norm_workspace)
_linear_workspace = lru_cache(maxsize=4096)(_lib.linear_workspace)


def _scratch(size: int, like: Tensor) -> Tensor | None:
    return like.new_empty(size, dtype=torch.uint8) if size else None


# -------------------------------------------------------------------- layer norm


@_on_device
def _norm_run(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float,
              stats: bool) -> tuple[Tensor, Tensor | None, Tensor | None]:
    rows = _rows(x)
    y = x.new_empty(x.shape)
    mean = rstd = None
    if stats:
        mean = x.new_empty(rows.shape[0], dtype=torch.float32)
        rstd = torch.empty_like(mean)
    params = weight if weight is not None else bias
    pcode = _DTYPES[(x if params is None else params).dtype]
    _lib.layer_norm_forward(rows, weight, bias, y, mean, rstd, eps, _DTYPES[x.dtype], pcode)
    return y, mean, rstd


@_on_device
def _norm_grad_run(x, weight, mean, rstd, grad, pdtype, need):
    """(dx, dweight, dbias), None where `need` is false; pdtype types the last two."""
    rows, g = _rows(x), _rows(grad)
    width = x.shape[-1]
    dx = x.new_empty(x.shape) if need[0] else None
    dw = x.new_empty(width, dtype=pdtype) if need[1] else None
    db = x.new_empty(width, dtype=pdtype) if need[2] else None
    code = _DTYPES[x.dtype]
    size = 0
    if need[1] or need[2]:
        size = _norm_workspace(rows.shape[0], width, code, x.device.index)
    _lib.layer_norm_backward(rows, weight, mean, rstd, g, dx, dw, db, _scratch(size, x), code,
                             _DTYPES[pdtype])
    return dx, dw, db


def _norm_grad_formula(x, weight, eps, grad):
    """The backward in differentiable PyTorch operations, for second derivatives."""
    xf, g = x.float(), grad.float()
    centred = xf - xf.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + eps)
    u = centred * rstd
    h = g if weight is None else g * weight.float()
    dx = rstd * (h - h.mean(-1, keepdim=True) - u * (h * u).mean(-1, keepdim=True))
    over = tuple(range(x.dim() - 1))
    return dx.to(x.dtype), (g * u).sum(over) if over else g * u, g.sum(over) if over else g


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _norm_run(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.eps = eps
        ctx.pdtype = (weight if weight is not None else bias if bias is not None else x).dtype
        return y

    @staticmethod
    def backward(ctx, grad):
        x, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        if torch.is_grad_enabled():
            dx, dw, db = _norm_grad_formula(x, weight, ctx.eps, grad)
            return (dx, dw.to(ctx.pdtype) if need[1] else None,
                    db.to(ctx.pdtype) if need[2] else None, None)
        return (*_norm_grad_run(x, weight, mean, rstd, grad, ctx.pdtype, need), None)


@torch.library.custom_op(f"{NAMESPACE}::layer_norm_forward", mutates_args=())
def _norm_op(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float
             ) -> tuple[Tensor, Tensor, Tensor]:
    return _norm_run(x, weight, bias, eps, True)


@_norm_op.register_fake
def _norm_op_fake(x, weight, bias, eps):
    rows = math.prod(x.shape[:-1])
    stat = x.new_empty(rows, dtype=torch.float32)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device), stat, torch.empty_like(stat)


@torch.library.custom_op(f"{NAMESPACE}::layer_norm_backward", mutates_args=())
def _norm_grad_op(x: Tensor, weight: Tensor | None, mean: Tensor, rstd: Tensor, grad: Tensor,
                  float_params: bool) -> tuple[Tensor, Tensor, Tensor]:
    pdtype = torch.float32 if float_params else x.dtype
    return _norm_grad_run(x, weight, mean, rstd, grad, pdtype, (True, True, True))


@_norm_grad_op.register_fake
def _norm_grad_op_fake(x, weight, mean, rstd, grad, float_params):
    dw = x.new_empty(x.shape[-1], dtype=torch.float32 if float_params else x.dtype)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device), dw, torch.empty_like(dw)


def _norm_op_setup(ctx, inputs, output):
    x, weight, bias, eps = inputs
    ctx.save_for_backward(x, weight, output[1], output[2])
    ctx.eps = eps
    ctx.pdtype = (weight if weight is not None else bias if bias is not None else x).dtype


def _norm_op_backward(ctx, grad, _mean_grad, _rstd_grad):
    x, weight, mean, rstd = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dw, db = _norm_grad_op(x, weight, mean, rstd, grad, ctx.pdtype == torch.float32)
    return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None, None)


_norm_op.register_autograd(_norm_op_backward, setup_context=_norm_op_setup)


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None,
               eps: float = 1e-5) -> Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, with the
    biased variance.  weight and bias: [x.shape[-1]], of x's type or float32."""
    what = "layer_norm"
    _check_input(what, x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm needs a last dimension of at least one element")
    if not eps >= 0:
        raise ValueError("eps must be >= 0")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check_like(what, name, t, x, float32_too=True)
            if t.shape != x.shape[-1:]:
                raise ValueError(f"layer_norm: {name} must have shape {tuple(x.shape[-1:])}, "
                                 f"got {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("layer_norm: weight and bias must have the same type")
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    if torch.compiler.is_compiling():
        return _norm_op(x, weight, bias, eps)[0]
    if torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad) or
            (bias is not None and bias.requires_grad)):
        return _LayerNormFunction.apply(x, weight, bias, eps)
    return _norm_run(x, weight, bias, eps, False)[0]


# ------------------------------------------------------------------------ linear


_ALIGNED, _PACKED = 1, 2  # layout flags of the C ABI


def _layout(x, w, g=None) -> int:
    """What the operands' row starts allow (all [rows, width], unit stride in a row)."""
    block = 16 // x.element_size()
    packed = aligned = True
    for t in (x, g):
        if t is not None:
            start = t.data_ptr() % 16 == 0
            rows = t.stride(0)
            packed = packed and start and (rows == t.shape[1] or t.shape[0] <= 1)
            aligned = aligned and start and rows % block == 0
    aligned = aligned and w.data_ptr() % 16 == 0 and w.stride(0) % block == 0
    return (_ALIGNED if aligned else 0) | (_PACKED if packed else 0)


@_on_device
def _linear_run(x, weight, bias, residual, code, save) -> tuple[Tensor, Tensor | None]:
    """(y, p): p, the float32 value before the activation, only when `save`."""
    rows, w = _rows(x), _rows(weight)
    r = None if residual is None else _rows(residual)
    m, n = rows.shape[0], w.shape[0]
    y = x.new_empty((*x.shape[:-1], n))
    preact = x.new_empty((m, n), dtype=torch.float32) if save else None
    dcode = _DTYPES[x.dtype]
    size = _linear_workspace(m, rows.shape[1], n, dcode, code, _layout(rows, w),
                             x.device.index)[0]
    _lib.linear_forward(rows, w, bias, r, y, preact, _scratch(size, x), n, dcode, code)
    return y, preact


@_on_device
def _linear_grad_run(x, weight, preact, grad, code, need):
    """(dx, dweight, dbias), None where `need` is false."""
    rows, w, g = _rows(x), _rows(weight), _rows(grad)
    m, k = rows.shape
    n = w.shape[0]
    dx = x.new_empty(x.shape) if need[0] else None
    dw = x.new_empty((n, k)) if need[1] else None
    db = x.new_empty(n) if need[2] else None
    dcode = _DTYPES[x.dtype]
    size = _linear_workspace(m, k, n, dcode, code, _layout(rows, w, g), x.device.index)[1]
    _lib.linear_backward(rows, w, preact, g, dx, dw, db, _scratch(size, x), m, k, n, dcode, code)
    return dx, dw, db


def _slope_formula(p: Tensor, code: int) -> Tensor:
    """act'(p) in differentiable PyTorch operations."""
    if code == ACTIVATIONS["relu"]:
        return (p > 0).to(p.dtype)
    if code == ACTIVATIONS["silu"]:
        s = torch.sigmoid(p)
        return s * (1 + p * (1 - s))
    if code == ACTIVATIONS["gelu"]:
        return 0.5 * (1 + torch.erf(p * math.sqrt(0.5))) + \
            p * torch.exp(-0.5 * p * p) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (p + 0.044715 * p ** 3))
    return 0.5 * (1 + t) + 0.5 * p * (1 - t * t) * c * (1 + 3 * 0.044715 * p * p)


def _linear_grad_formula(x, weight, bias, code, grad, need):
    """The backward as a differentiable composition, for second derivatives: the products
    are linear layers again and run on the same kernels."""
    rows, g = _rows(x), _rows(grad)
    if code:
        p = linear(rows, weight, bias).float()
        g = (g.float() * _slope_formula(p, code)).to(x.dtype)
    dx = linear(g, weight.t()).reshape(x.shape) if need[0] else None
    dw = linear(g.t(), rows.t()) if need[1] else None
    return dx, dw, g.float().sum(0).to(x.dtype) if need[2] else None


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, code):
        y, preact = _linear_run(x, weight, bias, residual, code, code != 0)
        ctx.save_for_backward(x, weight, bias, preact)
        ctx.code = code
        return y

    @staticmethod
    def backward(ctx, grad):
        x, weight, bias, preact = ctx.saved_tensors
        need = ctx.needs_input_grad
        if torch.is_grad_enabled():
            grads = _linear_grad_formula(x, weight, bias, ctx.code, grad, need)
        else:
            grads = _linear_grad_run(x, weight, preact, grad, ctx.code, need)
        return (*grads, grad if need[3] else None, None)


@torch.library.custom_op(f"{NAMESPACE}::linear_forward", mutates_args=())
def _linear_op(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, code: int,
               save: bool) -> tuple[Tensor, Tensor]:
    y, preact = _linear_run(x, weight, bias, residual, code, save)
    return y, preact if save else x.new_empty(0, dtype=torch.float32)


@_linear_op.register_fake
def _linear_op_fake(x, weight, bias, residual, code, save):
    n = weight.shape[0]
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    shape = (math.prod(x.shape[:-1]), n) if save else (0,)
    return y, x.new_empty(shape, dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::linear_backward", mutates_args=())
def _linear_grad_op(x: Tensor, weight: Tensor, preact: Tensor, grad: Tensor, code: int
                    ) -> tuple[Tensor, Tensor, Tensor]:
    return _linear_grad_run(x, weight, preact if code else None, grad, code, (True, True, True))


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


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, activation: str = "none",
           residual: Tensor | None = None) -> Tensor:
    """act(x weight^T + bias) + residual: x [..., in], weight [out, in], bias [out],
    residual [..., out]; activation one of ACTIVATIONS."""
    what = "linear"
    _check_input(what, x)
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: x [..., in] and weight [out, in] do not match: "
                         f"{tuple(x.shape)} and {tuple(weight.shape)}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("linear needs at least one input and one output feature")
    _check_like(what, "weight", weight, x)
    if bias is not None:
        _check_like(what, "bias", bias, x)
        if bias.shape != weight.shape[:1]:
            raise ValueError(f"linear: bias must have shape {tuple(weight.shape[:1])}, "
                             f"got {tuple(bias.shape)}")
        bias = bias.contiguous()
    if residual is not None:
        _check_like(what, "residual", residual, x)
        if residual.shape != (*x.shape[:-1], weight.shape[0]):
            raise ValueError(f"linear: residual must have the output's shape "
                             f"{(*x.shape[:-1], weight.shape[0])}, got {tuple(residual.shape)}")
    wanted = torch.is_grad_enabled() and (
        x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
        (residual is not None and residual.requires_grad))
    if torch.compiler.is_compiling():
        return _linear_op(x, weight, bias, residual, code, wanted and code != 0)[0]
    if wanted:
        return _LinearFunction.apply(x, weight, bias, residual, code)
    return _linear_run(x, weight, bias, residual, code, False)[0]


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
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, "
                             f"got {activation!r}")
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)
        self.activation = activation

    def forward(self, x: Tensor, residual: Tensor | None = None) -> Tensor:
        return linear(x, self.weight, self.bias, self.activation, residual)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"


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


class RadialTrunk(torch.nn.Module):
    """Radial basis [..., in_features] to the hidden features [..., hidden] that
    ``RadialUvuTensorProduct`` takes: an embedding layer, residual blocks and a final
    layer norm."""

    def __init__(self, in_features: int, hidden: int, blocks: int = 1, activation: str = "silu",
                 device=None, dtype=None):
        super().__init__()
        if int(blocks) < 0:
            raise ValueError("blocks must be >= 0")
        kw = {"device": device, "dtype": dtype}
        self.embed = Linear(in_features, hidden, activation=activation, **kw)
        self.blocks = torch.nn.ModuleList(
            ResidualBlock(hidden, activation=activation, **kw) for _ in range(int(blocks)))
        self.norm = LayerNorm(hidden, **kw)

    def forward(self, basis: Tensor) -> Tensor:
        h = self.embed(basis)
        for block in self.blocks:
            h = block(h)
        return self.norm(h)
