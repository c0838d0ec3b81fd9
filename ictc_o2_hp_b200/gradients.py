"""The global norm of a training step's gradients, and clipping by it, on the GPU.

    norm = clip_grad_norm_(model.parameters(), 1.0)          # in place, as torch's
    clipped, norm = clip_grads(torch.autograd.grad(...), 1.0)
    norm = grad_norm(grads)                                  # for a log line

The reference leaves this to PyTorch.  All tensors of a call go into one launch for the norm
and one for the scaling, whatever their number (up to 1,024 each), sizes and types: CUDA
float32, bfloat16 and float16 on one device.  The norm is a float32 scalar on that device,
and nothing waits for it.  2-norms (sums of squares in float64) and the largest magnitude
(``norm_type=math.inf``).  Non-finite gradients scale as in PyTorch: a NaN norm makes
every gradient NaN, an infinite one makes finite gradients 0.

Nothing here is differentiable: results carry no graph, and tensors with forward-mode tangents
raise NotImplementedError.  Other devices and types raise TypeError instead of falling back.
"""

from __future__ import annotations

import ctypes
import importlib.util
import math
from collections.abc import Iterable, Sequence
from pathlib import Path

import torch
from torch import Tensor

from . import _lib
from .ops import NAMESPACE

EXTENSION = Path(__file__).resolve().parent / "_lib" / "_gradient_lists.so"
_native = None


def _load():
    """Loads the extension module once and binds it to the kernel library."""
    global _native
    if _native is None:
        if not EXTENSION.exists():
            raise RuntimeError(f"{EXTENSION} is missing: build it with `python -m "
                               "ictc_o2_hp_b200.build` (gradient clipping has no fallback)")
        spec = importlib.util.spec_from_file_location("_gradient_lists", EXTENSION)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        lib = _lib.load()
        names = ("ictc_o2_last_error", "ictc_o2_grad_norm_workspace", "ictc_o2_grad_norm",
                 "ictc_o2_clip_grads")
        module.bind(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names))
        _native = module
    return _native


# ------------------- custom operators, for torch.compile and whatever watches the dispatcher


@torch.library.custom_op(f"{NAMESPACE}::grad_norm", mutates_args=())
def _norm_op(grads: Sequence[Tensor], largest: bool) -> Tensor:
    return _load().grad_norm(list(grads), largest)


@_norm_op.register_fake
def _norm_op_fake(grads, largest):
    return grads[0].new_empty((), dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::clip_grads", mutates_args={"out"})
def _clip_op(grads: Sequence[Tensor], out: Sequence[Tensor], max_norm: float, largest: bool
             ) -> Tensor:
    return _load().clip_grads(list(grads), max_norm, largest, list(out))[1]


@_clip_op.register_fake
def _clip_op_fake(grads, out, max_norm, largest):
    return grads[0].new_empty((), dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::clip_grads_", mutates_args={"grads"})
def _clip_in_place_op(grads: Sequence[Tensor], max_norm: float, largest: bool) -> Tensor:
    return _load().clip_grads(list(grads), max_norm, largest, list(grads))[1]


@_clip_in_place_op.register_fake
def _clip_in_place_op_fake(grads, max_norm, largest):
    return grads[0].new_empty((), dtype=torch.float32)


# ---------------------------------------------------------------------- functions


def _is_largest(norm_type: float) -> bool:
    kind = float(norm_type)
    if kind != 2.0 and kind != math.inf:
        raise ValueError(f"norm_type must be 2 or math.inf, got {norm_type}")
    return kind == math.inf


def grad_norm(tensors: Tensor | Iterable[Tensor], norm_type: float = 2.0) -> Tensor:
    """The norm of all tensors together, as if they were one vector: a float32 scalar on
    their device (0 on the CPU for no tensors)."""
    if not isinstance(tensors, (list, tuple)):
        tensors = [tensors] if isinstance(tensors, Tensor) else list(tensors)
    largest = _is_largest(norm_type)
    if not tensors:
        return torch.zeros(())
    norm = None
    if not torch.compiler.is_compiling():
        norm = (_native or _load()).grad_norm(tensors, largest)
    if norm is None:
        with torch.no_grad():
            norm = _norm_op(list(tensors), largest)
    return norm


def clip_grads(grads: Sequence[Tensor], max_norm: float, norm_type: float = 2.0,
               out: Sequence[Tensor] | None = None) -> tuple[list[Tensor], Tensor]:
    """The gradients times min(1, max_norm / (norm + 1e-6)), and their norm.

    ``out``: tensors of the same shapes and types to write (flat buckets' views, say);
    ``out=grads`` scales in place.  Without it new tensors are made, parts of one allocation
    (which lives as long as any of them).  An output may be its own gradient, but share no
    memory with any other."""
    if not isinstance(grads, (list, tuple)):
        grads = list(grads)
    if out is not None and not isinstance(out, (list, tuple)):
        out = list(out)
    largest, max_norm = _is_largest(norm_type), float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    if not grads:
        if out:
            raise ValueError(f"0 gradients and {len(out)} outputs")
        return [], torch.zeros(())
    result = None
    if not torch.compiler.is_compiling():
        result = (_native or _load()).clip_grads(grads, max_norm, largest, out)
    if result is None:
        result = _clip_watched(list(grads), max_norm, largest, out)
    return result


@torch.no_grad()
def _clip_watched(grads, max_norm, largest, out):
    if out is not None and len(out) == len(grads) and all(o is g for o, g in zip(out, grads)):
        return list(out), _clip_in_place_op(grads, max_norm, largest)
    out = [torch.empty_like(g) for g in grads] if out is None else list(out)
    return out, _clip_op(grads, out, max_norm, largest)


def clip_grad_norm_(parameters: Tensor | Iterable[Tensor], max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False) -> Tensor:
    """``torch.nn.utils.clip_grad_norm_`` for CUDA gradients: scales every ``.grad`` in place
    so that their norm is at most max_norm, and returns the norm from before.  With
    ``error_if_nonfinite`` it waits for the norm and raises RuntimeError instead of scaling.
    A parameter may be listed once only."""
    parameters = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if error_if_nonfinite and not torch.isfinite(norm := grad_norm(grads, norm_type)):
        raise RuntimeError(f"the gradients' norm is {norm.item()}: they were not clipped")
    return clip_grads(grads, max_norm, norm_type, out=grads)[1]
