"""Cases and plain forms of the dense operators around the tensor products: layer norm
over the last dimension, and the linear layer act(x W^T + b) + residual.

A case is a dict of plain values.  ``run`` computes one pass: in elementary torch
operations in 32 bits when ``own`` is false, through ``ictc_o2_hp_b200.dense`` when it
is true.  ``train`` passes return the output and every gradient.
"""

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")
EPS = 1e-5

# The largest listed sizes; a drawn case stays within all three.
MOST_PRODUCT = 16384 * 4096 * 4096   # rows x in x out of a linear layer
MOST_VALUES = 1048576 * 128          # rows x (in + out) of a linear layer
MOST_NORM = 1048576 * 64             # rows x width of a layer norm


def _norm(name, rows, width, dtype, train):
    return {"name": name, "op": "layer_norm", "rows": rows, "width": width, "dtype": dtype,
            "train": train}


def _linear(name, rows, inner, outer, dtype, train, activation, residual):
    return {"name": name, "op": "linear", "rows": rows, "in": inner, "out": outer,
            "dtype": dtype, "train": train, "activation": activation, "residual": residual}


def listed():
    return [
        # One edge's radial hidden features, as a single energy query evaluates them.
        _norm("norm_f32_1x64", 1, 64, "float32", False),
        # The radial hidden features of 1,048,576 edges, one training step.
        _norm("norm_train_f32_1048576x64", 1048576, 64, "float32", True),
        # The rows of 65,536 nodes at 64 channels, order 3, both parities; inference.
        _norm("norm_f32_65536x896", 65536, 896, "float32", False),
        # Wide 16-bit activations of a token-like batch, one training step.
        _norm("norm_train_bf16_16384x4096", 16384, 4096, "bfloat16", True),
        # Odd rows and an odd width: rows that start off every vector boundary.
        _norm("norm_train_f16_9973x1337", 9973, 1337, "float16", True),
        # Radial basis to hidden features for the edges of one small molecule.
        _linear("linear_f32_37x8x64", 37, 8, 64, "float32", False, "silu", False),
        # A residual radial layer on 1,048,576 edges, one training step.
        _linear("linear_train_f32_1048576x64x64", 1048576, 64, 64, "float32", True, "silu", True),
        # The widening product of a node feed-forward block, one training step.
        _linear("linear_train_f32_65536x128x512", 65536, 128, 512, "float32", True, "gelu",
                False),
        # One token of a wide 16-bit model.
        _linear("linear_bf16_1x4096x4096", 1, 4096, 4096, "bfloat16", False, "silu", True),
        # A small serving batch against weights larger than the L2 cache.
        _linear("linear_bf16_16x4096x16384", 16, 4096, 16384, "bfloat16", False, "gelu_tanh",
                False),
        # Ragged everything: no dimension a multiple of any tile or vector.
        _linear("linear_train_f16_4999x1111x777", 4999, 1111, 777, "float16", True, "gelu",
                True),
        # A large compute-bound training step.
        _linear("linear_train_bf16_16384x4096x4096", 16384, 4096, 4096, "bfloat16", True, "silu",
                True),
    ]


def _log_int(rng, low, high):
    if high <= low:
        return low
    value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, value + 1 if value == 3072 else value))


def draw(rng):
    dtype = rng.choice(list(DTYPES))
    train = rng.random() < 0.6
    if rng.random() < 0.4:
        width = _log_int(rng, 1, 16384)
        rows = _log_int(rng, 1, min(1048576, MOST_NORM // width))
        return {"op": "layer_norm", "rows": rows, "width": width, "dtype": dtype, "train": train}
    inner, outer = _log_int(rng, 1, 16384), _log_int(rng, 1, 16384)
    while inner * outer > 4096 * 16384:
        inner, outer = _log_int(rng, 1, 16384), _log_int(rng, 1, 16384)
    most = min(1048576, MOST_PRODUCT // (inner * outer), MOST_VALUES // (inner + outer))
    return {"op": "linear", "rows": _log_int(rng, 1, most), "in": inner, "out": outer,
            "dtype": dtype, "train": train, "activation": rng.choice(ACTIVATIONS),
            "residual": rng.random() < 0.5}


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    dtype, train = DTYPES[case["dtype"]], case["train"]

    def randn(*shape, scale=1.0, shift=0.0):
        t = torch.randn(*shape, device=device, generator=gen)
        return t.mul_(scale).add_(shift).to(dtype)

    rows = case["rows"]
    state = {"case": dict(case)}
    if case["op"] == "layer_norm":
        width = case["width"]
        state["x"] = randn(rows, width, scale=1.5, shift=0.5)
        state["weight"] = randn(width, scale=0.1, shift=1.0)
        state["bias"] = randn(width, scale=0.1)
        outer = width
    else:
        inner, outer = case["in"], case["out"]
        state["x"] = randn(rows, inner)
        state["weight"] = randn(outer, inner, scale=1.5 / math.sqrt(inner))
        state["bias"] = randn(outer, scale=0.1)
        if case["residual"]:
            state["residual"] = randn(rows, outer)
    if train:
        for name in ("x", "weight", "bias", "residual"):
            if name in state:
                state[name].requires_grad_(True)
        state["grad"] = randn(rows, outer)
    return state


def _activate(p, activation):
    if activation == "none":
        return p
    if activation == "relu":
        return torch.where(p > 0, p, torch.zeros_like(p))
    if activation == "silu":
        return p / (1 + torch.exp(-p))
    if activation == "gelu":
        return 0.5 * p * (1 + torch.erf(p * math.sqrt(0.5)))
    return 0.5 * p * (1 + torch.tanh(math.sqrt(2 / math.pi) * (p + 0.044715 * p * p * p)))


def _slope(p, activation):
    """The activation's derivative at p."""
    if activation == "relu":
        return (p > 0).to(p.dtype)
    if activation == "silu":
        s = 1 / (1 + torch.exp(-p))
        return s * (1 + p * (1 - s))
    if activation == "gelu":
        density = torch.exp(-0.5 * p * p) * (1 / math.sqrt(2 * math.pi))
        return 0.5 * (1 + torch.erf(p * math.sqrt(0.5))) + p * density
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (p + 0.044715 * p * p * p))
    return 0.5 * (1 + t) + 0.5 * p * (1 - t * t) * c * (1 + 3 * 0.044715 * p * p)


def _plain_norm(state, train, dtype):
    x, weight, bias = (state[k].detach().float() for k in ("x", "weight", "bias"))
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    unit = centred * rstd
    y = (unit * weight + bias).to(dtype)
    if not train:
        return {"y": y}
    g = state["grad"].float()
    h = g * weight
    dx = rstd * (h - h.mean(-1, keepdim=True) - unit * (h * unit).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(dtype), "dweight": (g * unit).sum(0).to(dtype),
            "dbias": g.sum(0).to(dtype)}


def _plain_linear(state, train, dtype, activation):
    x, weight, bias = (state[k].detach().float() for k in ("x", "weight", "bias"))
    p = torch.matmul(x, weight.t()) + bias
    y = _activate(p, activation)
    residual = state.get("residual")
    if residual is not None:
        y = y + residual.detach().float()
    y = y.to(dtype)
    if not train:
        return {"y": y}
    g = state["grad"].float()
    d = g if activation == "none" else g * _slope(p, activation)
    out = {"y": y, "dx": torch.matmul(d, weight).to(dtype),
           "dweight": torch.matmul(d.t(), x).to(dtype), "dbias": d.sum(0).to(dtype)}
    if residual is not None:
        out["dresidual"] = state["grad"].clone()
    return out


def run(state):
    case = state["case"]
    train, dtype = case["train"], DTYPES[case["dtype"]]
    norm = case["op"] == "layer_norm"
    if not own:
        if norm:
            return _plain_norm(state, train, dtype)
        return _plain_linear(state, train, dtype, case["activation"])
    from ictc_o2_hp_b200 import dense
    x, weight, bias = state["x"], state["weight"], state["bias"]
    residual = state.get("residual")
    if norm:
        y = dense.layer_norm(x, weight, bias, EPS)
    else:
        y = dense.linear(x, weight, bias, activation=case["activation"], residual=residual)
    if not train:
        return {"y": y}
    inputs = [x, weight, bias] + ([residual] if residual is not None else [])
    grads = torch.autograd.grad(y, inputs, state["grad"])
    names = ("dx", "dweight", "dbias", "dresidual")
    return {"y": y.detach(), **dict(zip(names, grads))}


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    rows, train = case["rows"], case["train"]
    if case["op"] == "layer_norm":
        # x read, y written; in training x and the output's gradient read, dx written.
        values = rows * case["width"] * (4 if train else 2) + case["width"] * (4 if train else 2)
        return {"bytes": size * values, "flops": rows * case["width"] * (20 if train else 8)}
    inner, outer = case["in"], case["out"]
    y, x, w = rows * outer, rows * inner, inner * outer
    values = x + w + outer + y + (y if case["residual"] else 0)
    if train:
        values += y + x + w + outer      # the output's gradient read, the gradients written
    return {"bytes": size * values, "flops": (6 if train else 2) * rows * inner * outer}


def exact(case, seed):
    """The definition in 64 bits, its gradients by automatic differentiation."""
    state = prepare(case, seed)
    wide = {k: v.detach().double().requires_grad_(case["train"] and k != "grad")
            for k, v in state.items() if k != "case"}
    x, weight, bias = wide["x"], wide["weight"], wide["bias"]
    if case["op"] == "layer_norm":
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        y = torch.addcmul(bias, (x - mean) / (var + EPS).sqrt(), weight)
    else:
        p = torch.einsum("rk,nk->rn", x, weight) + bias
        name = case["activation"]
        if name == "relu":
            p = p.clamp(min=0)
        elif name == "silu":
            p = p * torch.sigmoid(p)
        elif name == "gelu":
            p = p * torch.special.ndtr(p)
        elif name == "gelu_tanh":
            # (1 + tanh(u)) / 2 is the logistic function of 2 u
            p = p * torch.sigmoid(math.sqrt(8 / math.pi) * (p + 0.044715 * p ** 3))
        y = p + wide["residual"] if "residual" in wide else p
    if not case["train"]:
        return {"y": y.detach()}
    names = {"x": "dx", "weight": "dweight", "bias": "dbias", "residual": "dresidual"}
    inputs = [k for k in names if k in wide]
    grads = torch.autograd.grad(y, [wide[k] for k in inputs], wide["grad"])
    return {"y": y.detach(), **{names[k]: g for k, g in zip(inputs, grads)}}
