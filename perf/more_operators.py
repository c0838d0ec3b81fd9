"""Cases and plain forms of the operators of a training step beyond the linear layer: the
gated linear layer act(x Wg^T + bg) * (x Wu^T + bu), and the global norm of many gradients
with clipping.

A case is a dict of plain values.  ``run`` computes one pass: in elementary torch
operations in 32 bits when ``own`` is false, through ``ictc_o2_hp_b200.dense`` and
``ictc_o2_hp_b200.gradients`` when it is true.  ``train`` passes of the gated layer return
the output and every gradient; passes over gradients return the norm and the gradients.
"""

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")
EPS = 1e-6   # added to the norm that the largest norm is divided by

# The largest listed sizes; a drawn case stays within them.
MOST_PRODUCT = 16384 * 4096 * 4096   # rows x in x hidden of a gated layer
MOST_VALUES = 1048576 * 192          # rows x (in + 2 hidden) of a gated layer
MOST_WEIGHTS = 4096 * 16384          # in x hidden
MOST_GRADIENTS = 268435456           # elements of all gradients together


def _gated(name, rows, inner, hidden, dtype, train, activation="silu"):
    return {"name": name, "op": "gated", "rows": rows, "in": inner, "hidden": hidden,
            "dtype": dtype, "train": train, "activation": activation}


def _grads(name, op, tensors, elements, dtype, packed=False):
    return {"name": name, "op": op, "tensors": tensors, "elements": elements, "dtype": dtype,
            "packed": packed}


def listed():
    return [
        # The edges of one small molecule through a gated radial layer: an energy query.
        _gated("gated_f32_37x64x64", 37, 64, 64, "float32", False),
        # A gated radial layer over the edges of a large batch, one training step.
        _gated("gated_train_f32_1048576x64x64", 1048576, 64, 64, "float32", True),
        # The widening half of a node feed-forward block, one training step.
        _gated("gated_train_f32_65536x128x512", 65536, 128, 512, "float32", True, "gelu"),
        # One row (a token, a single node) of a wide 16-bit model.
        _gated("gated_bf16_1x4096x16384", 1, 4096, 16384, "bfloat16", False),
        # A small serving batch against weights larger than the L2 cache.
        _gated("gated_bf16_16x4096x16384", 16, 4096, 16384, "bfloat16", False, "gelu_tanh"),
        # Ragged everything: no dimension a multiple of any tile or vector.
        _gated("gated_train_f16_4999x1111x777", 4999, 1111, 777, "float16", True, "gelu"),
        # A large compute-bound training step.
        _gated("gated_train_bf16_16384x4096x4096", 16384, 4096, 4096, "bfloat16", True),
        # The gradients of a small radial network, clipped before the optimiser's step.
        _grads("clip_f32_16x24768", "clip", 16, 24768, "float32"),
        # Many tensors of odd sizes and two types, clipped into flat buckets without padding.
        _grads("clip_mixed_300x40000003", "clip", 300, 40000003, "mixed", True),
        # All gradients of a large float32 model, clipped out of place.
        _grads("clip_f32_48x268435456", "clip", 48, 268435456, "float32"),
        # A healthy step: the gradients of a 16-bit model stay below the limit, in place.
        _grads("clip_quiet_bf16_48x268435456", "quiet", 48, 268435456, "bfloat16"),
        # The norm alone, for a log line: float16 gradients of a middling model.
        _grads("norm_f16_200x9999991", "norm", 200, 9999991, "float16"),
    ]


def _log_int(rng, low, high):
    if high <= low:
        return low
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    if rng.random() < 0.35:
        op = rng.choice(("clip", "clip", "quiet", "norm"))
        tensors = _log_int(rng, 1, 1500)
        return {"op": op, "tensors": tensors, "elements": _log_int(rng, tensors, MOST_GRADIENTS),
                "dtype": rng.choice(("float32", "bfloat16", "float16", "mixed")),
                "packed": rng.random() < 0.5}
    inner, hidden = _log_int(rng, 1, 16384), _log_int(rng, 1, 16384)
    while inner * hidden > MOST_WEIGHTS:
        inner, hidden = _log_int(rng, 1, 16384), _log_int(rng, 1, 16384)
    most = min(1048576, MOST_PRODUCT // (inner * hidden), MOST_VALUES // (inner + 2 * hidden))
    return {"op": "gated", "rows": _log_int(rng, 1, most), "in": inner, "hidden": hidden,
            "dtype": rng.choice(list(DTYPES)), "train": rng.random() < 0.6,
            "activation": rng.choice(ACTIVATIONS)}


def _counts(case):
    """Elements of each gradient: sizes over two orders of magnitude, none empty, their sum
    the case's."""
    n, total = case["tensors"], case["elements"]
    rng = random.Random(n * 1000003 + total)
    weights = [math.exp(rng.uniform(0, math.log(100))) for _ in range(n)]
    scale = (total - n) / sum(weights)
    counts = [1 + int(w * scale) for w in weights]
    counts[-1] += total - sum(counts)
    return counts


def _types(case):
    if case["dtype"] != "mixed":
        return [DTYPES[case["dtype"]]] * case["tensors"]
    return [torch.float32 if i % 3 == 0 else torch.bfloat16 for i in range(case["tensors"])]


def _flat_views(counts, types, packed, device):
    """One flat buffer for each type and, for each tensor, its part of it: one behind the
    other, or each at a multiple of 64 elements."""
    unit = 1 if packed else 64
    at, places = {}, []
    for count, dtype in zip(counts, types):
        places.append(at.get(dtype, 0))
        at[dtype] = places[-1] + -(-count // unit) * unit
    flats = {dtype: torch.zeros(size, dtype=dtype, device=device) for dtype, size in at.items()}
    return flats, [flats[t][p:p + c] for c, t, p in zip(counts, types, places)]


def _prepare_grads(case, seed, device, gen):
    counts, types = _counts(case), _types(case)
    spread = random.Random(seed)
    flats, grads = _flat_views(counts, types, case["packed"], device)
    for flat in flats.values():
        flat.normal_(generator=gen)
    # layers differ in the size of their gradients
    for g in grads:
        g.mul_(math.exp(spread.uniform(-2, 1)) * 1e-2)
    if not case["packed"]:
        # what lies between the tensors is theirs no more
        for flat in flats.values():
            view = torch.zeros_like(flat)
            for g in grads:
                if g.dtype == flat.dtype:
                    at = g.storage_offset()
                    view[at:at + g.numel()] = g
            flat.copy_(view)
    state = {"case": dict(case), "grads": grads, "flats": flats}
    # the norm is near 1e-2 sqrt(elements): clipped by about four, or left alone
    typical = 1e-2 * math.sqrt(case["elements"])
    state["most"] = 0.25 * typical if case["op"] == "clip" else 1e3 * typical
    if case["op"] == "clip":
        state["out_flats"], state["out"] = _flat_views(counts, types, case["packed"], device)
    return state


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    if case["op"] != "gated":
        return _prepare_grads(case, seed, device, gen)
    dtype, train = DTYPES[case["dtype"]], case["train"]
    rows, inner, hidden = case["rows"], case["in"], case["hidden"]

    def randn(*shape, scale=1.0):
        t = torch.randn(*shape, device=device, generator=gen)
        return t.mul_(scale).to(dtype)

    state = {"case": dict(case), "x": randn(rows, inner),
             "weight": randn(2 * hidden, inner, scale=1.5 / math.sqrt(inner)),
             "bias": randn(2 * hidden, scale=0.1)}
    if train:
        for name in ("x", "weight", "bias"):
            state[name].requires_grad_(True)
        state["grad"] = randn(rows, hidden)
    return state


# ------------------------------------------------------------------------ plain forms


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
    if activation == "none":
        return torch.ones_like(p)
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


def _plain_gated(state, case):
    dtype = DTYPES[case["dtype"]]
    x, weight, bias = (state[k].detach().float() for k in ("x", "weight", "bias"))
    hidden = case["hidden"]
    p = torch.matmul(x, weight.t()) + bias
    gate, up = p[:, :hidden], p[:, hidden:]
    acted = _activate(gate, case["activation"])
    y = (acted * up).to(dtype)
    if not case["train"]:
        return {"y": y}
    g = state["grad"].float()
    d = torch.cat([g * up * _slope(gate, case["activation"]), g * acted], 1)
    return {"y": y, "dx": torch.matmul(d, weight).to(dtype),
            "dweight": torch.matmul(d.t(), x).to(dtype), "dbias": d.sum(0).to(dtype)}


def _plain_grads(state, case):
    """On the flat buffers, which hold the gradients and nothing else: squares in 32 bits,
    their long sums in 64."""
    wide = {t: f.float() for t, f in state["flats"].items()}
    sums = [torch.sum(f * f, dtype=torch.float64) for f in wide.values()]
    norm = torch.sqrt(torch.stack(sums).sum())
    if case["op"] == "norm":
        return {"norm": norm.float()}
    factor = torch.clamp(state["most"] / (norm + EPS), max=1.0).float()
    targets = state["out_flats"] if case["op"] == "clip" else state["flats"]
    return {"norm": norm.float(), "grads": [targets[t].copy_(f * factor) for t, f in wide.items()]}


def run(state):
    case = state["case"]
    if not own:
        return _plain_gated(state, case) if case["op"] == "gated" else _plain_grads(state, case)
    if case["op"] == "gated":
        from ictc_o2_hp_b200 import dense
        inputs = [state[k] for k in ("x", "weight", "bias")]
        y = dense.gated_linear(*inputs, activation=case["activation"])
        if not case["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, inputs, state["grad"])
        return {"y": y.detach(), **dict(zip(("dx", "dweight", "dbias"), grads))}
    from ictc_o2_hp_b200 import gradients
    if case["op"] == "norm":
        return {"norm": gradients.grad_norm(state["grads"])}
    if case["op"] == "clip":
        _, norm = gradients.clip_grads(state["grads"], state["most"], out=state["out"])
        return {"norm": norm, "grads": list(state["out_flats"].values())}
    _, norm = gradients.clip_grads(state["grads"], state["most"], out=state["grads"])
    return {"norm": norm, "grads": list(state["flats"].values())}


def work(case):
    if case["op"] != "gated":
        sizes = [c * (4 if t == torch.float32 else 2)
                 for c, t in zip(_counts(case), _types(case))]
        # every gradient read; clipped ones written (those below the limit stay as they are)
        passes = 2 if case["op"] == "clip" else 1
        return {"bytes": passes * sum(sizes),
                "flops": case["elements"] * (3 if case["op"] == "clip" else 2)}
    size = 4 if case["dtype"] == "float32" else 2
    rows, inner, hidden, train = case["rows"], case["in"], case["hidden"], case["train"]
    x, w, y = rows * inner, 2 * hidden * (inner + 1), rows * hidden
    values = x + w + y
    if train:
        values += y + x + w      # the output's gradient read, the gradients written
    return {"bytes": size * values, "flops": (12 if train else 4) * rows * inner * hidden}


# --------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    """The definitions in 64 bits, the gated layer's gradients by automatic differentiation."""
    state = prepare(case, seed)
    if case["op"] != "gated":
        squares = [torch.linalg.vector_norm(g.double()) ** 2 for g in state["grads"]]
        norm = torch.stack(squares).sum().sqrt()
        if case["op"] == "norm":
            return {"norm": norm}
        factor = min(1.0, state["most"] / (norm.item() + EPS))
        return {"norm": norm, "grads": [f.double() * factor for f in state["flats"].values()]}
    names = {"x": "dx", "weight": "dweight", "bias": "dbias"}
    wide = {k: state[k].detach().double().requires_grad_(case["train"]) for k in names}
    gate, up = (torch.einsum("rk,nk->rn", wide["x"], w) + b for w, b in
                zip(wide["weight"].chunk(2), wide["bias"].chunk(2)))
    name = case["activation"]
    if name == "relu":
        gate = gate.clamp(min=0)
    elif name == "silu":
        gate = gate * torch.sigmoid(gate)
    elif name == "gelu":
        gate = gate * torch.special.ndtr(gate)
    elif name == "gelu_tanh":
        # (1 + tanh(u)) / 2 is the logistic function of 2 u
        gate = gate * torch.sigmoid(math.sqrt(8 / math.pi) * (gate + 0.044715 * gate ** 3))
    y = gate * up
    if not case["train"]:
        return {"y": y.detach()}
    grads = torch.autograd.grad(y, list(wide.values()), state["grad"].double())
    return {"y": y.detach(), **dict(zip(names.values(), grads))}
