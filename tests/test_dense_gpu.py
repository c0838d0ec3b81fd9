"""Layer norm and the linear layer on the GPU against plain float64 formulas.

Tolerances are error bounds of the arithmetic, element by element, with U the unit
roundoff of float32 and u that of the operand type:
- a sum of n terms added one after another is off by at most n U sum |term|; the
  tensor-core products truncate (2 U) once per 16 elements of the sum, and the float32
  parts that are left out stay below 4 U |a b|;
- an output of a 16-bit type is off by u |y| more, and the rounded d = g act'(p) that a
  16-bit backward multiplies with adds u sum |d| |w|;
- activations have slopes below 1.2 and curvatures below 1.1; their own evaluation is
  good to 16 U (|p| + 1).
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def rand(shape, dtype, device, seed, scale=1.0, shift=0.0):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    return (torch.randn(shape, device=device, generator=gen) * scale + shift).to(dtype)


def within(name, got, want, bound):
    assert got.shape == want.shape, f"{name}: {tuple(got.shape)} and {tuple(want.shape)}"
    if got.numel() == 0:
        return
    over = ((got.double() - want).abs() - bound).max().item()
    assert over <= 0, f"{name}: over its bound by {over:.3e}"


# ---------------------------------------------------------------- plain formulas


def act64(p, name):
    if name == "relu":
        return p.clamp(min=0)
    if name == "silu":
        return p * torch.sigmoid(p)
    if name == "gelu":
        return 0.5 * p * (1 + torch.erf(p / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * p * (1 + torch.tanh(math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3)))
    return p


def slope64(p, name):
    if name == "none":
        return torch.ones_like(p)
    if name == "relu":
        return (p > 0).double()
    q = p.detach().clone().requires_grad_(True)
    return torch.autograd.grad(act64(q, name).sum(), q)[0]


def linear64(x, w, b, r, act, g):
    """Float64 results and, for each, the bound's magnitude terms."""
    x, w, g = x.double(), w.double(), g.double()
    p = x @ w.t() + (0 if b is None else b.double())
    y = act64(p, act) + (0 if r is None else r.double())
    s = slope64(p, act)
    d = g * s
    return p, y, s, d, d @ w, d.t() @ x, d.sum(0)


def sum_error(k):
    """Relative error of a tensor-core sum over k elements."""
    return (2 * (k / 16) + k / 64 + 64) * U


def check_linear(x, w, b, r, act, g, y, grads, dtype):
    u, k, n, m = UNIT[dtype], w.shape[1], w.shape[0], x.shape[0]
    p, y64, s, d, dx, dw, db = linear64(x, w, b, r, act, g)
    ax, aw, ag = x.double().abs(), w.double().abs(), g.double().abs()
    ep = sum_error(k) * (ax @ aw.t() + (0 if b is None else b.double().abs())) + 16 * U * (
        p.abs() + 1) * (act != "none")
    tiny = TINY[dtype]
    within("y", y, y64, 1.2 * ep + (u + 2 * U) * (
        y64.abs() + (0 if r is None else r.double().abs()) * U / u) * 1.01 + tiny)
    if grads is None:
        return
    ed = ag * (1.1 * ep + 16 * U) * (act != "none")
    if act == "relu":  # the slope of a p within its error of 0 may go either way
        ed = ag * (p.abs() <= ep)
    if dtype != torch.float32 and act != "none":
        ed = ed + u * d.abs() + tiny
    ad = d.abs() + ed
    within("dx", grads[0], dx, ed @ aw + sum_error(n) * (ad @ aw) + (u + 2 * U) * (
        dx.abs() + ed @ aw) + tiny)
    within("dweight", grads[1], dw, ed.t() @ ax + sum_error(m) * (ad.t() @ ax) + (u + 2 * U) * (
        dw.abs() + ed.t() @ ax) + tiny)
    if b is not None:
        eds = ag * (1.1 * ep + 16 * U) * (act != "none") if act != "relu" else ed
        within("dbias", grads[2], db, eds.sum(0) + (m + 64) * U * ad.sum(0) + (u + 2 * U) * (
            db.abs() + eds.sum(0)) + tiny)


LINEAR_SHAPES = [
    (1, 1, 1), (1, 64, 64), (3, 7, 5), (4, 129, 1), (5, 8, 64), (37, 8, 64), (127, 63, 65),
    (128, 64, 128), (129, 65, 127), (200, 257, 3), (255, 16, 130), (300, 1000, 72), (64, 2049, 33),
    (1000, 33, 200), (2500, 64, 64), (5000, 7, 3), (3000, 64, 1), (129, 1, 64), (513, 61, 59),
    (6, 16, 16), (700, 1025, 769), (2053, 211, 333), (4097, 702, 6), (5000, 1536, 8), (4100, 1030, 1),
    (4500, 3, 130), (4099, 8, 520),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", LINEAR_SHAPES)
def test_linear_against_float64(shape, dtype, cuda_device):
    from ictc_o2_hp_b200 import _lib, dense
    m, k, n = shape
    act = ACTS[(m + k + n) % len(ACTS)]
    x = rand((m, k), dtype, cuda_device, 1).requires_grad_(True)
    w = rand((n, k), dtype, cuda_device, 2, 1.5 / math.sqrt(k)).requires_grad_(True)
    b = rand((n,), dtype, cuda_device, 3).requires_grad_(True) if (m + n) % 3 else None
    r = rand((m, n), dtype, cuda_device, 4).requires_grad_(True) if (m + k) % 2 else None
    g = rand((m, n), dtype, cuda_device, 5)
    y = dense.linear(x, w, b, act, r)
    inputs = [t for t in (x, w, b, r) if t is not None]
    grads = torch.autograd.grad(y, inputs, g)
    check_linear(x.detach(), w.detach(), None if b is None else b.detach(),
                 None if r is None else r.detach(), act, g, y.detach(), grads, dtype)
    if r is not None:
        assert torch.equal(grads[-1], g)
    with torch.no_grad():
        assert torch.equal(dense.linear(x, w, b, act, r), y)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_linear_activations(act, dtype, cuda_device):
    """Every activation on p over a wide range, with residual."""
    from ictc_o2_hp_b200 import dense
    m, k, n = 150, 40, 72
    x = rand((m, k), dtype, cuda_device, 11, 3.0).requires_grad_(True)
    w = rand((n, k), dtype, cuda_device, 12, 1.0).requires_grad_(True)
    b = rand((n,), dtype, cuda_device, 13).requires_grad_(True)
    r = rand((m, n), dtype, cuda_device, 14)
    g = rand((m, n), dtype, cuda_device, 15)
    y = dense.linear(x, w, b, act, r)
    grads = torch.autograd.grad(y, (x, w, b), g)
    check_linear(x.detach(), w.detach(), b.detach(), r, act, g, y.detach(), grads, dtype)


@pytest.mark.parametrize("rows", [4, 5000])
def test_gelu_to_float32_rounding(rows, cuda_device):
    """gelu and its slope by themselves (one input and a weight of 1: p is exact), also in
    the tail, where the normal tail Q is all there is: its exponential is off by 1.5 p^2 U
    (the rounded argument) and 4 U, what multiplies it by some 12 U."""
    from ictc_o2_hp_b200 import dense
    p = torch.linspace(-8, 8, rows * 13, device=cuda_device).reshape(rows, 13)
    x = p.reshape(-1, 1).clone().requires_grad_(True)
    w = torch.ones(1, 1, device=cuda_device)
    y = dense.linear(x, w, None, "gelu")
    slope = torch.autograd.grad(y, x, torch.ones_like(y))[0]
    q = x.detach().double()
    tail = 0.5 * torch.special.erfc(q.abs() * math.sqrt(0.5))
    off = tail * (16 + 3 * q * q) * U
    below = 0.5 * torch.special.erfc(-q * math.sqrt(0.5))  # the distribution function
    want = q * below
    within("y", y.detach(), want, q.abs() * (off + U * (q > 0)) + 2 * U * want.abs())
    density = torch.exp(-0.5 * q * q) / math.sqrt(2 * math.pi)
    want = below + q * density
    within("slope", slope, want, off + U * (q > 0) + q.abs() * density * (8 + 1.5 * q * q) * U +
           2 * U * want.abs())


@pytest.mark.parametrize("rows", [3, 40, 700])
@pytest.mark.parametrize("act", ACTS)
def test_activations_far_from_zero(act, rows, cuda_device):
    """Finite p up to the end of float32: the activation is p or 0, its slope 1 or 0."""
    from ictc_o2_hp_b200 import dense
    p = torch.tensor([200.0, 3e3, 1e10, 1e19, 5e19, 1e25, 1e38, 3.4e38], device=cuda_device)
    p = torch.cat([p, -p]).repeat(rows, 1)
    x = p.reshape(-1, 1).clone().requires_grad_(True)
    w = torch.ones(1, 1, device=cuda_device)
    y = dense.linear(x, w, None, act)
    slope = torch.autograd.grad(y, x, torch.ones_like(y))[0]
    full = torch.ones_like(x, dtype=torch.bool) if act == "none" else x.detach() > 0
    assert torch.equal(y.detach(), torch.where(full, x.detach(), torch.zeros_like(y)))
    assert torch.equal(slope, full.float())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(16, 4096, 520), (700, 1024, 768), (4096, 256, 256),
                                   (20000, 64, 64), (33, 8200, 24), (40000, 24, 8)])
def test_linear_larger(shape, dtype, cuda_device):
    """K split over the SMs, several tiles per CTA, long sums over the rows."""
    from ictc_o2_hp_b200 import dense
    m, k, n = shape
    x = rand((m, k), dtype, cuda_device, 21).requires_grad_(True)
    w = rand((n, k), dtype, cuda_device, 22, 1.5 / math.sqrt(k)).requires_grad_(True)
    b = rand((n,), dtype, cuda_device, 23).requires_grad_(True)
    g = rand((m, n), dtype, cuda_device, 25)
    y = dense.linear(x, w, b, "silu")
    grads = torch.autograd.grad(y, (x, w, b), g)
    check_linear(x.detach(), w.detach(), b.detach(), None, "silu", g, y.detach(), grads, dtype)
    again = torch.autograd.grad(dense.linear(x, w, b, "silu"), (x, w, b), g)
    assert all(torch.equal(p, q) for p, q in zip(grads, again)), "not the same bits twice"


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_narrow_many_tiles(dtype, cuda_device):
    """Many tiles per CTA: a stage that is written again while it is still read shows as
    another tile's rows, in a few rows of a million."""
    from ictc_o2_hp_b200 import dense
    m, k, n = 700001, 64, 64
    x = rand((m, k), dtype, cuda_device, 71)
    w = rand((n, k), dtype, cuda_device, 72, 0.2)
    g = rand((m, n), dtype, cuda_device, 73)
    p = x.double() @ w.double().t()
    bound = sum_error(k) * (x.double().abs() @ w.double().abs().t())
    within("y", dense.linear(x, w), p, bound + (UNIT[dtype] + 2 * U) * p.abs() + TINY[dtype])
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    first = None
    for _ in range(8):
        y = dense.linear(*leaves, activation="silu", residual=g)
        out = (y.detach(), *torch.autograd.grad(y, leaves, g))
        first = out if first is None else first
        assert all(torch.equal(a, b) for a, b in zip(out, first))


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_narrow_many_odd_tiles(dtype, cuda_device):
    """The same over rows that are not whole 16-byte blocks, whose values are read one by
    one: every slot of the ring is written again many times."""
    from ictc_o2_hp_b200 import dense
    m, k, n = 700001, 61, 59
    x = rand((m, k), dtype, cuda_device, 75)
    w = rand((n, k), dtype, cuda_device, 76, 0.2)
    g = rand((m, n), dtype, cuda_device, 77)
    p = x.double() @ w.double().t()
    bound = sum_error(k) * (x.double().abs() @ w.double().abs().t())
    within("y", dense.linear(x, w), p, bound + (UNIT[dtype] + 2 * U) * p.abs() + TINY[dtype])
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    first = None
    for _ in range(8):
        y = dense.linear(*leaves, activation="silu", residual=g)
        out = (y.detach(), *torch.autograd.grad(y, leaves, g))
        if first is None:
            first = out
            check_linear(x, w, None, g, "silu", g, out[0], out[1:], dtype)
        assert all(torch.equal(a, b) for a, b in zip(out, first))


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_strides_and_batches(dtype, cuda_device):
    """Column slices (rows off every vector boundary), transposed weights, expanded
    gradients and leading batch dimensions."""
    from ictc_o2_hp_b200 import dense
    big = rand((70, 3, 90), dtype, cuda_device, 31)
    wide = rand((50, 120), dtype, cuda_device, 32, 0.2)
    res = rand((70, 3, 77), dtype, cuda_device, 33)
    for x in (big[..., 1:41], big[:, :, :40], big[:, 1, 3:43], big[..., ::2][..., :40]):
        for w in (wide[:, 2:42], wide[:24, 5:45], wide.t()[:40].t().contiguous().t().t(),
                  wide[:40, :50].t()):
            n = w.shape[0]
            r = res[..., 9:9 + n] if x.dim() == 3 else res[:, 2, 1:1 + n]
            xx, ww = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
            y = dense.linear(xx, ww, None, "gelu", r)
            g = rand((1,), dtype, cuda_device, 34).expand(y.shape)
            grads = torch.autograd.grad(y, (xx, ww), g)
            flat = x.reshape(-1, 40)
            check_linear(flat, w, None, r.reshape(-1, n), "gelu", g.reshape(-1, n),
                         y.detach().reshape(-1, n), (grads[0].reshape(-1, 40), grads[1]), dtype)


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("shape", [(1100, 100000, 1100), (96, 60000, 520), (70, 40001, 40)])
def test_linear_long_sums_of_one_sign(shape, dtype, cuda_device):
    """The tensor core truncates each time it adds 16 products to an accumulator (by up to
    2 U of it, which grows to the sum), always to the same side of a sum of one sign.
    Sums over more than 16,384 elements are taken in parts of at most 8,192; seen in the
    float32 value before the activation, which is not rounded to 16 bits."""
    from ictc_o2_hp_b200 import dense
    m, k, n = shape
    x = rand((m, k), dtype, cuda_device, 46).abs()
    w = rand((n, k), dtype, cuda_device, 47, 0.01).abs()
    p = dense._load().linear_forward(x, w, None, None, dense.ACTIVATIONS["silu"], True)[1]
    want = x.double() @ w.double().t()
    within("p", p, want, (1024 + 64) * U * want)


THIN = [1, 2, 3, 5, 7, 8]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("small", THIN)
@pytest.mark.parametrize("side", ["rows", "in", "out"])
def test_linear_thin(side, small, dtype, cuda_device):
    """A dimension of at most eight: every form, with rows on and off the 16-byte boundaries
    and lengths that no lane, strip or unrolled step divides."""
    from ictc_o2_hp_b200 import _lib, dense
    sizes = [(9, 9), (37, 64), (128, 33), (301, 1029), (1026, 2056), (40001, 24), (6001, 70)]
    for i, (one, two) in enumerate(sizes):
        if side == "rows":
            m, k, n = small, one % 5000 + 8, two
        elif side == "in":
            m, k, n = one, small, two
        else:
            m, k, n = one, two, small
        act = ACTS[(i + small) % len(ACTS)]
        x = rand((m, k), dtype, cuda_device, 1).requires_grad_(True)
        w = rand((n, k), dtype, cuda_device, 2, 1.5 / math.sqrt(k)).requires_grad_(True)
        b = rand((n,), dtype, cuda_device, 3).requires_grad_(True)
        r = rand((m, n), dtype, cuda_device, 4) if i % 2 else None
        g = rand((m, n), dtype, cuda_device, 5)
        y = dense.linear(x, w, b, act, r)
        grads = torch.autograd.grad(y, (x, w, b), g)
        check_linear(x.detach(), w.detach(), b.detach(), r, act, g, y.detach(), grads, dtype)
        again = torch.autograd.grad(dense.linear(x, w, b, act, r), (x, w, b), g)
        assert all(torch.equal(p, q) for p, q in zip(grads, again)), "not the same bits twice"
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(6, 90, 70), (500, 90, 6), (500, 6, 90), (3, 6, 5), (500, 64, 8)])
def test_linear_thin_strides(shape, dtype, cuda_device):
    """Slices, transposed weights, repeated rows and expanded gradients in the thin forms."""
    from ictc_o2_hp_b200 import dense
    m, k, n = shape
    big = rand((m + 3, 2 * k + 9), dtype, cuda_device, 31)
    wide = rand((2 * n + 9, 2 * k + 9), dtype, cuda_device, 32, 0.2)
    res = rand((m, n + 9), dtype, cuda_device, 33)
    b = rand((n,), dtype, cuda_device, 35)
    for x in (big[:m, :k], big[3:, 1:k + 1], big[:m, :2 * k:2], big[:1, :k].expand(m, k)):
        for w in (wide[:n, 8:k + 8], wide[n:2 * n, 3:k + 3], wide.t()[:n, :k]):
            if w.shape != (n, k):
                continue
            for r, g in ((res[:, 1:n + 1], rand((m, n), dtype, cuda_device, 36)),
                         (res[:, :n], rand((1,), dtype, cuda_device, 37).expand(m, n)),
                         (None, rand((m, n + 3), dtype, cuda_device, 38)[:, 3:])):
                leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
                y = dense.linear(*leaves, "silu", r)
                grads = torch.autograd.grad(y, leaves, g)
                check_linear(x, w, b, r, "silu", g, y.detach(), grads, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(300007, 21, 2), (300007, 2, 21), (2, 300, 4001), (4100, 9000, 1)])
def test_linear_thin_large(shape, dtype, cuda_device):
    """Many blocks of rows: sums joined over CTAs, rows off the boundaries."""
    from ictc_o2_hp_b200 import dense
    m, k, n = shape
    x = rand((m, k), dtype, cuda_device, 41).requires_grad_(True)
    w = rand((n, k), dtype, cuda_device, 42, 1.5 / math.sqrt(k)).requires_grad_(True)
    b = rand((n,), dtype, cuda_device, 43).requires_grad_(True)
    g = rand((m, n), dtype, cuda_device, 45)
    y = dense.linear(x, w, b, "gelu")
    grads = torch.autograd.grad(y, (x, w, b), g)
    check_linear(x.detach(), w.detach(), b.detach(), None, "gelu", g, y.detach(), grads, dtype)


def test_views_with_a_negative_bit(cuda_device):
    """The imaginary part of a conjugate is the memory's negative: as rows of one column and
    one bias it is read where it lies."""
    from ictc_o2_hp_b200 import dense
    z = torch.complex(*(rand((40, 1), torch.float32, cuda_device, s) for s in (36, 37)))
    x = z.conj().imag
    assert x.is_neg()
    plain = x.resolve_neg()
    w = rand((3, 1), torch.float32, cuda_device, 38)
    one = torch.complex(*(rand((1,), torch.float32, cuda_device, s) for s in (39, 40))).conj().imag
    assert torch.equal(dense.linear(x, w), dense.linear(plain, w))
    assert torch.equal(dense.linear(plain, x[:5]), dense.linear(plain, plain[:5]))
    assert torch.equal(dense.linear(plain, w[:1], one), dense.linear(plain, w[:1],
                                                                    one.resolve_neg()))
    assert torch.equal(dense.layer_norm(x, one, one),
                       dense.layer_norm(plain, one.resolve_neg(), one.resolve_neg()))
    leaf = plain.clone().requires_grad_(True)
    y = dense.linear(leaf, w[:1], None, "silu")
    assert torch.equal(*(torch.autograd.grad(y, leaf, g, retain_graph=True)[0]
                         for g in (x, plain)))


@pytest.mark.parametrize("rows", [2, 64])
def test_linear_float32_range(rows, cuda_device):
    """Magnitudes from 1e-30 to 1e30: the cut into bf16 parts keeps every bit."""
    from ictc_o2_hp_b200 import dense
    scale = 10.0 ** torch.linspace(-30, 30, 96, device=cuda_device, dtype=torch.float64)
    x = (rand((rows, 96), torch.float32, cuda_device, 41).double() * scale).float()
    w = (rand((40, 96), torch.float32, cuda_device, 42).double() / scale).float()
    y = dense.linear(x, w)
    within("y", y, x.double() @ w.double().t(),
           sum_error(96) * (x.double().abs() @ w.double().abs().t()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 150])
def test_linear_nonfinite(rows, dtype, cuda_device):
    """An infinity or NaN reaches exactly the outputs that a product in order gives it,
    with its sign; the others keep their values."""
    from ictc_o2_hp_b200 import dense
    k, n = 72, 140
    x = rand((rows, k), dtype, cuda_device, 51)
    w = rand((n, k), dtype, cuda_device, 52)
    clean = dense.linear(x, w)
    w[:, 7] = 1.0
    w[5, 7] = -2.0
    w[9, 7] = 0.0
    x2 = x.clone()
    x2[1, 7] = math.inf
    x2[2, 3] = math.nan
    w2 = w.clone()
    w2[20, 30] = -math.inf
    y = dense.linear(x2, w2)
    want = x2.double() @ w2.double().t()
    assert torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y.isinf(), want.isinf())
    assert torch.equal(y[y.isinf()].double(), want[y.isinf()])
    assert y[1, 0] == math.inf and y[1, 5] == -math.inf and y[1, 9].isnan()
    assert y[2].isnan().all() and y[0, 20].isinf()
    base = dense.linear(x, w)
    keep = want.isfinite()
    assert torch.equal(y[keep], base[keep]) and clean.isfinite().all()


@pytest.mark.parametrize("shape", [(700, 48, 40), (700, 48, 140)])
def test_linear_nonfinite_gradients(shape, cuda_device):
    """Infinities and NaN in the gradient and in x reach the sums they belong to."""
    from ictc_o2_hp_b200 import dense
    m, k, n = shape
    x = rand((m, k), torch.float32, cuda_device, 55)
    w = rand((n, k), torch.float32, cuda_device, 56)
    g = rand((m, n), torch.float32, cuda_device, 57)

    def grads(x, w, g):
        leaves = [t.clone().requires_grad_(True) for t in (x, w)]
        return torch.autograd.grad(dense.linear(*leaves), leaves, g)

    base = grads(x, w, g)
    x2, w2, g2 = x.clone(), w.clone(), g.clone()
    x2[300, 5] = math.inf
    g2[20, 7] = -math.inf
    g2[650, 30] = math.nan
    w2[3, 9] = math.inf
    got = grads(x2, w2, g2)
    want = (g2.double() @ w2.double(), g2.double().t() @ x2.double())
    for p, q, r in zip(got, want, base):
        assert torch.equal(p.isnan(), q.isnan()) and torch.equal(p.isinf(), q.isinf())
        assert torch.equal(p[p.isinf()].double(), q[q.isinf()])
        keep = q.isfinite()
        assert keep.any() and torch.equal(p[keep], r[keep])


@pytest.mark.parametrize("shape", [(1048576, 64, 64), (262147, 61, 59), (65536, 128, 512),
                                   (300000, 96, 72), (40000, 65, 30)])
def test_linear_nonfinite_rows_of_many(shape, cuda_device):
    """A row of NaN, an infinity: every weight gradient that they reach, over long sums, for
    the cost of a clean step (the extra time allowed is that of launching it)."""
    from ictc_o2_hp_b200 import _lib, dense
    m, k, n = shape
    x = rand((m, k), torch.float32, cuda_device, 58)
    w = rand((n, k), torch.float32, cuda_device, 59, 1.5 / math.sqrt(k))
    g = rand((m, n), torch.float32, cuda_device, 60)

    def step(x, w, g):
        leaves = [t.clone().requires_grad_(True) for t in (x, w)]
        y = dense.linear(*leaves, activation="silu")
        return y.detach(), *torch.autograd.grad(y, leaves, g)

    def cost(*args):
        start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        for i in range(6):
            if i == 2:
                start.record()
            out = step(*args)
        stop.record()
        torch.cuda.synchronize()
        return out, start.elapsed_time(stop) / 4

    base, clean = cost(x, w, g)
    x2 = x.clone()
    x2[m // 2] = math.nan
    (y, dx, dw), spent = cost(x2, w, g)
    keep = torch.ones(m, dtype=torch.bool, device=cuda_device)
    keep[m // 2] = False
    assert y[m // 2].isnan().all() and dx[m // 2].isnan().all() and dw.isnan().all()
    assert torch.equal(y[keep], base[0][keep]) and torch.equal(dx[keep], base[1][keep])
    assert spent <= 2 * clean + 0.5, f"{spent:.2f} ms with a NaN row, {clean:.2f} without"
    g2 = g.clone()
    g2[m // 3, 5] = math.inf
    (y, dx, dw), spent = cost(x, w, g2)
    slope = torch.autograd.functional.jvp(
        lambda p: p * torch.sigmoid(p), x[m // 3].double() @ w[5].double(),
        torch.ones((), dtype=torch.float64, device=cuda_device))[1].sign()
    assert torch.equal(dw[5], x[m // 3].sign() * math.inf * slope.float())
    assert torch.equal(y, base[0])
    assert dw[torch.arange(n, device=cuda_device) != 5].isfinite().all()
    assert torch.equal(dx[m // 3], w[5].sign() * math.inf * slope.float())
    assert spent <= 2 * clean + 0.5, f"{spent:.2f} ms with an infinity, {clean:.2f} without"
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_empty_and_partial_gradients(dtype, cuda_device):
    from ictc_o2_hp_b200 import dense
    w = rand((6, 5), dtype, cuda_device, 61).requires_grad_(True)
    b = rand((6,), dtype, cuda_device, 62).requires_grad_(True)
    x = torch.empty(0, 5, dtype=dtype, device=cuda_device, requires_grad=True)
    y = dense.linear(x, w, b, "silu")
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (0, 6) and gx.shape == (0, 5)
    assert not gw.any() and not gb.any()
    x = rand((30, 5), dtype, cuda_device, 63).requires_grad_(True)
    g = rand((30, 6), dtype, cuda_device, 64)
    full = torch.autograd.grad(dense.linear(x, w, b, "gelu"), (x, w, b), g)
    for i, t in enumerate((x, w, b)):
        others = [q if q is t else q.detach() for q in (x, w, b)]
        alone = torch.autograd.grad(dense.linear(*others, "gelu"), t, g)[0]
        assert torch.equal(alone, full[i])


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_batch_with_create_graph(dtype, act, cuda_device):
    """No rows, gradients that are differentiated again: zeros, as without create_graph."""
    from ictc_o2_hp_b200 import dense
    w = rand((6, 5), dtype, cuda_device, 65).requires_grad_(True)
    b = rand((6,), dtype, cuda_device, 66).requires_grad_(True)
    scale = rand((6,), dtype, cuda_device, 67).requires_grad_(True)
    x = torch.empty(0, 5, dtype=dtype, device=cuda_device, requires_grad=True)
    leaves = (x, w, b, scale)
    y = dense.layer_norm(dense.linear(x, w, b, act), scale)
    first = torch.autograd.grad(y, leaves, torch.empty_like(y), create_graph=True)
    assert [g.shape for g in first] == [t.shape for t in leaves]
    assert not any(g.any() for g in first)
    total = sum((g.float() ** 2).sum() for g in first)
    second = torch.autograd.grad(total, leaves, allow_unused=True)
    assert all(g is None or (g.shape == t.shape and not g.any()) for g, t in zip(second, leaves))


# -------------------------------------------------------------------- layer norm


def norm64(x, w, b, eps, g):
    x, g = x.double(), g.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    u = (x - mean) * rstd
    w64 = torch.ones_like(x[0]) if w is None else w.double()
    y = u * w64 + (0 if b is None else b.double())
    h = g * w64
    mh, mhu = h.mean(-1, keepdim=True), (h * u).mean(-1, keepdim=True)
    return mean, rstd, u, y, h, rstd * (h - mh - u * mhu), (g * u).sum(0), g.sum(0)


def check_norm(x, w, b, eps, g, y, grads, dtype, pdtype):
    u8, c, rows = UNIT[dtype], x.shape[-1], x.shape[0]
    up = UNIT[pdtype]
    mean, rstd, u, y64, h, dx, dw, db = norm64(x, w, b, eps, g)
    aw = torch.ones_like(u[0]) if w is None else w.double().abs()
    # u = (x - mean) rstd: the mean is off by chain U mean|x|, which shifts u by that
    # times rstd; rstd by twice the chain
    chain = (40 + c / 256) * U
    shift = x.double().abs().mean(-1, keepdim=True) * rstd
    eu = chain * (shift + x.double().abs() * rstd * 0.1 + 4 * u.abs() + shift * u.abs())
    within("y", y, y64, eu * aw + (u8 + 4 * U) * (
        y64.abs() + 0.1 * (0 if b is None else b.double().abs())) + TINY[dtype])
    if grads is None:
        return
    ah = h.abs()
    mah, mahu = ah.mean(-1, keepdim=True), (ah * (u.abs() + eu)).mean(-1, keepdim=True)
    e = rstd * (2 * chain * (1 + shift) * (ah + mah + u.abs() * mahu) + eu * mahu +
                u.abs() * (ah * eu).mean(-1, keepdim=True))
    within("dx", grads[0], dx, e + (u8 + 4 * U) * (dx.abs() + e) + TINY[dtype])
    long = (64 + rows) * U
    ag = g.double().abs()
    if w is not None:
        e = (ag * eu).sum(0) + long * (ag * u.abs()).sum(0)
        within("dweight", grads[1], dw, e + (up + 4 * U) * (dw.abs() + e) + TINY[pdtype])
    if b is not None:
        e = long * ag.sum(0)
        within("dbias", grads[-1], db, e + (up + 4 * U) * (db.abs() + e) + TINY[pdtype])


NORM_SHAPES = [(1, 1), (1, 64), (5, 2), (3, 7), (1000, 64), (129, 33), (77, 128), (64, 255),
               (33, 896), (50, 1337), (20, 4096), (9, 5000), (6, 8192), (7, 8193), (5, 12288),
               (4, 16384), (3, 16385), (2, 40000), (100000, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_layer_norm_against_float64(shape, dtype, cuda_device):
    from ictc_o2_hp_b200 import dense
    rows, c = shape
    pdtype = torch.float32 if rows % 2 else dtype
    x = rand((rows, c), dtype, cuda_device, 71, 1.5, 0.5).requires_grad_(True)
    w = rand((c,), pdtype, cuda_device, 72, 0.2, 1.0).requires_grad_(True)
    b = rand((c,), pdtype, cuda_device, 73, 0.2).requires_grad_(True)
    g = rand((rows, c), dtype, cuda_device, 74)
    y = dense.layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), g)
    check_norm(x.detach(), w.detach(), b.detach(), 1e-5, g, y.detach(), grads, dtype, pdtype)
    with torch.no_grad():
        assert torch.equal(dense.layer_norm(x, w, b), y)
    again = torch.autograd.grad(dense.layer_norm(x, w, b), (x, w, b), g)
    assert all(torch.equal(p, q) for p, q in zip(grads, again)), "not the same bits twice"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("affine", ["none", "weight", "bias"])
def test_layer_norm_parameters(affine, dtype, cuda_device):
    from ictc_o2_hp_b200 import dense
    x = rand((40, 3, 100), dtype, cuda_device, 81, 2.0, -1.0).requires_grad_(True)
    w = rand((100,), dtype, cuda_device, 82).requires_grad_(True) if affine == "weight" else None
    b = rand((100,), dtype, cuda_device, 83).requires_grad_(True) if affine == "bias" else None
    g = rand((40, 3, 100), dtype, cuda_device, 84)
    y = dense.layer_norm(x, w, b, 1e-3)
    grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], g)
    flat = [t.detach().reshape(120, 100) for t in (x, g, y, grads[0])]
    check_norm(flat[0], w, b, 1e-3, flat[1], flat[2], (flat[3], *grads[1:]), dtype, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [24, 64, 1000])
def test_layer_norm_strides(width, dtype, cuda_device):
    """Row slices at every offset, an expanded row, an expanded gradient."""
    from ictc_o2_hp_b200 import dense
    big = rand((60, width + 9), dtype, cuda_device, 91)
    w = rand((width,), dtype, cuda_device, 92)
    for x in [big[:, o:o + width] for o in (0, 1, 8)] + [big[:1, :width].expand(60, width)]:
        xx = x.detach().requires_grad_(True)
        y = dense.layer_norm(xx, w, None)
        g = rand((60, 1), dtype, cuda_device, 93).expand(60, width)
        grads = torch.autograd.grad(y, xx, g)
        check_norm(x, w, None, 1e-5, g, y.detach(), (grads[0],
                   norm64(x, w, None, 1e-5, g)[6].to(dtype)), dtype, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [24, 64, 1000, 8200])
def test_layer_norm_parameter_gradients_over_strides(width, dtype, cuda_device):
    """The column sums over row slices at every offset, an expanded row, expanded and sliced
    gradients: blocks at the tensors' ends, strides of 0, rows wider than a CTA holds."""
    from ictc_o2_hp_b200 import dense
    big = rand((60, width + 9), dtype, cuda_device, 94, 1.0, 0.3)
    wide = rand((60, width + 9), dtype, cuda_device, 95)
    w = rand((width,), dtype, cuda_device, 96)
    b = rand((width,), dtype, cuda_device, 97)
    rows = [big[:, o:o + width] for o in (0, 1, 8)] + [big[:1, :width].expand(60, width)]
    grads = [wide[:, o:o + width] for o in (0, 3, 8)] + [
        wide[:1, 1:width + 1].expand(60, width), wide[:, :1].expand(60, width)]
    for x in rows:
        for g in grads:
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
            y = dense.layer_norm(*leaves)
            got = torch.autograd.grad(y, leaves, g)
            check_norm(x, w, b, 1e-5, g, y.detach(), got, dtype, dtype)


def test_layer_norm_large_mean_and_constant_rows(cuda_device):
    """A mean far above the spread loses only what float32 inputs lose; constant rows
    give the bias."""
    from ictc_o2_hp_b200 import dense
    x = rand((50, 300), torch.float32, cuda_device, 101, 1.0, 1000.0)
    g = rand((50, 300), torch.float32, cuda_device, 102)
    x.requires_grad_(True)
    y = dense.layer_norm(x)
    grads = torch.autograd.grad(y, x, g)
    check_norm(x.detach(), None, None, 1e-5, g, y.detach(), grads, torch.float32, torch.float32)
    b = rand((64,), torch.float32, cuda_device, 103)
    flat = torch.full((10, 64), 0.75, device=cuda_device)
    assert torch.equal(dense.layer_norm(flat, None, b), b.expand(10, 64))


@pytest.mark.parametrize("width", [3, 41, 300, 896, 1337, 5000, 20000])
def test_layer_norm_mean_correction(width, cuda_device):
    """The mean is that of the row, not a rounded sum times a rounded 1 / width: constant
    rows give the bias, and rows far from zero are centred to the last bit that they hold.
    The mean kept for the backward is off by at most its own rounding (U |mean|) and that of
    sums over deviations, which stay below 2 sigma + 0.3 |mean| 2^-18 on average."""
    from ictc_o2_hp_b200 import dense
    b = rand((width,), torch.float32, cuda_device, 104)
    for value in (0.1, 1000.0, 1e5, -12345.678):
        flat = torch.full((7, width), value, device=cuda_device)
        assert torch.equal(dense.layer_norm(flat, None, b), b.expand(7, width))
    chain = (40 + width / 256) * U
    for mean in (1000.0, 1e5):
        x = rand((9, width), torch.float32, cuda_device, 105, 1.0, mean)
        y, got_mean, got_rstd = dense._load().norm_forward(x, None, None, 1e-5)
        want_mean, rstd, u = norm64(x, None, None, 1e-5, x)[:3]
        spread = 2 / rstd.squeeze(-1) + 0.3 * mean * 2.0 ** -18
        within("mean", got_mean, want_mean.squeeze(-1), 1.01 * U * mean + chain * spread)
        within("rstd", got_rstd, rstd.squeeze(-1), 3 * chain * rstd.squeeze(-1))
        within("y", y, u, chain * (2 + 0.3 * mean * 2.0 ** -18 * rstd + 4 * u.abs()))


def test_layer_norm_empty_and_nonfinite(cuda_device):
    from ictc_o2_hp_b200 import dense
    w = torch.ones(8, device=cuda_device, requires_grad=True)
    x = torch.empty(0, 8, device=cuda_device, requires_grad=True)
    y = dense.layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == gx.shape == (0, 8) and not gw.any()
    x = rand((20, 64), torch.float32, cuda_device, 111)
    base = dense.layer_norm(x)
    x[3, 5], x[7, 0] = math.nan, math.inf
    y = dense.layer_norm(x)
    bad = torch.zeros(20, dtype=torch.bool, device=cuda_device)
    bad[3] = bad[7] = True
    assert y[bad].isnan().all() and torch.equal(y[~bad], base[~bad])


# ------------------------------------------------- differences and second derivatives


def test_gradients_against_differences(cuda_device):
    """Directional derivatives against central differences of the float64 formulas."""
    from ictc_o2_hp_b200 import dense
    m, k, n, h = 40, 24, 32, 1e-5
    x, w, b = (rand(s, torch.float32, cuda_device, i) for i, s in enumerate(
        [(m, k), (n, k), (n,)]))
    g = rand((m, n), torch.float32, cuda_device, 9)
    gn = rand((m, k), torch.float32, cuda_device, 10)
    nw, nb = rand((k,), torch.float32, cuda_device, 11), rand((k,), torch.float32, cuda_device, 12)

    def total(x, w, b, act):
        return (act64(x @ w.t() + b, act) * g.double()).sum()

    def total_norm(x, w, b):
        return (norm64(x, w, b, 1e-5, gn)[3] * gn.double()).sum()

    def differences(f, point):
        for i, t in enumerate(point):
            v = rand(t.shape, torch.float32, cuda_device, 20 + i).double()
            plus = [q.double() + h * v if j == i else q.double() for j, q in enumerate(point)]
            minus = [q.double() - h * v if j == i else q.double() for j, q in enumerate(point)]
            yield v, (f(*plus) - f(*minus)).item() / (2 * h)

    for act in ACTS[:1] + ACTS[2:]:
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        grads = torch.autograd.grad(dense.linear(*leaves, act), leaves, g)
        for grad, (v, slope) in zip(grads, differences(lambda *a: total(*a, act), (x, w, b))):
            size = (grad.double().abs() * v.abs()).sum().item()
            assert abs((grad.double() * v).sum().item() - slope) <= 1e-5 * size
    leaves = [t.clone().requires_grad_(True) for t in (x, nw, nb)]
    grads = torch.autograd.grad(dense.layer_norm(*leaves), leaves, gn)
    for grad, (v, slope) in zip(grads, differences(total_norm, (x, nw, nb))):
        size = (grad.double().abs() * v.abs()).sum().item()
        assert abs((grad.double() * v).sum().item() - slope) <= 1e-5 * size


@pytest.mark.parametrize("act", ACTS)
def test_second_derivatives(act, cuda_device):
    """A force-like loss: squared input gradients, differentiated by every operand."""
    from ictc_o2_hp_b200 import dense
    m, k, n = 50, 24, 40
    base = [rand((m, k), torch.float32, cuda_device, 1),
            rand((n, k), torch.float32, cuda_device, 2, 0.3),
            rand((n,), torch.float32, cuda_device, 3),
            rand((k,), torch.float32, cuda_device, 4, 0.2, 1.0),
            rand((k,), torch.float32, cuda_device, 5)]
    g = rand((m, n), torch.float32, cuda_device, 6)

    def loss(x, w, b, nw, nb, g, lin, norm):
        e = (lin(norm(x, nw, nb), w, b) * g).sum()
        f = torch.autograd.grad(e, x, create_graph=True)[0]
        return (f * f).sum()

    ours = [t.clone().requires_grad_(True) for t in base]
    got = torch.autograd.grad(loss(*ours, g, lambda x, w, b: dense.linear(x, w, b, act),
                                   dense.layer_norm), ours, allow_unused=True)
    wide = [t.double().requires_grad_(True) for t in base]
    want = torch.autograd.grad(
        loss(*wide, g.double(), lambda x, w, b: act64(x @ w.t() + b, act),
             lambda x, w, b: torch.nn.functional.layer_norm(x, (k,), w, b, 1e-5)),
        wide, allow_unused=True)
    for p, q in zip(got, want):
        if q is None or not q.any():
            assert p is None or not p.any()
            continue
        assert (p.double() - q).norm() <= 1e-5 * q.norm()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_create_graph_keeps_first_gradients(act, dtype, cuda_device):
    """The gradients that are differentiated again keep the error bounds of those that are
    not; p far from zero, where rounding it to 16 bits would move the slope."""
    from ictc_o2_hp_b200 import dense
    m, k, n = 150, 40, 72
    x = rand((m, k), dtype, cuda_device, 16, 2.0).requires_grad_(True)
    w = rand((n, k), dtype, cuda_device, 17, 0.3).requires_grad_(True)
    b = rand((n,), dtype, cuda_device, 18).requires_grad_(True)
    g = rand((m, n), dtype, cuda_device, 19)
    y = dense.linear(x, w, b, act)
    grads = torch.autograd.grad(y, (x, w, b), g, create_graph=True)
    assert all(t.requires_grad for t in grads[:2])
    check_linear(x.detach(), w.detach(), b.detach(), None, act, g, y.detach(),
                 [t.detach() for t in grads], dtype)


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("act", ACTS)
def test_second_derivatives_16_bit(act, dtype, cuda_device):
    """As above in 16-bit types: some six tensors between the operands and a second
    derivative are rounded, and the squares double what is off: 16 u in the 2-norm."""
    from ictc_o2_hp_b200 import dense
    m, k, n = 50, 24, 40
    base = [rand((m, k), dtype, cuda_device, 1), rand((n, k), dtype, cuda_device, 2, 0.3),
            rand((n,), dtype, cuda_device, 3)]
    g = rand((m, n), dtype, cuda_device, 6)

    def loss(x, w, b, g, lin):
        f = torch.autograd.grad((lin(x, w, b) * g).sum(), x, create_graph=True)[0]
        return (f.float() ** 2).sum() if f.dtype != torch.float64 else (f ** 2).sum()

    ours = [t.clone().requires_grad_(True) for t in base]
    got = torch.autograd.grad(loss(*ours, g, lambda x, w, b: dense.linear(x, w, b, act)), ours,
                              allow_unused=True)
    wide = [t.double().requires_grad_(True) for t in base]
    want = torch.autograd.grad(
        loss(*wide, g.double(), lambda x, w, b: act64(x @ w.t() + b, act)), wide,
        allow_unused=True)
    for p, q in zip(got, want):
        if q is None or not q.any():
            assert p is None or not p.any()
            continue
        assert (p.double() - q).norm() <= 16 * UNIT[dtype] * q.norm()


# ----------------------------------------------------------- modules, streams, compile


def test_modules_match_torch(cuda_device):
    from ictc_o2_hp_b200 import LayerNorm, Linear, RadialTrunk, ResidualBlock
    torch.manual_seed(3)
    ours = Linear(20, 30, activation="silu").to(cuda_device)
    torch.manual_seed(3)
    theirs = torch.nn.Linear(20, 30).to(cuda_device)
    assert torch.equal(ours.weight, theirs.weight) and torch.equal(ours.bias, theirs.bias)
    theirs.load_state_dict(ours.state_dict())
    assert set(LayerNorm(8).state_dict()) == set(torch.nn.LayerNorm(8).state_dict())
    x = rand((9, 20), torch.float32, cuda_device, 1)
    want = torch.nn.functional.silu(theirs.double()(x.double()))
    assert (ours(x).double() - want).norm() <= 1e-6 * want.norm()
    block = ResidualBlock(20, 48).to(cuda_device)
    h = torch.nn.functional.layer_norm(x.double(), (20,))
    h = torch.nn.functional.silu(h @ block.up.weight.double().t() + block.up.bias.double())
    want = x.double() + h @ block.down.weight.double().t() + block.down.bias.double()
    assert (block(x).double() - want).norm() <= 1e-6 * want.norm()
    trunk = RadialTrunk(8, 64, blocks=2).to(cuda_device)
    out = trunk(rand((5, 11, 8), torch.float32, cuda_device, 2))
    assert out.shape == (5, 11, 64)
    assert out.mean(-1).abs().max() <= 1e-5


def test_trunk_feeds_the_radial_product(cuda_device):
    """Trunk, final affine layer and per-edge product together, against the same network
    of torch modules in front of the product."""
    from ictc_o2_hp_b200 import Linear, RadialTrunk, RadialUvuTensorProduct, UvuTensorProduct
    torch.manual_seed(0)
    tp = UvuTensorProduct(16, 1, 2, parity="full", parity_in2="canonical", shared_weights=False)
    product = RadialUvuTensorProduct(tp, Linear(32, tp.weight_numel)).to(cuda_device)
    trunk = RadialTrunk(8, 32).to(cuda_device)
    basis = rand((300, 8), torch.float32, cuda_device, 1)
    x = rand((300, tp.input1_dimension), torch.float32, cuda_device, 2)
    y = rand((300, tp.input2_dimension), torch.float32, cuda_device, 3)
    out = product(x, y, trunk(basis))
    f = torch.nn.functional

    def torch_trunk(b):
        h = f.silu(f.linear(b, trunk.embed.weight, trunk.embed.bias))
        for q in trunk.blocks:
            z = f.layer_norm(h, (32,), q.norm.weight, q.norm.bias)
            z = f.silu(f.linear(z, q.up.weight, q.up.bias))
            h = h + f.linear(z, q.down.weight, q.down.bias)
        return f.layer_norm(h, (32,), trunk.norm.weight, trunk.norm.bias)

    want = product(x, y, torch_trunk(basis))
    assert (out - want).norm() <= 1e-5 * want.norm()
    params = list(trunk.parameters())
    g = rand(out.shape, torch.float32, cuda_device, 4)
    for p, q in zip(torch.autograd.grad(out, params, g), torch.autograd.grad(want, params, g)):
        assert (p - q).norm() <= 1e-4 * q.norm()


def test_other_stream_and_graph_capture(cuda_device):
    """Work goes to the caller's stream: a captured graph replays on new inputs."""
    from ictc_o2_hp_b200 import dense
    x = rand((200, 96), torch.float32, cuda_device, 1)
    w = rand((96, 96), torch.float32, cuda_device, 2, 0.1)

    def block(x):
        return dense.linear(dense.layer_norm(x), w, None, "gelu", x)

    want = block(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    held = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        out = block(held)
    held.copy_(x)
    graph.replay()
    assert torch.equal(out, want)


def test_compile_fullgraph(cuda_device):
    from ictc_o2_hp_b200 import ResidualBlock
    torch.manual_seed(1)
    block = ResidualBlock(32).to(cuda_device)
    x = rand((64, 32), torch.float32, cuda_device, 1).requires_grad_(True)
    g = rand((64, 32), torch.float32, cuda_device, 2)
    want = torch.autograd.grad(block(x), (x, *block.parameters()), g)
    run = torch.compile(block, fullgraph=True, backend="aot_eager")
    got = torch.autograd.grad(run(x), (x, *block.parameters()), g)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_traces_record_the_operators(cuda_device):
    """torch.jit.trace and make_fx see the operators: a replay on other inputs computes with
    those."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from ictc_o2_hp_b200 import dense
    w = rand((32, 32), torch.float32, cuda_device, 2, 0.2)
    b = rand((32,), torch.float32, cuda_device, 3)
    first, second = (rand((50, 32), torch.float32, cuda_device, s) for s in (4, 5))
    g = rand((50, 32), torch.float32, cuda_device, 6)

    def block(x):
        return dense.linear(dense.layer_norm(x, None, b), w, b, "silu", x)

    def step(x):
        y = block(x)
        return y, torch.autograd.grad(y, x, g)[0]

    want = step(second.clone().requires_grad_(True))
    traced = torch.jit.trace(block, (first.clone().requires_grad_(True),), check_trace=False)
    leaf = second.clone().requires_grad_(True)
    y = traced(leaf)
    assert torch.equal(y, want[0])
    assert torch.equal(torch.autograd.grad(y, leaf, g)[0], want[1])
    recorded = make_fx(step)(first.clone().requires_grad_(True))
    got = recorded(second.clone().requires_grad_(True))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    # the backward alone is watched: its nodes were made outside
    leaf = second.clone().requires_grad_(True)
    y = block(leaf)
    back = make_fx(lambda g: torch.autograd.grad(y, leaf, g, retain_graph=True)[0])(g.clone())
    twice = torch.autograd.grad(y, leaf, 2 * g)[0]
    assert torch.equal(back(2 * g), twice) and not torch.equal(twice, want[1])
    with pytest.raises(RuntimeError):  # custom operators have no rules for these transforms
        torch.func.grad(lambda x: (block(x) * g).sum())(second)
    batches = second.reshape(5, 10, 32)
    assert torch.equal(torch.func.vmap(block)(batches), torch.stack([block(t) for t in batches]))


def test_autocast_casts_operands_of_different_types(cuda_device):
    """float32 parameters beside 16-bit activations, as torch.nn.Linear takes them under
    autocast; without it, and for operands of one type, nothing changes."""
    from ictc_o2_hp_b200 import Linear, dense
    layer = Linear(24, 40, activation="silu").to(cuda_device)
    x = rand((30, 24), torch.float16, cuda_device, 1).requires_grad_(True)
    r = rand((30, 40), torch.float32, cuda_device, 2)
    g = rand((30, 40), torch.bfloat16, cuda_device, 3)
    with pytest.raises(ValueError):
        layer(x, r)
    args = [t.detach().bfloat16().requires_grad_(True) for t in (x, layer.weight, layer.bias)]
    want = dense.linear(*args, "silu", r.bfloat16())
    grads = torch.autograd.grad(want, args, g)
    for run in (layer, torch.compile(layer, fullgraph=True, backend="aot_eager")):
        with torch.autocast("cuda", torch.bfloat16):
            y = run(x, r)
        got = torch.autograd.grad(y, (x, layer.weight, layer.bias), g)
        assert torch.equal(y, want)
        assert [t.dtype for t in got] == [torch.float16, torch.float32, torch.float32]
        assert all(torch.equal(p, q.to(p.dtype)) for p, q in zip(got, grads))
    with torch.autocast("cuda", torch.bfloat16):
        assert layer(x.float(), r).dtype == torch.float32
        with pytest.raises(TypeError):
            dense.linear(x.double(), layer.weight)


def test_dual_tensors_are_refused(cuda_device):
    """A tangent is not dropped silently, whichever operand carries it."""
    from torch.autograd import forward_ad

    from ictc_o2_hp_b200 import dense
    x, w, r = (rand((6, 6), torch.float32, cuda_device, s) for s in (1, 2, 3))
    b = rand((6,), torch.float32, cuda_device, 4)
    linear = [x, w, b, "none", r]
    for leaf in (False, True):
        with forward_ad.dual_level():
            for i in (0, 1, 2, 4):
                args = list(linear)
                args[i] = forward_ad.make_dual(args[i].clone().requires_grad_(leaf),
                                               torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    dense.linear(*args)
            for i in range(3):
                args = [x, b, b]
                args[i] = forward_ad.make_dual(args[i].clone(), torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    dense.layer_norm(*args)


def test_fake_tensors_forward_and_backward(cuda_device):
    from torch._subclasses.fake_tensor import FakeTensorMode

    from ictc_o2_hp_b200 import dense
    with FakeTensorMode():
        x = torch.empty(3, 7, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.empty(24, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        scale = torch.empty(24, device="cuda", requires_grad=True)
        y = dense.layer_norm(dense.linear(x, w, activation="silu"), scale)
        grads = torch.autograd.grad(y, (x, w, scale), torch.empty_like(y))
        assert [(g.shape, g.dtype) for g in grads] == [(t.shape, t.dtype) for t in (x, w, scale)]


def test_refusals(cuda_device):
    from ictc_o2_hp_b200 import dense
    x = torch.randn(4, 6, device=cuda_device)
    w = torch.randn(5, 6, device=cuda_device)
    with pytest.raises(TypeError):
        dense.linear(x.double(), w.double())
    with pytest.raises(TypeError):
        dense.layer_norm(x.double())
    bad = [
        lambda: dense.linear(x, w.half()),
        lambda: dense.linear(x, w[:, :5]),
        lambda: dense.linear(x, w[0]),
        lambda: dense.linear(x, w, torch.randn(6, device=cuda_device)),
        lambda: dense.linear(x, w, w[:, 0].cpu()),
        lambda: dense.linear(x, w, activation="swish"),
        lambda: dense.linear(x, w, residual=x),
        lambda: dense.linear(x, w, residual=torch.randn(1, 5, device=cuda_device)),
        lambda: dense.linear(x[:, :0], w[:, :0]),
        lambda: dense.layer_norm(x, w[0, :5]),
        lambda: dense.layer_norm(x, w[0].half()),
        lambda: dense.layer_norm(x.half(), w[0].bfloat16()),
        lambda: dense.layer_norm(x, w[0], w[0].half()),
        lambda: dense.layer_norm(x, eps=-1.0),
        lambda: dense.layer_norm(x[:, :0]),
        lambda: dense.LayerNorm(5).to(cuda_device)(x),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
