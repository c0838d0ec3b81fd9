"""The gated linear layer on the GPU against plain float64 formulas.

Tolerances are error bounds of the arithmetic, element by element, with U the unit roundoff
of float32 and u that of the operand type (test_dense_gpu.py has those of sums and
activations).  With e(t) the error of t, a = act(pg), s = act'(pg), pg and pu sums over k:
- e(a) <= 1.2 e(pg) + 16 U (|pg| + 1) and e(s) <= 1.1 e(pg) + 16 U (for relu: |s| <= 1 where pg
  is within its error of 0);
- y = a pu: e(a) (|pu| + e(pu)) + |a| e(pu), its rounding u |y|, one product in float32;
- dg = g pu s and du = g a: |g| times the same, a 16-bit backward rounds them (u |d|);
- dx, dW and db are sums over those.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_dense_gpu import ACTS, DTYPES, TINY, U, UNIT, act64, rand, slope64, sum_error, within

pytestmark = pytest.mark.gpu


def gated64(x, w, b, act, g):
    x, w, g = x.double(), w.double(), g.double()
    pg, pu = (x @ w.t() + (0 if b is None else b.double())).chunk(2, -1)
    a, s = act64(pg, act), slope64(pg, act)
    d = torch.cat([g * pu * s, g * a], -1)
    return pg, pu, a, s, a * pu, d, d @ w, d.t() @ x, d.sum(0)


def check_gated(x, w, b, act, g, y, grads, dtype):
    u, (m, k), n2 = UNIT[dtype], x.shape, w.shape[0]
    pg, pu, a, s, y64, d, dx, dw, db = gated64(x, w, b, act, g)
    ax, aw, ag = x.double().abs(), w.double().abs(), g.double().abs()
    ep = sum_error(k) * (ax @ aw.t() + (0 if b is None else b.double().abs()))
    epg, epu = ep.chunk(2, -1)
    own = 16 * U * (pg.abs() + 1) * (act != "none")
    ea = 1.2 * epg + own
    es = (1.1 * epg + 16 * U) * (act != "none")
    if act == "relu":
        es = (pg.abs() <= epg).double()
    tiny = TINY[dtype]
    ey = ea * (pu.abs() + epu) + a.abs() * epu
    within("y", y, y64, ey + (u + 2 * U) * (y64.abs() + ey) + tiny)
    if grads is None:
        return
    ed = torch.cat([ag * (es * (pu.abs() + epu) + s.abs() * epu), ag * ea], -1) + 4 * U * d.abs()
    eds = ed
    if dtype != torch.float32:
        ed = ed + u * (d.abs() + ed) + tiny
    ad = d.abs() + ed
    if grads[0] is not None:
        within("dx", grads[0], dx, ed @ aw + sum_error(n2) * (ad @ aw) + (u + 2 * U) * (
            dx.abs() + ed @ aw) + tiny)
    if grads[1] is not None:
        within("dweight", grads[1], dw, ed.t() @ ax + sum_error(m) * (ad.t() @ ax) +
               (u + 2 * U) * (dw.abs() + ed.t() @ ax) + tiny)
    if b is not None and grads[2] is not None:
        within("dbias", grads[2], db, eds.sum(0) + (m + 64) * U * ad.sum(0) + (u + 2 * U) * (
            db.abs() + eds.sum(0)) + tiny)


def operands(m, k, n, dtype, device, seed=0, bias=True):
    x = rand((m, k), dtype, device, seed + 1)
    w = rand((2 * n, k), dtype, device, seed + 2, 1.5 / math.sqrt(k))
    b = rand((2 * n,), dtype, device, seed + 3) if bias else None
    return x, w, b, rand((m, n), dtype, device, seed + 5)


def step(x, w, b, act, g):
    """Output and gradients, b's left out with b."""
    from ictc_o2_hp_b200 import dense
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = dense.gated_linear(*leaves, activation=act)
    return y.detach(), torch.autograd.grad(y, leaves, g)


SHAPES = [
    (1, 1, 1), (1, 64, 64), (3, 7, 5), (4, 129, 1), (5, 8, 64), (37, 8, 64), (37, 64, 64),
    (127, 63, 65), (128, 64, 128), (129, 65, 127), (200, 257, 3), (255, 16, 130), (300, 1000, 72),
    (64, 2049, 33), (1000, 33, 200), (2500, 64, 64), (2500, 64, 32), (5000, 7, 3), (3000, 64, 1),
    (129, 1, 64), (513, 61, 59), (6, 16, 16), (16, 512, 96), (31, 520, 264), (700, 1025, 769),
    (2053, 211, 333), (4097, 702, 6), (5000, 1536, 8), (4500, 3, 130), (4099, 8, 520), (2, 4096, 40),
    (4, 8192, 513), (1, 1000, 2048), (700, 1024, 768), (4096, 256, 256), (16, 4096, 520),
    (20000, 64, 64), (33, 8200, 24), (40000, 24, 8), (260, 96, 4100), (9001, 64, 48), (64, 24, 3000),
    (777, 8, 8), (130, 16, 24), (5000, 56, 40), (1, 40, 24), (300, 48, 16), (641, 4, 12),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_float64(shape, dtype, cuda_device):
    from ictc_o2_hp_b200 import _lib, dense
    m, k, n = shape
    act = ACTS[(m + k + n) % len(ACTS)]
    x, w, b, g = operands(m, k, n, dtype, cuda_device, bias=(m + n) % 3 > 0)
    y, grads = step(x, w, b, act, g)
    check_gated(x, w, b, act, g, y, (*grads, None), dtype)
    plain = dense.gated_linear(x, w, b, act)
    check_gated(x, w, b, act, g, plain, None, dtype)
    y2, again = step(x, w, b, act, g)
    assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(grads, again)), \
        "not the same bits twice"
    assert torch.equal(dense.gated_linear(x, w, b, act), plain)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", [(150, 40, 72), (3, 40, 72), (1300, 48, 24), (20, 512, 200)])
def test_activations(shape, act, dtype, cuda_device):
    """Every activation on p over a wide range."""
    x, w, b, g = operands(*shape, dtype, cuda_device, 10)
    w = w * 2.0
    y, grads = step(x, w, b, act, g)
    check_gated(x, w, b, act, g, y, grads, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(40, 24), (64, 64), (264, 40)])
def test_strides_and_batches(k, n, dtype, cuda_device):
    """Column slices (rows off every vector boundary), repeated rows, transposed weights,
    expanded gradients and leading batch dimensions."""
    from ictc_o2_hp_b200 import dense
    big = rand((70, 3, 2 * k + 9), dtype, cuda_device, 31)
    wide = rand((2 * n + 9, 2 * k + 9), dtype, cuda_device, 32, 0.2)
    gw = rand((70, 3, n + 9), dtype, cuda_device, 33)
    b = rand((2 * n,), dtype, cuda_device, 35)
    for x in (big[..., 1:k + 1], big[:, :, :k], big[:, 1, 3:k + 3], big[..., ::2][..., :k],
              big[:1, :1, 8:k + 8].expand(70, 3, k), big[0, 0, :k]):
        for w in (wide[:2 * n, 8:k + 8], wide[3:2 * n + 3, 5:k + 5],
                  wide[:2 * n, :k].t().contiguous().t()):
            lead = x.shape[:-1]
            full = gw[..., :n] if x.dim() == 3 else gw[:, 1, 5:n + 5] if x.dim() == 2 else gw[0, 0, 1:n + 1]
            for g in (full, rand((1,), dtype, cuda_device, 34).expand(*lead, n)):
                xx, ww = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
                y = dense.gated_linear(xx, ww, b, "gelu")
                assert y.shape == (*lead, n) and y.is_contiguous()
                grads = torch.autograd.grad(y, (xx, ww), g)
                check_gated(x.reshape(-1, k), w, b, "gelu", g.reshape(-1, n),
                            y.detach().reshape(-1, n),
                            (grads[0].reshape(-1, k), grads[1], None), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(700001, 64, 64), (300007, 61, 59), (400003, 24, 40),
                                   (900001, 8, 8), (500001, 64, 24), (500001, 40, 64),
                                   (60001, 72, 136)])
def test_many_tiles(shape, dtype, cuda_device):
    """Many tiles per CTA, run after run: a buffer that is written again while it is still
    read shows as another tile's rows, in a few rows of a million."""
    from ictc_o2_hp_b200 import dense
    x, w, b, g = operands(*shape, dtype, cuda_device, 70)
    first = None
    for _ in range(6):
        y, grads = step(x, w, b, "silu", g)
        out = (y, *grads, dense.gated_linear(x, w, b, "silu"))
        if first is None:
            first = out
            check_gated(x, w, b, "silu", g, y, grads, dtype)
            check_gated(x, w, b, "silu", g, out[-1], None, dtype)
        assert all(torch.equal(p, q) for p, q in zip(out, first))


@pytest.mark.parametrize("scale", [1e-18, 1e-13, 1e15, 1e17])
@pytest.mark.parametrize("shape", [(300, 64, 64), (300, 72, 40), (300, 33, 77)])
def test_relu_slopes_of_small_and_large_operands(shape, scale, cuda_device):
    """Operands whose squares leave float32's range while their products do not."""
    from ictc_o2_hp_b200 import dense
    m, k, n = shape
    x, w, _, g = operands(m, k, n, torch.float32, cuda_device, 143, bias=False)
    x, w = x * scale, w * scale
    at = torch.arange(n, device=cuda_device)
    p = in_order(x, w[:n])
    b = torch.zeros(2 * n, device=cuda_device)
    b[:n] = -torch.nextafter(p[at * 37 % m, at], torch.full((n,), math.inf, device=cuda_device))
    p = p + b[:n]
    native, code = dense._load(), dense.ACTIVATIONS["relu"]
    _, kept = native.gated_forward(x, w, b, code, True)
    assert torch.equal(kept[:, :n] > 0, p > 0)
    y, (dx, dw, db) = step(x, w, b, "relu", torch.ones_like(g))
    pu = (x.double() @ w.double()[n:].t())
    want = (pu * (p > 0)).sum(0)
    size = (pu.abs() * (p > 0)).sum(0) + sum_error(k) * (x.double().abs() @ w.double()[n:].abs().t()).sum(0)
    within("dbias", db[:n], want, sum_error(k) * (x.double().abs() @ w.double()[n:].abs().t()).sum(0) +
           (m + 64) * U * size)


@pytest.mark.parametrize("shape", [(300, 64, 64), (5, 8, 4), (300, 72, 40), (300, 33, 77), (40, 2048, 24)])
def test_relu_of_zero_and_infinite_rows(shape, cuda_device):
    """Rows and columns of zeros have a p of exactly 0 and relu's slope there, which is 0;
    infinities have the slope of their sign, and NaN has none."""
    m, k, n = shape
    x, w, _, g = operands(m, k, n, torch.float32, cuda_device, 142, bias=False)
    x[1] = 0
    x[m - 1] = 0
    w[2] = 0
    base = step(x, w, None, "relu", g)
    for t in (base[1][0], base[1][1]):
        assert t.isfinite().all()
    assert not base[1][0][1].any() and not base[1][0][m - 1].any() and not base[1][1][2].any()
    pg, pu, a, s, y64, d, dx, dw, _ = gated64(x, w, None, "relu", g)
    check_gated(x, w, None, "relu", g, base[0], (*base[1], None), torch.float32)
    x[3, 5] = math.inf
    w[:, 5] = w[:, 5].abs() + 0.1
    w[1, 5] = -1.0
    w[n + 1, 5] = 1.0
    y, (dx, dw) = step(x, w, None, "relu", g)
    want = torch.full((n,), math.inf, device=cuda_device)
    want[1] = math.nan  # relu(-inf) inf
    assert torch.equal(y[3].isnan(), want.isnan()) and torch.equal(y[3].isinf(), want.isinf())
    keep = torch.arange(m, device=cuda_device) != 3
    assert dx[keep].isfinite().all() and not dx[3].isfinite().any()


def whole_operands(m, k, n, dtype, device, seed):
    """Operands of -1, 0 and 1: with an activation of slope 0 or 1 every product and sum is a
    whole number below 2^24, exact in float32 in any order, and D is exact in every type."""
    gen = torch.Generator(device=device).manual_seed(seed)

    def draw(*shape):
        return torch.randint(-1, 2, shape, generator=gen, device=device).to(dtype)

    return draw(m, k), draw(2 * n, k), draw(2 * n), draw(m, n)


def exact_step(x, w, b, act, g):
    """y, dx, dW and db in float64, in blocks of rows; and the largest partial sum there is."""
    n = w.shape[0] // 2
    wide, outs, dxs = w.double(), [], []
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    db = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device)
    most = 0.0
    for rows, grad in zip(x.split(50000), g.split(50000)):
        rows, grad = rows.double(), grad.double()
        pg, pu = (rows @ wide.t() + b.double()).split(n, 1)
        a, slope = (pg.clamp(min=0), (pg > 0).double()) if act == "relu" else (pg, torch.ones_like(pg))
        d = torch.cat([grad * pu * slope, grad * a], 1)
        outs.append(a * pu)
        dxs.append(d @ wide)
        dw += d.t() @ rows
        db += d.sum(0)
        most = max(most, dw.abs().max().item(), db.abs().max().item(), d.abs().max().item())
    return torch.cat(outs), torch.cat(dxs), dw, db, most


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("shape", [(700001, 64, 64), (300007, 61, 59), (400003, 24, 40),
                                   (900001, 8, 8), (500001, 64, 24), (300001, 40, 64),
                                   (200001, 72, 136), (38000, 200, 72)])
def test_every_row_counts_once(shape, act, dtype, cuda_device):
    """Whole numbers, whose sums over many tiles are exact: a tile that is left out, taken twice
    or read too early shows whatever the bounds of rounding.  Each set of gradients that a
    caller can ask for, in rows of W of their own distance too."""
    m, k, n = shape
    x, w, b, g = whole_operands(m, k, n, dtype, cuda_device, 150)
    y, *grads, most = exact_step(x, w, b, act, g)
    assert most < 2 ** 22  # far from where float32 stops holding whole numbers, on the way too
    want = [t.to(dtype) for t in grads]
    from ictc_o2_hp_b200 import dense
    apart = torch.cat([w, w.new_zeros(2 * n, 16)], 1)[:, :k]
    for needs in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (1, 0, 1)):
        for weight in (w, apart) if all(needs) else (w,):
            leaves = [t.detach().requires_grad_(bool(q)) for t, q in zip((x, weight, b), needs)]
            out = dense.gated_linear(*leaves, activation=act)
            assert torch.equal(out, y.to(dtype))
            asked = [t for t in leaves if t.requires_grad]
            got = torch.autograd.grad(out, asked, g)
            assert all(map(torch.equal, got, [t for t, q in zip(want, needs) if q])), needs


def test_weight_gradients_past_32_bits(cuda_device):
    """D of more than 2^31 elements: every row's part of dW and db, exactly."""
    x, w, b, _ = whole_operands(140001, 16, 8192, torch.bfloat16, cuda_device, 151)
    g = x.new_ones(1).expand(140001, 8192)
    y, (dx, dw, db) = step(x, w, b, "none", g)
    y64, dx64, dw64, db64, most = exact_step(x, w, b, "none", g)
    assert most < 2 ** 22
    for got, want in ((y, y64), (dx, dx64), (dw, dw64), (db, db64)):
        assert torch.equal(got, want.to(got.dtype))


def test_offsets_past_32_bits(cuda_device):
    """p and D of more than 2^31 elements, y of more than 2^30: rows on both sides of such
    offsets, the last ones, and the bias gradient over all."""
    from ictc_o2_hp_b200 import dense
    m, k, n = 140001, 16, 8192
    x, w, b, _ = operands(1, k, n, torch.bfloat16, cuda_device, 75)
    x = rand((m, k), torch.bfloat16, cuda_device, 76)
    g = rand((1,), torch.bfloat16, cuda_device, 77).expand(m, n)
    y, (dx, dw, db) = step(x, w, b, "silu", g)
    for at in (0, 2 ** 31 // n - 150, 2 ** 31 // (2 * n) - 150, 2 ** 30 // n - 150, m - 300):
        q = slice(at, at + 300)
        check_gated(x[q], w, b, "silu", g[q], y[q], (dx[q], None, None), torch.bfloat16)
    total = torch.zeros(2 * n, dtype=torch.float64, device=cuda_device)
    size = torch.zeros_like(total)
    for rows in x.split(10000):
        d = gated64(rows, w, b, "silu", g[:len(rows)])[5]
        total += d.sum(0)
        size += d.abs().sum(0)
    within("dbias", db, total, 1.01 * (m + 200) * U * size + 2 * UNIT[torch.bfloat16] * total.abs())
    assert dw.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(5, 9), (30, 64), (30, 5), (300, 70), (2000, 48)])
def test_partial_gradients(shape, dtype, cuda_device):
    """Each gradient alone is the one of all together."""
    from ictc_o2_hp_b200 import dense
    m, k = shape
    x, w, b, g = operands(m, k, 24, dtype, cuda_device, 60)
    full = step(x, w, b, "gelu", g)[1]
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        y = dense.gated_linear(*leaves, "gelu")
        assert torch.equal(torch.autograd.grad(y, leaves[i], g)[0], full[i])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 40, 24), (700, 64, 64), (700, 24, 56), (1000, 63, 61),
                                   (300, 264, 200)])
def test_recomputed_p(shape, dtype, cuda_device):
    """A backward that is given no p computes it again, whichever kernels the layer takes; a
    gradient off the boundaries is copied first."""
    from ictc_o2_hp_b200 import dense
    x, w, b, g = operands(*shape, dtype, cuda_device, 65)
    native, code = dense._load(), dense.ACTIVATIONS["silu"]
    y, p = native.gated_forward(x, w, b, code, True)
    assert p.shape == (shape[0], 2 * shape[2]) and p.dtype == torch.float32
    none = torch.empty(0, device=cuda_device)
    odd = rand((shape[0] * shape[2] + 1,), dtype, cuda_device, 66)[1:].view(*g.shape)
    for grad in (g, odd, g[:1].expand_as(g)):
        for kept in (p, none):
            grads = native.gated_backward(x, w, b, kept, grad, code)
            check_gated(x, w, b, "silu", grad, y, grads, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(300, 64, 64), (700, 24, 40), (129, 16, 8)])
def test_infinite_bias(shape, dtype, cuda_device):
    """Rows past the last of a tile have a bias too: it must not reach the sums."""
    m, k, n = shape
    x, w, b, g = operands(m, k, n, dtype, cuda_device, 67)
    base = step(x, w, b, "none", g)
    b[n + 2] = math.inf
    y, (dx, dw, db) = step(x, w, b, "none", g)
    keep = torch.arange(2 * n, device=cuda_device) != 2
    assert torch.equal(y[:, keep[:n]], base[0][:, keep[:n]]) and not y[:, 2].isfinite().any()
    assert torch.equal(dw[keep], base[1][1][keep]) and torch.equal(db[keep], base[1][2][keep])
    assert not dw[2].isfinite().any() and not dx.isfinite().any()


def in_order(x, w):
    """x w^T by float32 fused multiply-adds in the order of k.  Products are exact in float64;
    a sum there is rounded to odd, so that rounding it again to float32 rounds once."""
    acc = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    for i in range(x.shape[1]):
        p = x[:, i:i + 1].double() * w[:, i].double()
        s = p + acc
        back = s - p
        lost = (p - (s - back)) + (acc - back)
        bits = s.view(torch.int64)
        away = torch.where((lost > 0) == (s > 0), 1, -1)
        bits = torch.where((lost != 0) & (bits % 2 == 0), bits + away, bits)
        acc = bits.view(torch.float64).float().double()
    return acc.float()


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("shape", [
    (1, 64, 64), (5, 8, 4), (37, 64, 64), (3, 700, 9), (3000, 64, 64), (20001, 40, 64), (9001, 64, 12),
    (2000, 16, 48), (300, 33, 77), (5000, 63, 61), (2000, 8, 3), (300, 264, 200), (2053, 211, 333),
    (4097, 702, 6), (5000, 1536, 8), (4500, 3, 130), (260, 96, 1100), (64, 2049, 33), (20, 8200, 24)])
def test_relu_slopes_are_those_of_the_sum_in_order(shape, bias, cuda_device):
    """The slope of a projection within its rounding of 0 does not depend on the kernel: it is
    that of float32 multiply-adds in the order of k, the bias last.  One row of every column is
    given a bias that leaves one ulp of it, 0 or minus one ulp; the gradients' bounds then have
    no room for a slope of the other side."""
    from ictc_o2_hp_b200 import dense
    m, k, n = shape
    x, w, b, g = operands(m, k, n, torch.float32, cuda_device, 140)
    p = in_order(x, w[:n])
    if bias:
        cols = torch.arange(n, device=cuda_device)
        at = p[cols * 37 % m, cols]
        step_to = torch.tensor([math.inf, 0.0, -math.inf], device=cuda_device)[cols % 3]
        b[:n] = -torch.where(cols % 3 == 1, at, torch.nextafter(at, step_to))
        p = p + b[:n]
        assert (p == 0).any() or n < 2
    else:
        b = None
    slope = (p > 0).double()
    native, code = dense._load(), dense.ACTIVATIONS["relu"]
    y, kept = native.gated_forward(x, w, b, code, True)
    assert torch.equal(kept[:, :n] > 0, p > 0)
    none = torch.empty(0, device=cuda_device)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = dense.gated_linear(*leaves, activation="relu")
    ways = [torch.autograd.grad(y, leaves, g, retain_graph=True),
            [t.detach() for t in torch.autograd.grad(y, leaves, g, create_graph=True)],
            native.gated_backward(x, w, b, kept, g, code),
            native.gated_backward(x, w, b, none, g, code)]

    pg, pu, a, _, _, _, _, _, _ = gated64(x, w, b, "relu", g)
    a = a * slope
    ax, aw, ag = x.double().abs(), w.double().abs(), g.double().abs()
    ep = sum_error(k) * (ax @ aw.t() + (0 if b is None else b.double().abs()))
    epg, epu = ep.chunk(2, -1)
    d = torch.cat([g * pu * slope, g * a], -1)
    ed = torch.cat([ag * slope * epu, ag * epg], -1) + 4 * U * d.abs()
    ad = d.abs() + ed
    for grads in ways:
        for name, got, left, right, count in (
                ("dx", grads[0], d, w.double(), 2 * n), ("dweight", grads[1], d.t(), x.double(), m),
                ("dbias", grads[2] if b is not None else None, d.t(), torch.ones(m, 1, device=cuda_device).double(), m)):
            if got is None:
                continue
            wide = left @ right
            e, size = (ed, ad) if name == "dx" else (ed.t(), ad.t())
            bound = e @ right.abs() + max(sum_error(count), (count + 64) * U * (name == "dbias")) * (
                size @ right.abs()) + 3 * U * (wide.abs() + e @ right.abs())
            within(name, got.reshape(wide.shape), wide, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["x strided", "x odd", "both"])
@pytest.mark.parametrize("shape", [(40000, 64, 32), (2000000, 64, 32), (50000, 96, 40)])
def test_one_operand_off_the_boundaries(shape, which, dtype, cuda_device):
    """Sizes whose operands are copied to aligned rows, with an x that is aligned but not
    contiguous beside a W off the boundaries, the other way round, and both off."""
    m, k, n = shape
    x, w, b, g = operands(m, k, n, dtype, cuda_device, 145)
    if which == "x strided":
        x = torch.cat([x, x], 1)[:, :k]
    else:
        x = torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].view(m, k)
    if which != "x odd":
        w = torch.cat([w.reshape(-1)[:1], w.reshape(-1)])[1:].view(2 * n, k)
    y, grads = step(x, w, b, "silu", g)
    check_gated(x, w, b, "silu", g, y, grads, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty(dtype, cuda_device):
    from ictc_o2_hp_b200 import dense
    w = rand((12, 5), dtype, cuda_device, 61).requires_grad_(True)
    b = rand((12,), dtype, cuda_device, 62).requires_grad_(True)
    x = torch.empty(0, 3, 5, dtype=dtype, device=cuda_device, requires_grad=True)
    y = dense.gated_linear(x, w, b)
    assert y.shape == (0, 3, 6)
    for graph in (False, True):
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y), retain_graph=True,
                                         create_graph=graph)
        assert gx.shape == x.shape and gw.shape == w.shape and gb.shape == b.shape
        assert not gw.any() and not gb.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 72, 140), (150, 72, 140), (12, 520, 64), (200, 48, 40)])
def test_nonfinite(shape, dtype, cuda_device):
    """An infinity or NaN reaches exactly the outputs that the formula gives it, with its
    sign (act none: products of infinities alone); the others keep their values."""
    from ictc_o2_hp_b200 import dense
    m, k, n = shape
    x, w, _, _ = operands(m, k, n, dtype, cuda_device, 50, bias=False)
    w[:, 7] = 1.0
    w[5, 7] = -2.0
    w[n + 9, 7] = -1.0
    base = dense.gated_linear(x, w, None, "none")
    x[1, 7] = math.inf
    x[2, 3] = math.nan
    w[20, 30] = -math.inf
    y = dense.gated_linear(x, w, None, "none")
    pg, pu = (x.double() @ w.double().t()).chunk(2, -1)
    want = pg * pu
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf())
    assert torch.equal(y[y.isinf()].double(), want[want.isinf()])
    keep = want.isfinite()
    assert keep.any() and torch.equal(y[keep], base[keep])


@pytest.mark.parametrize("shape", [(3, 40, 48), (700, 48, 40), (700, 48, 140)])
def test_nonfinite_gradients(shape, cuda_device):
    """Infinities and NaN in the gradient and in x reach the sums they belong to, and no
    others."""
    m, k, n = shape
    x, w, _, g = operands(m, k, n, torch.float32, cuda_device, 55, bias=False)
    base = step(x, w, None, "none", g)[1]
    g = g.clone()
    g[m - 1, 7] = math.nan
    dx, dw = step(x, w, None, "none", g)[1]
    rows = torch.arange(m, device=cuda_device) != m - 1
    cols = torch.arange(2 * n, device=cuda_device) % n != 7
    assert dx[m - 1].isnan().all() and torch.equal(dx[rows], base[0][rows])
    assert dw[~cols].isnan().all() and torch.equal(dw[cols], base[1][cols])


def test_gradients_against_differences(cuda_device):
    """Directional derivatives against central differences of the float64 formula."""
    m, k, n, h = 40, 24, 32, 1e-5
    x, w, b, g = operands(m, k, n, torch.float32, cuda_device, 80)

    def total(x, w, b, act):
        pg, pu = (x @ w.t() + b).chunk(2, -1)
        return (act64(pg, act) * pu * g.double()).sum()

    for act in ("none", "silu", "gelu", "gelu_tanh"):
        grads = step(x, w, b, act, g)[1]
        point = [t.double() for t in (x, w, b)]
        for i, grad in enumerate(grads):
            v = rand(grad.shape, torch.float32, cuda_device, 20 + i).double()
            ends = [total(*(t + sign * h * v if j == i else t for j, t in enumerate(point)), act)
                    for sign in (1, -1)]
            slope = (ends[0] - ends[1]).item() / (2 * h)
            size = (grad.double().abs() * v.abs()).sum().item()
            assert abs((grad.double() * v).sum().item() - slope) <= 1e-5 * size


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_second_derivatives(act, dtype, cuda_device):
    """A force-like loss: squared input gradients, differentiated by every operand.  In
    16-bit types some eight tensors between the operands and a second derivative are rounded,
    and the squares double what is off: 24 u in the 2-norm."""
    from ictc_o2_hp_b200 import dense
    x, w, b, g = operands(50, 24, 40, dtype, cuda_device, 90)

    def loss(x, w, b, g, layer):
        f = torch.autograd.grad((layer(x, w, b) * g).sum(), x, create_graph=True)[0]
        return (f.double() ** 2).sum() if f.dtype == torch.float64 else (f.float() ** 2).sum()

    def plain(x, w, b):
        pg, pu = (x @ w.t() + b).chunk(2, -1)
        return act64(pg, act) * pu

    ours = [t.clone().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(loss(*ours, g, lambda *t: dense.gated_linear(*t, act)), ours)
    wide = [t.double().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(loss(*wide, g.double(), plain), wide)
    limit = 1e-5 if dtype == torch.float32 else 24 * UNIT[dtype]
    for p, q in zip(got, want):
        assert (p.double() - q).norm() <= limit * q.norm()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_create_graph_keeps_first_gradients(act, dtype, cuda_device):
    """The gradients that are differentiated again keep the error bounds of those that are
    not."""
    from ictc_o2_hp_b200 import dense
    x, w, b, g = operands(150, 40, 72, dtype, cuda_device, 16)
    x = x * 2.0
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = dense.gated_linear(*leaves, act)
    grads = torch.autograd.grad(y, leaves, g, create_graph=True)
    assert all(t.requires_grad for t in grads)
    check_gated(x, w, b, act, g, y.detach(), [t.detach() for t in grads], dtype)


# ----------------------------------------------------------- modules, streams, compile


def test_modules(cuda_device):
    from ictc_o2_hp_b200 import GatedBlock, GatedLinear, RadialTrunk
    torch.manual_seed(3)
    ours = GatedLinear(20, 30).to(cuda_device)
    torch.manual_seed(3)
    theirs = torch.nn.Linear(20, 60).to(cuda_device)
    theirs.load_state_dict(ours.state_dict())
    assert torch.equal(ours.weight, theirs.weight)
    x = rand((9, 20), torch.float32, cuda_device, 1)
    f = torch.nn.functional

    def gated(layer, x):
        pg, pu = f.linear(x, layer.weight.double(), layer.bias.double()).chunk(2, -1)
        return f.silu(pg) * pu

    want = gated(ours, x.double())
    assert (ours(x).double() - want).norm() <= 1e-6 * want.norm()
    block = GatedBlock(20, 48).to(cuda_device)
    h = gated(block.gated, f.layer_norm(x.double(), (20,)))
    want = x.double() + f.linear(h, block.down.weight.double(), block.down.bias.double())
    assert (block(x).double() - want).norm() <= 1e-6 * want.norm()
    trunk = RadialTrunk(8, 64, blocks=2, gated=True).to(cuda_device)
    assert all(isinstance(b, GatedBlock) for b in trunk.blocks)
    out = trunk(rand((5, 11, 8), torch.float32, cuda_device, 2))
    assert out.shape == (5, 11, 64) and out.mean(-1).abs().max() <= 1e-5


def test_gated_trunk_feeds_the_radial_product(cuda_device):
    """Gated trunk, final affine layer and per-edge product together, against the same
    network of torch modules in front of the product."""
    from ictc_o2_hp_b200 import Linear, RadialTrunk, RadialUvuTensorProduct, UvuTensorProduct
    torch.manual_seed(0)
    tp = UvuTensorProduct(16, 1, 2, parity="full", parity_in2="canonical", shared_weights=False)
    product = RadialUvuTensorProduct(tp, Linear(32, tp.weight_numel)).to(cuda_device)
    trunk = RadialTrunk(8, 32, gated=True).to(cuda_device)
    basis = rand((300, 8), torch.float32, cuda_device, 1)
    x = rand((300, tp.input1_dimension), torch.float32, cuda_device, 2)
    y = rand((300, tp.input2_dimension), torch.float32, cuda_device, 3)
    out = product(x, y, trunk(basis))
    f = torch.nn.functional

    def torch_trunk(b):
        h = f.silu(f.linear(b, trunk.embed.weight, trunk.embed.bias))
        for q in trunk.blocks:
            z = f.layer_norm(h, (32,), q.norm.weight, q.norm.bias)
            pg, pu = f.linear(z, q.gated.weight, q.gated.bias).chunk(2, -1)
            h = h + f.linear(f.silu(pg) * pu, q.down.weight, q.down.bias)
        return f.layer_norm(h, (32,), trunk.norm.weight, trunk.norm.bias)

    want = product(x, y, torch_trunk(basis))
    assert (out - want).norm() <= 1e-5 * want.norm()
    params = list(trunk.parameters())
    g = rand(out.shape, torch.float32, cuda_device, 4)
    for p, q in zip(torch.autograd.grad(out, params, g), torch.autograd.grad(want, params, g)):
        assert (p - q).norm() <= 1e-4 * q.norm()


def test_example_runs(cuda_device):
    import subprocess
    import sys
    from pathlib import Path
    example = Path(__file__).resolve().parents[1] / "examples" / "radial_trunk.py"
    run = subprocess.run([sys.executable, str(example), "--edges", "700", "--hidden", "32",
                          "--steps", "3", "--gated", "--clip", "0.5"], capture_output=True,
                         text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    assert "700 edges" in run.stdout


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3000, 64, 64), (700, 512, 256), (700, 511, 255), (300, 72, 40)])
def test_first_call_of_a_thread(shape, dtype, cuda_device):
    """A thread that has no context yet, because its memory comes from the allocator's cache."""
    import threading

    from ictc_o2_hp_b200 import dense
    x, w, b, g = operands(*shape, dtype, cuda_device, 125)
    native, code = dense._load(), dense.ACTIVATIONS["silu"]
    _, p = native.gated_forward(x, w, b, code, True)
    none = torch.empty(0, device=cuda_device)
    for call in (lambda: (dense.gated_linear(x, w, b),), lambda: native.gated_forward(x, w, b, code, True),
                 lambda: native.gated_backward(x, w, b, p, g, code),
                 lambda: native.gated_backward(x, w, b, none, g, code),
                 lambda: (dense.linear(x, w, b),)):
        want = [t.clone() for t in call()]
        held = call()
        torch.cuda.synchronize()
        del held
        got, failed = [], []

        def run():
            try:
                got.extend(call())
            except Exception as e:  # noqa: BLE001
                failed.append(e)

        thread = threading.Thread(target=run)
        thread.start()
        thread.join()
        assert not failed, failed
        assert all(map(torch.equal, got, want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 96, 64), (20, 512, 64), (200, 96, 64), (2000, 64, 64)])
def test_other_stream_and_graph_capture(shape, dtype, cuda_device):
    """Work goes to the caller's stream; a captured step replays on new inputs, two captured
    steps do not touch each other's buffers."""
    from ictc_o2_hp_b200 import dense
    x, w, b, g = operands(*shape, dtype, cuda_device, 120)
    want = step(x, w, b, "gelu", g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, w, b, "gelu", g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and all(map(torch.equal, got[1], want[1]))
    leaves = [torch.zeros_like(t).requires_grad_(True) for t in (x, w, b)]
    held = torch.zeros_like(g)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = dense.gated_linear(*leaves, "gelu")
            outs.append((y, *torch.autograd.grad(y, leaves, held)))
        graphs.append(graph)
    with torch.no_grad():
        for t, source in zip((*leaves, held), (x, w, b, g)):
            t.copy_(source)
    graphs[0].replay()
    graphs[1].replay()
    for out in outs:
        assert torch.equal(out[0], want[0]) and all(map(torch.equal, out[1:], want[1]))


@pytest.mark.parametrize("shape", [(5, 8, 4), (2000, 64, 64), (700, 200, 72), (300, 33, 77)])
def test_relu_captured_and_traced(shape, cuda_device):
    """The passes that decide relu's slopes in a captured step, beside another captured one, and
    through the dispatcher."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from ictc_o2_hp_b200 import dense
    x, w, b, g = operands(*shape, torch.float32, cuda_device, 127)
    want = step(x, w, b, "relu", g)
    leaves = [torch.zeros_like(t).requires_grad_(True) for t in (x, w, b)]
    held = torch.zeros_like(g)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = dense.gated_linear(*leaves, activation="relu")
            outs.append((y, *torch.autograd.grad(y, leaves, held)))
        graphs.append(graph)
    with torch.no_grad():
        for t, source in zip((*leaves, held), (x, w, b, g)):
            t.copy_(source)
    for graph in graphs:
        graph.replay()
    for out in outs:
        assert torch.equal(out[0], want[0]) and all(map(torch.equal, out[1:], want[1]))

    def whole(x, w, b):
        y = dense.gated_linear(x, w, b, "relu")
        return (y, *torch.autograd.grad(y, (x, w, b), g))

    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    got = make_fx(whole)(*leaves)(*leaves)
    # the recorded step may keep p where the other computes it again: other kernels, same slopes
    check_gated(x, w, b, "relu", g, got[0].detach(), got[1:], torch.float32)


def test_compile_and_traces(cuda_device):
    from torch.fx.experimental.proxy_tensor import make_fx

    from ictc_o2_hp_b200 import GatedBlock
    torch.manual_seed(1)
    block = GatedBlock(32).to(cuda_device)
    x, other = (rand((64, 32), torch.float32, cuda_device, s).requires_grad_(True) for s in (1, 3))
    g = rand((64, 32), torch.float32, cuda_device, 2)
    params = list(block.parameters())
    want = torch.autograd.grad(block(x), (x, *params), g)
    run = torch.compile(block, fullgraph=True, backend="aot_eager")
    assert all(map(torch.equal, torch.autograd.grad(run(x), (x, *params), g), want))

    def whole(x):
        y = block(x)
        return y, torch.autograd.grad(y, x, g)[0]

    recorded = make_fx(whole)(other.detach().clone().requires_grad_(True))
    got = recorded(x.detach().clone().requires_grad_(True))
    assert torch.equal(got[0], block(x)) and torch.equal(got[1], want[0])


def test_autocast(cuda_device):
    from ictc_o2_hp_b200 import GatedLinear, dense
    layer = GatedLinear(24, 40).to(cuda_device)
    x = rand((30, 24), torch.float16, cuda_device, 1).requires_grad_(True)
    g = rand((30, 40), torch.bfloat16, cuda_device, 3)
    with pytest.raises(ValueError):
        layer(x)
    args = [t.detach().bfloat16().requires_grad_(True) for t in (x, layer.weight, layer.bias)]
    want = dense.gated_linear(*args)
    grads = torch.autograd.grad(want, args, g)
    for run in (layer, torch.compile(layer, fullgraph=True, backend="aot_eager")):
        with torch.autocast("cuda", torch.bfloat16):
            y = run(x)
        got = torch.autograd.grad(y, (x, layer.weight, layer.bias), g)
        assert torch.equal(y, want)
        assert all(torch.equal(p, q.to(p.dtype)) for p, q in zip(got, grads))


def test_views_with_a_negative_bit(cuda_device):
    from ictc_o2_hp_b200 import dense
    z = torch.complex(*(rand((40, 1), torch.float32, cuda_device, s) for s in (36, 37)))
    x = z.conj().imag
    assert x.is_neg()
    w = rand((6, 1), torch.float32, cuda_device, 38)
    assert torch.equal(dense.gated_linear(x, w), dense.gated_linear(x.resolve_neg(), w))


def test_changed_operands_are_noticed(cuda_device):
    """A backward that would compute p again from other values refuses."""
    from ictc_o2_hp_b200 import dense
    x, w, b, g = operands(300, 64, 64, torch.float32, cuda_device, 130)
    for i in range(3):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = dense.gated_linear(*leaves)
        with torch.no_grad():
            leaves[i].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, g)


def test_refusals(cuda_device):
    from torch.autograd import forward_ad

    from ictc_o2_hp_b200 import dense
    x = torch.randn(4, 6, device=cuda_device)
    w = torch.randn(10, 6, device=cuda_device)
    with pytest.raises(TypeError):
        dense.gated_linear(x.double(), w.double())
    for call in (
        lambda: dense.gated_linear(x, w.half()),
        lambda: dense.gated_linear(x, w[:, :5]),
        lambda: dense.gated_linear(x, w[:9]),
        lambda: dense.gated_linear(x, w[:0]),
        lambda: dense.gated_linear(x, w[0]),
        lambda: dense.gated_linear(x, w, w[:5, 0]),
        lambda: dense.gated_linear(x, w, w[:, 0].cpu()),
        lambda: dense.gated_linear(x, w, activation="swish"),
        lambda: dense.gated_linear(x[:, :0], w[:, :0]),
    ):
        with pytest.raises(ValueError):
            call()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.clone(), torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            dense.gated_linear(dual, w)
