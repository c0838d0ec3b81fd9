"""The gradients' norm and clipping on the GPU against float64.

Bounds, with U the unit roundoff of float32 and u that of the operand type: squares are
added in float32 over at most eight values, all positive (8 U), in float64 beyond, so a norm
is off by 4 U and its own rounding: 5 U.  The factor divides by it plus a rounded sum: 8 U;
a scaled value is one float32 product more, rounded to its type: 9 U + u.
"""

from __future__ import annotations

import math

import pytest
import torch

from test_dense_gpu import DTYPES, TINY, U, UNIT, rand, within

pytestmark = pytest.mark.gpu


def norm64(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


def check_norm(got, want):
    assert got.shape == () and got.dtype == torch.float32 and got.is_cuda
    assert abs(got.item() - want) <= 5 * U * want, f"{got.item()} and {want}"


def check_clipped(got, grads, max_norm, want=None):
    want = norm64(grads) if want is None else want
    factor = min(1.0, max_norm / (want + 1e-6))
    assert len(got) == len(grads)
    for o, g in zip(got, grads):
        assert o.dtype == g.dtype and o.device == g.device and not o.requires_grad
        exact = g.double() * factor
        within("clipped", o, exact, (9 * U + (g.dtype != torch.float32) * UNIT[g.dtype]) * 1.01 *
               exact.abs() + TINY[g.dtype])


def lists(device):
    """Lists of every kind of size: single values, odd lengths, off the 16-byte boundaries,
    more than a launch holds, empties, tensors of several chunks."""
    flat = {t: rand((400_000,), t, device, 3, 0.1) for t in DTYPES}

    def parts(sizes, kinds, start=0):
        out, at = [], start
        for i, n in enumerate(sizes):
            out.append(flat[kinds[i % len(kinds)]][at:at + n])
            at += n
        return out

    yield "one value", [rand((1,), torch.float32, device, 1)]
    yield "scalars", [rand((), t, device, 2) for t in DTYPES]
    for t in DTYPES:
        yield f"odd {t}", parts([1, 2, 3, 5, 7, 8, 9, 15, 17, 31, 33, 255, 257, 8191, 8193, 16385,
                                 40001], [t])
    yield "mixed", parts([63, 64, 65, 1000, 2049, 30011], DTYPES, 1)
    yield "empties", parts([0, 5, 0, 0, 70001, 0], DTYPES)
    yield "many", parts([1 + i % 97 for i in range(2500)], DTYPES)
    yield "65 tensors", parts([3000 + i for i in range(65)], [torch.float32])
    yield "1024 tensors", parts([100 + i % 7 for i in range(1024)], [torch.bfloat16])
    yield "1025 tensors", parts([100 + i % 7 for i in range(1025)], [torch.float16])
    yield "large", [rand((5_000_011,), torch.float32, device, 5, 1e-3),
                    rand((3001, 1777), torch.bfloat16, device, 6), rand((77,), torch.float16, device, 7)]


def test_norm_and_clipping_against_float64(cuda_device):
    from ictc_o2_hp_b200 import gradients
    for name, grads in lists(cuda_device):
        want = norm64(grads)
        norm = gradients.grad_norm(grads)
        check_norm(norm, want)
        most = max((float(t.double().abs().max()) for t in grads if t.numel()), default=0.0)
        assert gradients.grad_norm(grads, math.inf).item() == most, name
        for factor in (0.3, 1.5):
            before = [t.clone() for t in grads]
            clipped, got = gradients.clip_grads(grads, factor * want)
            assert torch.equal(got, norm), name
            check_clipped(clipped, grads, factor * want)
            assert all(map(torch.equal, grads, before)), "inputs were written"
            apart = [g.clone() for g in grads]
            same, got = gradients.clip_grads(apart, factor * want, out=apart)
            assert torch.equal(got, norm) and all(a is b for a, b in zip(same, apart))
            assert all(map(torch.equal, apart, clipped)), name
            if factor > 1:
                assert all(map(torch.equal, clipped, grads)), name
        assert torch.equal(gradients.grad_norm(grads), norm), "not the same bits twice"


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_of_inputs_and_outputs(dtype, cuda_device):
    """Every pair of offsets from a 16-byte boundary; what lies around the outputs stays."""
    from ictc_o2_hp_b200 import gradients
    n, size = 20011, 16 // torch.empty((), dtype=dtype).element_size()
    source = rand((n + 16,), dtype, cuda_device, 11)
    for i in range(size):
        grads = [source[i:i + n]]
        for o in range(size):
            flat = torch.full((n + 16,), 7.0, dtype=dtype, device=cuda_device)
            _, norm = gradients.clip_grads(grads, 1.0, out=[flat[o:o + n]])
            check_norm(norm, norm64(grads))
            check_clipped([flat[o:o + n]], grads, 1.0)
            assert (flat[:o] == 7).all() and (flat[o + n:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-38, 1e-25, 1e-16, 1e16, 1e19, 1e30, 3e37])
def test_range(scale, dtype, cuda_device):
    """Squares leave float32 long before the gradients do; the norm does not."""
    from ictc_o2_hp_b200 import gradients
    grads = [rand((1003,), dtype, cuda_device, 21).clamp(-3, 3) * scale,
             rand((40,), dtype, cuda_device, 22) * scale * 1e-3]
    grads = [g.clamp(-3e38, 3e38) for g in grads]
    want = norm64(grads)
    if want < 3.4e38:
        norm = gradients.grad_norm(grads)
        assert abs(norm.item() - want) <= 5 * U * want + 2.0 ** -149
    if 1e-3 < want < 1e37:
        clipped, _ = gradients.clip_grads(grads, want / 8)
        check_clipped(clipped, grads, want / 8)


def test_offsets_past_32_bits(cuda_device):
    """One tensor of more than 2^31 elements, a value past the end of 32 bits that decides."""
    from ictc_o2_hp_b200 import gradients
    n = 2 ** 31 + 100_003
    big = torch.zeros(n, dtype=torch.bfloat16, device=cuda_device)
    big[-3], big[5] = 3.0, 4.0
    assert gradients.grad_norm([big]).item() == 5.0
    assert gradients.grad_norm([big], math.inf).item() == 4.0
    _, norm = gradients.clip_grads([big], 2.5, out=[big])
    assert norm.item() == 5.0 and abs(big[-3].item() - 1.5) <= 1.5 * 2.0 ** -8
    assert abs(big[5].item() - 2.0) <= 2.0 * 2.0 ** -8 and big.count_nonzero().item() == 2


def test_new_outputs_are_tensors_of_their_own(cuda_device):
    """Parts of one allocation: aligned, apart, usable as leaves and in place."""
    from ictc_o2_hp_b200 import gradients
    grads = [rand((n,), t, cuda_device, 26) for n in (1, 7, 100, 0) for t in DTYPES]
    grads.append(rand((5, 9), torch.float32, cuda_device, 27).t())
    clipped, _ = gradients.clip_grads(grads, 0.1)
    check_clipped(clipped, grads, 0.1)
    assert clipped[-1].stride() == grads[-1].stride()
    assert all(t.data_ptr() % 64 == 0 for t in clipped if t.numel())
    before = [t.clone() for t in clipped]
    clipped[2].add_(1)
    clipped[2].requires_grad_(True)
    (clipped[2].float() * 3).sum().backward()
    assert torch.equal(clipped[2].grad, torch.full_like(before[2], 3.0))
    assert all(torch.equal(a, b) for i, (a, b) in enumerate(zip(clipped, before)) if i != 2)
    held = clipped[5]
    del clipped
    torch.empty(1 << 20, device=cuda_device).fill_(7.0)
    assert torch.equal(held, before[5])


def test_a_single_tensor(cuda_device):
    from ictc_o2_hp_b200 import gradients
    g = rand((3, 50), torch.float32, cuda_device, 25)
    check_norm(gradients.grad_norm(g), norm64([g]))
    clipped, norm = gradients.clip_grads((t for t in [g]), 0.1)
    check_clipped(clipped, [g], 0.1)


def test_zeros(cuda_device):
    from ictc_o2_hp_b200 import gradients
    grads = [torch.zeros(100_000, dtype=t, device=cuda_device) for t in DTYPES]
    for kind in (2.0, math.inf):
        clipped, norm = gradients.clip_grads(grads, 1.0, kind)
        assert norm.item() == 0 and not any(t.any() for t in clipped)
    clipped, norm = gradients.clip_grads([torch.ones(50, device=cuda_device)], 0.0)
    assert not clipped[0].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nonfinite(bad, kind, dtype, cuda_device):
    """As torch.nn.utils: a NaN norm makes all NaN, an infinite one zeros and NaN."""
    from ictc_o2_hp_b200 import gradients
    for at in (0, 7, 30_000, 40_010):
        params = [torch.nn.Parameter(torch.zeros(s, dtype=dtype, device=cuda_device))
                  for s in (9, 40_011)]
        for i, p in enumerate(params):
            p.grad = rand(p.shape, dtype, cuda_device, 30 + i)
        params[1].grad[at] = bad
        copies = [torch.nn.Parameter(torch.zeros_like(p)) for p in params]
        for p, q in zip(params, copies):
            q.grad = p.grad.clone()
        norm = gradients.clip_grad_norm_(params, 1.0, kind)
        want = torch.nn.utils.clip_grad_norm_(copies, 1.0, kind)
        assert norm.isnan() if math.isnan(bad) else norm.item() == math.inf == want.item()
        for p, q in zip(params, copies):
            assert torch.equal(p.grad.nan_to_num(5.0), q.grad.nan_to_num(5.0))
        for p, q in zip(params, copies):
            p.grad = q.grad = rand(p.shape, dtype, cuda_device, 33)
        params[0].grad = params[0].grad.clone()
        params[0].grad[3] = bad
        before = [p.grad.clone() for p in params]
        with pytest.raises(RuntimeError, match="not clipped"):
            gradients.clip_grad_norm_(params, 1.0, kind, error_if_nonfinite=True)
        assert all(torch.equal(p.grad.nan_to_num(5.0), b.nan_to_num(5.0))
                   for p, b in zip(params, before))


def test_strides(cuda_device):
    """Transposed, sliced, expanded and negated gradients; outputs of other orders."""
    from ictc_o2_hp_b200 import gradients
    for dtype in DTYPES:
        base = rand((60, 70), dtype, cuda_device, 41)
        z = torch.complex(*(rand((50,), torch.float32, cuda_device, s) for s in (42, 43)))
        grads = [base.t(), base[:, 3:50], base[::2], base[:1].expand(9, 70),
                 rand((5, 6, 7), dtype, cuda_device, 44).permute(2, 0, 1), z.conj().imag]
        assert grads[-1].is_neg()
        want = norm64(grads)
        check_norm(gradients.grad_norm(grads), want)
        clipped, norm = gradients.clip_grads(grads, 0.4 * want)
        check_norm(norm, want)
        check_clipped(clipped, grads, 0.4 * want)
        outs = [torch.empty(g.shape[::-1], dtype=g.dtype, device=cuda_device).permute(
            *range(g.dim())[::-1]) for g in grads]
        gradients.clip_grads(grads, 0.4 * want, out=outs)
        assert all(map(torch.equal, outs, clipped))
        # in place, where the memory has gaps
        wide = rand((40, 90), dtype, cuda_device, 45)
        held, keep = wide[:, 5:60], wide.clone()
        gradients.clip_grads([held], 0.5, out=[held])
        check_clipped([held], [keep[:, 5:60]], 0.5)
        keep[:, 5:60] = held
        assert torch.equal(wide, keep)


def test_parameters(cuda_device):
    """Gradients in place, those that are None left out, the same tensors and versions
    counted up."""
    from ictc_o2_hp_b200 import gradients
    model = torch.nn.Sequential(torch.nn.Linear(30, 50), torch.nn.Linear(50, 7)).to(cuda_device)
    other = torch.nn.Parameter(torch.ones(3, device=cuda_device))
    loss = model(rand((20, 30), torch.float32, cuda_device, 51)).square().sum()
    loss.backward()
    params = [*model.parameters(), other]
    before = [p.grad.clone() for p in params[:-1]]
    held = [(p.grad, p.grad._version) for p in params[:-1]]
    norm = gradients.clip_grad_norm_(iter(params), 0.7)
    check_norm(norm, norm64(before))
    check_clipped([p.grad for p in params[:-1]], before, 0.7)
    assert other.grad is None
    assert all(p.grad is g and g._version > v for p, (g, v) in zip(params, held))
    want = torch.nn.utils.clip_grad_norm_(params, 0.7)
    assert abs(want.item() - 0.7) <= 1e-5
    check_norm(gradients.clip_grad_norm_(params[0], 1e9), norm64([params[0].grad]))
    assert gradients.clip_grad_norm_([other], 1.0).item() == 0
    assert gradients.grad_norm([]).item() == 0 and gradients.clip_grads([], 1.0)[0] == []
    with torch.inference_mode():
        grads = [torch.ones(9, device=cuda_device)]
        gradients.clip_grads(grads, 1.5, out=grads)
        check_clipped(grads, [torch.ones(9, device=cuda_device)], 1.5)


def test_gradients_that_require_grad(cuda_device):
    """Gradients under create_graph are clipped as values."""
    from ictc_o2_hp_b200 import gradients
    w = rand((6, 5), torch.float32, cuda_device, 61).requires_grad_(True)
    g = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    assert g[0].requires_grad
    clipped, norm = gradients.clip_grads(g, 1.0)
    assert not norm.requires_grad and not clipped[0].requires_grad
    check_clipped(clipped, [g[0].detach()], 1.0)


def test_other_stream_and_graph_capture(cuda_device):
    """Two captured steps and an eager one share nothing."""
    from ictc_o2_hp_b200 import gradients
    for sizes in ((9, 100), (9, 100, 70_001, 2_000_003)):
        sets = [[rand((n,), torch.float32, cuda_device, 70 + 10 * k + n % 7) for n in sizes]
                for k in range(2)]
        want = [gradients.clip_grads(s, 1.0) for s in sets]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = gradients.clip_grads(sets[0], 1.0)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got[1], want[0][1]) and all(map(torch.equal, got[0], want[0][0]))
        graphs, held, outs = [], [[torch.zeros_like(t) for t in s] for s in sets], []
        for grads in held:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(gradients.clip_grads(grads, 1.0))
            graphs.append(graph)
        for grads, source in zip(held, sets):
            for t, s in zip(grads, source):
                t.copy_(s)
        for graph in (graphs[0], graphs[1], graphs[0]):
            graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out[1], w[1]) and all(map(torch.equal, out[0], w[0]))


def test_compile_and_traces(cuda_device):
    from torch.fx.experimental.proxy_tensor import make_fx

    from ictc_o2_hp_b200 import gradients
    a, b = (rand((n,), torch.float32, cuda_device, 80 + n % 9) for n in (300, 77))

    def whole(a, b):
        clipped, norm = gradients.clip_grads([a * 2, b], 1.0)
        return *clipped, norm, gradients.grad_norm([a, b], math.inf)

    want = whole(a, b)
    run = torch.compile(whole, fullgraph=True, backend="aot_eager")
    assert all(map(torch.equal, run(a, b), want))
    recorded = make_fx(whole)(torch.zeros_like(a), torch.ones_like(b))
    assert all(map(torch.equal, recorded(a, b), want))

    def in_place(a, b):
        return gradients.clip_grads([a, b], 1.0, out=[a, b])[1]

    held = [a.clone(), b.clone()]
    norm = torch.compile(in_place, fullgraph=True, backend="aot_eager")(*held)
    check_norm(norm, norm64([a, b]))
    check_clipped(held, [a, b], 1.0)


def test_training_step_of_gated_blocks(cuda_device):
    """Gated block, loss, backward, clipping: the gradients of the same network in float64,
    scaled."""
    from ictc_o2_hp_b200 import GatedBlock, Linear, gradients
    torch.manual_seed(2)
    model = torch.nn.Sequential(GatedBlock(24, 56), Linear(24, 5)).to(cuda_device)
    x = rand((300, 24), torch.float32, cuda_device, 1)
    model(x).square().sum().backward()
    params = dict(model.named_parameters())
    wide = {k: p.detach().double().requires_grad_(True) for k, p in params.items()}
    f = torch.nn.functional
    z = f.layer_norm(x.double(), (24,), wide["0.norm.weight"], wide["0.norm.bias"])
    pg, pu = f.linear(z, wide["0.gated.weight"], wide["0.gated.bias"]).chunk(2, -1)
    h = x.double() + f.linear(f.silu(pg) * pu, wide["0.down.weight"], wide["0.down.bias"])
    f.linear(h, wide["1.weight"], wide["1.bias"]).square().sum().backward()
    want = norm64([p.grad for p in wide.values()])
    norm = gradients.clip_grad_norm_(params.values(), 2.0)
    assert abs(norm.item() - want) <= 1e-5 * want
    for k, p in params.items():
        exact = wide[k].grad * (2.0 / want)
        assert (p.grad.double() - exact).norm() <= 2e-5 * max(exact.norm().item(), 1e-3), k


def test_refusals(cuda_device):
    from ictc_o2_hp_b200 import gradients
    a, b = (torch.ones(8, device=cuda_device) for _ in range(2))
    for bad in (a.double(), a.to(torch.complex64), a.int(), a.cpu(), a.to_sparse()):
        with pytest.raises(TypeError):
            gradients.grad_norm([a, bad])
        with pytest.raises(TypeError):
            gradients.clip_grads([bad, a], 1.0)
    for call in (
        lambda: gradients.grad_norm([a], 1.0),
        lambda: gradients.clip_grads([a], -1.0),
        lambda: gradients.clip_grads([a], math.nan),
        lambda: gradients.clip_grads([a], 1.0, out=[]),
        lambda: gradients.clip_grads([a], 1.0, out=[b[:7]]),
        lambda: gradients.clip_grads([a], 1.0, out=[b.half()]),
        lambda: gradients.clip_grads([a], 1.0, out=[b.cpu()]),
        lambda: gradients.clip_grads([a], 1.0, out=[b[:1].expand(8)]),
        lambda: gradients.clip_grads([a, a], 1.0, out=[a, a]),
        lambda: gradients.clip_grads([a, b], 1.0, out=[b, a]),
        lambda: gradients.clip_grads([a[:4], b], 1.0, out=[a[2:6], b]),
        lambda: gradients.clip_grads([a, b], 1.0, out=[b, b]),
        lambda: gradients.clip_grads([], 1.0, out=[a]),
    ):
        with pytest.raises(ValueError):
            call()
    assert (a == 1).all() and (b == 1).all()
    # gradients that share memory with each other are read, and may
    both, norm = gradients.clip_grads([a, a, a[2:5]], 1.0, out=[b, torch.empty_like(b), b.new_empty(3)])
    assert abs(norm.item() - math.sqrt(19)) <= 1e-6 and torch.equal(both[0], both[1])
    b.fill_(1)
    whole = torch.ones(64, device=cuda_device)
    for grads, outs in (([whole[:8], whole[40:48]], [whole[8:16], whole[44:52]]),
                        ([whole[40:48], whole[:8]], [whole[16:24], whole[20:28]]),
                        ([whole[:32], whole[32:]], [whole[32:], whole[:32]])):
        with pytest.raises(ValueError, match="share memory"):
            gradients.clip_grads(grads, 1.0, out=outs)
    assert (whole == 1).all()
    p = torch.nn.Parameter(a)
    p.grad = b
    with pytest.raises(ValueError, match="once"):
        gradients.clip_grad_norm_([p, p], 1.0)


def test_outputs_with_gaps_that_share_memory(cuda_device):
    """Slices are refused where they share elements with another output or gradient, and only
    there: slices of one tensor may lie in each other's gaps."""
    from ictc_o2_hp_b200 import gradients
    wide = torch.ones(30, 24, device=cuda_device)
    like = torch.ones(30, 8, device=cuda_device)
    cube = torch.ones(6, 4, 10, device=cuda_device)
    v = wide[:, 5:20]
    for grads, outs in (
        ([v, v], [v, v]),
        ([v, wide[:, 5:20]], [v, wide[:, 5:20]]),
        ([like, like], [wide[:, :8], wide[:, 7:15]]),
        ([like, wide.view(-1)[24:48]], [wide[:, :8], wide.view(-1)[24:48]]),
        ([like, torch.ones(24, device=cuda_device)], [wide[:, :8], wide[7]]),
        ([like, wide[3]], [wide[:, 16:24], torch.ones(24, device=cuda_device)]),
        ([wide[:, :8]], [wide[:, 4:12]]),
        ([wide[:, ::2], wide[:, ::3]], [wide[:, ::2], wide[:, ::3]]),
        ([cube[:, 1:3], cube[:, :, 3:5]], [cube[:, 1:3], cube[:, :, 3:5]]),
        ([torch.ones(8, 3, device=cuda_device)], [wide.view(-1).as_strided((8, 3), (2, 3))]),
    ):
        with pytest.raises(ValueError, match="share memory"):
            gradients.clip_grads(grads, 0.5, out=outs)
    assert (wide == 1).all() and (cube == 1).all()
    p = torch.nn.Parameter(v.clone())
    p.grad = v
    with pytest.raises(ValueError, match="once"):
        gradients.clip_grad_norm_([p, p], 0.5)
    assert (wide == 1).all()

    for lists in ([wide[:, :8], wide[:, 8:16], wide[:, 16:]], [wide[:, ::2], wide[:, 1::2]],
                  [wide[::2], wide[1::2]], [cube[:, ::2], cube[:, 1::2]],
                  [cube[:, :, :5], cube[:, 1:3, 5:], wide.t()[:, :30]],
                  [wide[:15, :20].t(), wide[15:, :20], wide[:15, 20:]]):
        before = [t.clone() for t in lists]
        gradients.clip_grads(lists, 0.5, out=lists)
        check_clipped(lists, before, 0.5)
        wide.fill_(1)
        cube.fill_(1)
    # a gradient by two views of it, the distance of a single row being nobody's
    one = wide[:, 3:4]
    gradients.clip_grads([one], 0.5, out=[wide.as_strided((30, 1), (24, 5), 3)])
    check_clipped([one], [torch.ones(30, 1, device=cuda_device)], 0.5)
    wide.fill_(1)
    # gradients that share memory with each other are read, and may
    clipped, _ = gradients.clip_grads([wide[:, :8], wide[:, 4:12]], 0.5,
                                      out=[torch.empty_like(like), torch.empty(8, 30, device=cuda_device).t()])
    assert torch.equal(clipped[0], clipped[1])


def test_dual_tensors_are_refused(cuda_device):
    """Scaling a dual tensor's value alone would leave it a tangent of another function."""
    from torch.autograd import forward_ad

    from ictc_o2_hp_b200 import gradients
    a, b = (torch.ones(8, device=cuda_device) for _ in range(2))
    p = torch.nn.Parameter(torch.ones(8, device=cuda_device))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(a, torch.ones_like(a))
        p.grad = dual
        for call in (lambda: gradients.grad_norm([b, dual]), lambda: gradients.clip_grads([dual], 0.5),
                     lambda: gradients.clip_grads([dual], 0.5, out=[dual]),
                     lambda: gradients.clip_grads([dual[::2]], 0.5, out=[dual[::2]]),
                     lambda: gradients.clip_grads([b], 0.5, out=[dual]),
                     lambda: gradients.clip_grad_norm_([p], 0.5)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        gradients.clip_grads([b], 0.5, out=[b])  # others go on
    assert (a == 1).all() and abs(b.norm().item() - 0.5) <= 1e-5
