"""``ops.orthogonalize`` and ``ops.muon_step_`` against float64 (``oracle/train.py``), within its bound on 22-bit operands and
FP32 sums (``schulz_bound``) and the output's own rounding."""

import math

import pytest
import torch

from flashim_amd import ops
from oracle import train as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0**-9, F16: 2.0**-12, F32: 2.0**-24}  # half a step
TINY = {BF16: 2.0**-134, F16: 2.0**-25, F32: 2.0**-150}


def _gradient(*shape, seed=0, dtype=F32, floor=0.05):
    """A few strong directions over a floor of noise."""
    g = torch.Generator().manual_seed(seed)
    few = min(6, *shape[-2:])
    strong = torch.randn(*shape[:-1], few, generator=g) * torch.exp(-0.5 * torch.arange(few))
    noise = torch.randn(*shape, generator=g)
    return ((strong @ torch.randn(*shape[:-2], few, shape[-1], generator=g) + floor * noise) * 1e-2).to(dtype)


def _check(got, u, what="", **kwargs):
    """Each matrix of ``got`` against ``orthogonalize(u)``."""
    kinds, half = got.dtype, 2 * U[got.dtype]
    got = got.double().cpu().reshape(-1, *u.shape[-2:])
    for i, m in enumerate(u.reshape(-1, *u.shape[-2:])):
        want = ref.orthogonalize(m, **kwargs)
        off, bound = (got[i] - want).norm().item(), ref.schulz_bound(m, **kwargs)
        rounding = half * want.norm().item() + TINY[kinds] * math.sqrt(want.numel())
        assert off <= bound + rounding, (what, i, off, bound, rounding)


SHAPES = [(1, 1), (1, 50), (7, 3), (16, 512), (16, 16), (17, 33), (32, 1000), (33, 31), (48, 100), (64, 256), (64, 448), (40, 64),
          (256, 64), (523, 60), (65, 65), (64, 600), (96, 96), (128, 512), (512, 128), (196, 523), (523, 196), (257, 129),
          (300, 1000)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, dtype):
    g = _gradient(*shape, seed=sum(shape), dtype=dtype)
    got = ops.orthogonalize(g.to(DEV))
    assert got.shape == g.shape and got.dtype == dtype
    _check(got, g)


@pytest.mark.parametrize("shape", [(5, 24, 40), (3, 2, 130, 70), (20, 64, 64)])
def test_stacks(shape):
    g = _gradient(*shape, seed=3)
    _check(ops.orthogonalize(g.to(DEV), out_dtype=BF16), g)
    _check(ops.orthogonalize(g.to(DEV)), g)


def test_large():
    g = _gradient(520, 2100, seed=5, dtype=BF16)
    _check(ops.orthogonalize(g.to(DEV), out_dtype=F32), g)


@pytest.mark.parametrize("shape", [(5, 7), (64, 256), (70, 600), (300, 90)])
def test_conversion_keeps_fp32(shape):
    """One step of X = 1 X: what the halves hold, element by element: 2^-23 of each, twice (X and a product of 1), 2^-24 where a
    term of the low halves is left out, and the sums' own roundings; a thousandth part of lo below FP16's normal numbers."""
    g = _gradient(*shape, seed=7)
    got = ops.orthogonalize(g.to(DEV), steps=1, coefficients=(1.0, 0.0, 0.0)).double().cpu()
    want = g.double() / (g.double().norm() + 1e-7)
    assert ((got - want).abs() <= 2.0**-20 * want.abs() + 2.0**-28).all()


@pytest.mark.parametrize("steps, coefficients", [(1, (1.5, -0.5, 0.0)), (12, (1.5, -0.5, 0.0)), (3, (0.0, 0.0, 1.0)),
                                                 (10, (1.875, -1.25, 0.375)), (6, (2.0, -1.5, 0.5)), (4, (-1.5, 0.5, 0.0))])
@pytest.mark.parametrize("shape", [(24, 40), (100, 600)])
def test_coefficients(shape, steps, coefficients):
    g = _gradient(*shape, seed=8)
    _check(ops.orthogonalize(g.to(DEV), steps=steps, coefficients=coefficients), g, steps=steps, coefficients=coefficients)


@pytest.mark.parametrize("shape", [(24, 40), (130, 200)])
@pytest.mark.parametrize("scale", [1e-30, 1e-9, 1e12, 1e30])
def test_magnitudes(shape, scale):
    """Squares past FP32's range; a norm near eps and below it."""
    g = (_gradient(*shape, seed=9) * scale).float()
    _check(ops.orthogonalize(g.to(DEV)), g)
    _check(ops.orthogonalize(g.to(DEV), eps=1e-3), g, eps=1e-3)


@pytest.mark.parametrize("shape", [(24, 40), (40, 24), (130, 200)])
def test_zeros_and_nonfinite(shape):
    zero = torch.zeros(shape, device=DEV)
    assert (ops.orthogonalize(zero) == 0).all()
    stack = torch.stack([_gradient(*shape, seed=10).to(DEV) for _ in range(4)])
    want = ops.orthogonalize(stack)
    stack[1, 3, 5], stack[2, 0, 0] = math.nan, math.inf
    got = ops.orthogonalize(stack)
    assert torch.isnan(got[1]).all() and torch.isnan(got[2]).all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 4, 4), (3, 0, 4)])
def test_empty(shape):
    g = torch.empty(shape, device=DEV)
    assert ops.orthogonalize(g).shape == g.shape
    ops.muon_step_([g], [g.clone()], [g.clone()], lr=0.1)


def test_layouts():
    """Transposed and strided gradients, and views at odd offsets: the values of their packed copies."""
    base = _gradient(90, 150, seed=11, dtype=BF16).to(DEV)
    for view in (base.t(), base[::2, 1:91], base[3:40], base.reshape(-1)[7:7 + 80 * 33].view(80, 33),
                 base.reshape(-1)[1:1 + 12 * 9 * 30].view(12, 9, 30).transpose(0, 1)):
        assert torch.equal(ops.orthogonalize(view), ops.orthogonalize(view.contiguous()))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(7, 3696), (2500, 30), (16, 2400), (40, 1500), (1300, 48), (64, 449), (4000, 63), (3, 20000), (2, 33, 1300)])
def test_thin(shape, dtype):
    """Few rows or columns, too long for one workgroup: slabs of the other side."""
    g = _gradient(*shape, seed=13, dtype=dtype)
    _check(ops.orthogonalize(g.to(DEV)), g)


def test_steps_of_thin_ones():
    shapes = [(16, 2400), (2400, 16), (3, 32, 1300), (64, 600), (700, 50), (5, 4000), (40, 1200), (1200, 33)]
    for p_dtype, g_dtype in ((F32, BF16), (BF16, F32)):
        _check_step(*_triples(shapes, p_dtype, g_dtype, seed=6), lr=0.3, weight_decay=0.2)
    _check_step(*_triples(shapes, F32, F32, seed=7), lr=0.3, nesterov=False, steps=1)


def test_many_small_ones():
    g = _gradient(700, 9, 14, seed=12)
    _check(ops.orthogonalize(g.to(DEV)), g)


# -- the step ------------------------------------------------------------------------------------------------------------


def _step(p, g, m, *, lr, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="original", steps=5):
    """One matrix or stack, float64: the parameter, the momentum, and the parameter's bound."""
    m = momentum * m.double() + g.double()
    u = g.double() + momentum * m if nesterov else m
    rows, cols = p.shape[-2:]
    f = {"original": max(1.0, rows / cols) ** 0.5, "match_rms": 0.2 * max(rows, cols) ** 0.5, "none": 1.0}[adjust]
    flat = u.reshape(-1, rows, cols)
    o = torch.stack([ref.orthogonalize(x, steps=steps) for x in flat]).reshape(u.shape)
    # u itself is rounded to FP32, one or two FMAs: as any operand's error
    off = torch.tensor([2 * ref.schulz_bound(x, steps=steps) for x in flat]).reshape(*u.shape[:-2], 1, 1)
    return p.double() * (1 - lr * weight_decay) - lr * f * o, m, lr * f * off


def _check_step(params, grads, momenta, **kwargs):
    before = [[t.cpu().clone() for t in ts] for ts in (params, grads, momenta)]
    ops.muon_step_(params, grads, momenta, **kwargs)
    for p, g, m, p0, g0, m0 in zip(params, grads, momenta, *before):
        want, want_m, off = _step(p0, g0, m0, **kwargs)
        assert torch.equal(g.cpu(), g0)
        assert ((m.double().cpu() - want_m).abs() <= 2.0**-22 * (m0.double().abs() + g0.double().abs())).all()
        error = (p.double().cpu() - want)
        per = error.reshape(-1, *error.shape[-2:]).norm(dim=(1, 2))
        bound = off.reshape(-1) + (2 * U[p.dtype] + 2.0**-22) * (want.abs() + p0.double().abs()).reshape(-1, *error.shape[-2:]).norm(dim=(1, 2))
        assert (per <= bound).all(), (p.shape, (per / bound).max())


def _triples(shapes, p_dtype, g_dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    params = [(torch.randn(s, generator=g) * s[-1] ** -0.5).to(p_dtype).to(DEV) for s in shapes]
    grads = [_gradient(*s, seed=seed + i, dtype=g_dtype).to(DEV) for i, s in enumerate(shapes)]
    momenta = [5 * _gradient(*s, seed=seed + 50 + i).to(DEV) for i, s in enumerate(shapes)]
    return params, grads, momenta


MIXED = [(64, 256), (256, 64), (17, 5), (1, 9), (90, 90), (3, 20, 30), (130, 260), (260, 130), (2, 70, 300), (16, 700), (33, 40)]


@pytest.mark.parametrize("p_dtype, g_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (BF16, F32), (F16, BF16)])
def test_step(p_dtype, g_dtype):
    _check_step(*_triples(MIXED, p_dtype, g_dtype), lr=0.3, weight_decay=0.2)


@pytest.mark.parametrize("kwargs", [dict(nesterov=False), dict(momentum=0.0), dict(momentum=0.5, steps=2), dict(adjust="match_rms"),
                                    dict(adjust="none", weight_decay=1.0), dict(lr=0.0, weight_decay=0.5)])
def test_step_options(kwargs):
    _check_step(*_triples([(24, 40), (130, 70), (40, 24)], F32, F32, seed=1), **{"lr": 0.1, **kwargs})


def test_step_of_many_matrices():
    """More than one launch's table."""
    _check_step(*_triples([(12 + i % 5, 20 + i % 7) for i in range(70)] + [(100, 68)] * 30, F32, F32, seed=2), lr=0.1)


def test_packed_views_at_odd_offsets_and_strided_tensors():
    shapes = [(7, 9), (65, 70), (20, 31)]
    sizes = [a * b for a, b in shapes]
    buckets = [torch.full((sum(sizes) + 4,), 9.0, dtype=t, device=DEV) for t in (BF16, F16, F32)]
    views = [[b[1:1 + sum(sizes)].split(sizes)[i].view(s) for i, s in enumerate(shapes)] for b in buckets]
    for view, new in zip(views, _triples(shapes, BF16, F16, seed=3)):
        for v, n in zip(view, new):
            v.copy_(n)
    _check_step(*views, lr=0.1)
    assert all((b[:1] == 9).all() and (b[-3:] == 9).all() for b in buckets)
    big = torch.randn(3, 40, 60, device=DEV)
    strided = [[big[i].t()[:, ::2]] for i in range(3)]
    rest = big.clone()
    _check_step(*strided, lr=0.1)
    assert torch.equal(big[0][1::2], rest[0][1::2]) and torch.equal(big[2][1::2], rest[2][1::2])


def test_same_bits_on_any_stream_and_versions():
    args = _triples([(64, 256), (130, 260)], F32, F32, seed=4)
    copies = [[[t.clone() for t in ts] for ts in args] for _ in range(3)]
    side = torch.cuda.Stream()
    for c in copies:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.muon_step_(*c, lr=0.1)
        side.synchronize()
    for c in copies[1:]:
        assert all(torch.equal(a, b) for x, y in zip(c, copies[0]) for a, b in zip(x, y))
    versions = [[t._version for t in ts] for ts in args]
    ops.muon_step_(*args, lr=0.1)
    assert [[t._version - v for t, v in zip(ts, vs)] for ts, vs in zip(args, versions)] == [[1, 1], [0, 0], [1, 1]]


def test_graph_capture():
    """Replayed on new gradients with eager work and synchronizations between, against eager steps from the same state."""
    shapes = [(64, 256), (130, 260), (512, 1100)]
    params, grads, momenta = _triples(shapes, F32, F32, seed=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.muon_step_([p.clone() for p in params], grads, [m.clone() for m in momenta], lr=0.1)
        ops.orthogonalize(grads[2])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_step_(params, grads, momenta, lr=0.1)
        o = ops.orthogonalize(grads[2])
    eager = [[t.clone() for t in ts] for ts in (params, momenta)]
    for seed in range(3):
        for g, new in zip(grads, _triples(shapes, F32, F32, seed=20 + seed)[1]):
            g.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        ops.muon_step_(eager[0], grads, eager[1], lr=0.1)
        assert torch.equal(o, ops.orthogonalize(grads[2]))
        assert all(torch.equal(a, b) for a, b in zip(params + momenta, eager[0] + eager[1]))


def test_refusals():
    g = torch.ones(4, 5, device=DEV)
    for bad in (g.double(), g[0], g.cpu(), g.long()):
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.orthogonalize(bad)
    for kwargs in (dict(steps=0), dict(steps=101), dict(coefficients=(1.0, 2.0)), dict(eps=-1.0), dict(out_dtype=torch.float64)):
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.orthogonalize(g, **kwargs)
    from flashim_amd._lib import UnsupportedShape

    for coefficients in ((9.0, -20.0, 9.0), (3.0, 1.0, 1.0), (math.nan, 0.0, 0.0), (100.0, 0.0, 0.0)):
        with pytest.raises(UnsupportedShape):
            ops.orthogonalize(g, coefficients=coefficients)
    p, m = g.clone(), g.clone()
    for args in (([p], [g], []), ([p], [g[:3]], [m]), ([p], [g], [m.bfloat16()]), ([p[0]], [g[0]], [m[0]]), ([p], [g.cpu()], [m]),
                 ([], [], []), ([p.double()], [g], [m]), (p, g, m)):
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.muon_step_(*args, lr=0.1)
    with pytest.raises(NotImplementedError, match="no HIP impl"):
        ops.muon_step_([p], [g], [m], lr=0.1, adjust="half")
    with pytest.raises(ValueError, match="twice"):
        ops.muon_step_([p, p], [g, g], [m, m.clone()], lr=0.1)
    leaf = g.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="not implemented"):
        ops.orthogonalize(leaf).sum().backward()
    with pytest.raises(NotImplementedError, match="no derivative"):
        torch.ops.flashim_amd.muon_step_([leaf], [g], [m], 0.1, 0.9, True, 0.0, 0, 5, 3.0, -3.0, 1.0, 1e-7)
    assert torch.equal(p, g) and torch.equal(m, g)


@pytest.mark.parametrize("shape", [(64, 70000), (64, 140000), (12, 300000), (140000, 40)])
def test_long_matrices_of_few_rows(shape):
    """On both sides of the length up to which slabs' workgroups read each other's parts."""
    g = _gradient(*shape, seed=31)
    _check(ops.orthogonalize(g.to(DEV)), g)


@pytest.mark.parametrize("shape", [(70, 5_500_000), (5_500_000, 70), (12, 5_000_000), (40, 8_000_000)])
def test_offsets_past_31_bits(shape):
    """Zero but for some columns at the ends and between: exact zeros there, and the others' own matrix orthogonalized."""
    m, n = min(shape), max(shape)
    g = torch.Generator().manual_seed(32)
    at = torch.cat([torch.arange(60), torch.randint(60, n - 60, (100,), generator=g).unique(), torch.arange(n - 60, n)])
    few = _gradient(m, at.numel(), seed=33)
    u = torch.zeros(m, n, device=DEV)
    u[:, at.to(DEV)] = few.to(DEV)
    got = ops.orthogonalize(u.t().contiguous() if shape[0] > shape[1] else u)
    del u
    got = got.t() if shape[0] > shape[1] else got
    _check(got[:, at.to(DEV)], few)
    assert got.count_nonzero().item() == got[:, at.to(DEV)].count_nonzero().item()


def test_tensors_that_overlap_are_refused():
    w = torch.randn(4, 16, 32, device=DEV)
    g, m = torch.randn_like(w), torch.zeros_like(w)
    square = torch.randn(16, 16, device=DEV)
    before = [t.clone() for t in (w, g, m, square)]
    for params, grads, momenta in (([w, w[1]], [g, g[1]], [m, m[1].clone()]),  # a part of another
                                   ([w[0], w[1]], [g[0], g[1]], [m[0], m[0]]),  # a momentum twice
                                   ([w], [w], [m]), ([w], [m], [m]),  # the gradient is written
                                   ([w], [g], [w]),
                                   ([square, square.t()], [g[0, :, :16], g[1, :, :16]], [m[0, :, :16], m[1, :, :16]]),
                                   ([w[:2], w[1:3]], [g[:2], g[1:3]], [m[:2], m[:2].clone()])):
        with pytest.raises(ValueError, match="overlaps"):
            ops.muon_step_(params, grads, momenta, lr=0.1)
    with pytest.raises(RuntimeError, match="single memory location"):
        ops.muon_step_([square[:1].expand(16, 16)], [g[0, :, :16]], [torch.zeros(16, 16, device=DEV)], lr=0.1)
    assert all(torch.equal(t, b) for t, b in zip((w, g, m, square), before))
    # neighbours, halves of one matrix's columns and a gradient for two parameters are apart
    ops.muon_step_([w[0], w[1], w[2, :, :16], w[2, :, 16:]], [g[0], g[0], g[2, :, :16], g[2, :, 16:]],
                   [m[0], m[1], m[2, :, :16], m[2, :, 16:]], lr=0.1)
    assert torch.equal(w[3], before[0][3]) and not torch.equal(w[2], before[0][2])


@pytest.mark.parametrize("shape", [(4, 4), (24, 40), (40, 24), (7, 3696), (130, 200), (200, 130)])
def test_norms_whose_scale_fp32_does_not_hold(shape):
    """2^15 / |g| is past FP32's largest number, or near its smallest; an eps beside which only a zero matrix counts."""
    for scale in (1e-34, 1e-41, 1e38):
        g = (_gradient(*shape, seed=41).double() * scale).float()
        assert g.count_nonzero() > 0
        _check(ops.orthogonalize(g.to(DEV), eps=0.0), g, scale, eps=0.0)
        _check(ops.orthogonalize(g.to(DEV), eps=1e-40), g, scale, eps=1e-40)
    zero = torch.zeros(shape, device=DEV)
    for eps in (1e-40, 5e-324):
        assert (ops.orthogonalize(zero, eps=eps) == 0).all()
    assert torch.isnan(ops.orthogonalize(zero, eps=0.0)).all()  # 0 / 0
    momentum = torch.zeros(shape, device=DEV)
    p = torch.ones(shape, device=DEV)
    ops.muon_step_([p], [zero], [momentum], lr=0.5, eps=1e-40)
    assert (p == 1).all()


def test_strided_tensors_that_overlap_are_refused():
    """Views with gaps, between whose rows another's may lie: what counts are the elements."""
    big, flat = torch.randn(40, 128, device=DEV), torch.randn(4000, device=DEV)
    g, m = torch.randn(40, 128, device=DEV), torch.zeros(40, 128, device=DEV)
    before = big.clone()

    def step(*params):
        grads = [g.reshape(-1)[:p.numel()].reshape(p.shape) for p in params]
        ops.muon_step_(list(params), grads, [torch.zeros_like(t) for t in grads], lr=0.1)

    for params in ((big[:, :64], big[:, 32:96]), (big[:, ::2], big[:, 2::4]), (big[::2, :10], big[10:11, 9:]), (big[:, :64], big[:, 63:].t()),
                   (flat.as_strided((5, 9), (30, 2)), flat.as_strided((4, 7), (13, 3), 1)), (big, flat.new_empty(3, 3), big[5:, 5:9])):
        with pytest.raises(ValueError, match="overlaps"):
            step(*params)
    with pytest.raises(ValueError, match="overlaps"):  # a gradient's elements
        ops.muon_step_([big[:, :64]], [big[:, 32:96]], [m[:, :64]], lr=0.1)
    with pytest.raises(ValueError, match="overlaps"):  # one tensor's own
        step(flat.as_strided((8, 8), (3, 2)))
    assert torch.equal(big, before)
    # apart, however their addresses interleave
    step(big[:, :64], big[:, 64:])
    step(big[:, ::2], big[:, 1::2].t())
    step(big[::2, :100], big[1::2], big[::2, 100:].t())
    step(flat.as_strided((5, 9), (90, 4)), flat.as_strided((4, 7), (90, 8), 2), flat.as_strided((9, 9), (11, 1), 3000))
    ops.muon_step_([big[:, :64]], [big[:, 64:]], [m[:, 3:67]], lr=0.1)


# -- precision of the products, and every form of them ------------------------------------------------------------------------


def _check_halves(got, u, **kwargs):
    """Each matrix of ``got`` (FP32) as near float64's result as FP32 arithmetic on two halves ends (``schulz_halves``), times 4: both
    are sums of hundreds and more of independent roundings of the same sizes, which pass through the same steps, in other orders.
    Half a step of the output's own besides. (What a product without its low halves would be off by is at least twice that at up to 130 rows:
    ``test_oracle_tells_a_product_without_its_low_halves``.)"""
    got = got.reshape(-1, *u.shape[-2:])
    for i, m in enumerate(u.reshape(-1, *u.shape[-2:])):
        m = m.to(DEV if m.numel() > 1 << 18 else "cpu")
        want = ref.orthogonalize(m, **kwargs)
        off, halves = ((t.to(want) - want).norm().item() for t in (got[i], ref.schulz_halves(m, **kwargs)))
        assert off <= 4 * halves + U[F32] * want.norm().item(), (i, off, halves)


@pytest.mark.parametrize("shape", [(16, 512), (64, 256), (256, 64), (48, 100), (40, 1500), (1500, 40), (7, 3696), (96, 96), (65, 65),
                                   (100, 200), (150, 130), (20, 64, 64), (300, 1000), (520, 2100)])
def test_products_keep_both_halves(shape):
    g = _gradient(*shape, seed=42)
    _check_halves(ops.orthogonalize(g.to(DEV)), g)


# (X X^T on tiles of 64 and 128, with two and four stages, whole and in parts; P and P X on either tile; by tiles a call, at 256 CUs)
PLANS = {"gram 64, square 64, two stages": [(200, 100, 200)], "gram 128, square 128": [(171, 130, 150)],
         "gram 128 with four stages": [(85, 130, 150), (100, 120)], "gram 128, square 64": [(100, 130, 150)],
         "apply 128 with four stages": [(33, 130, 150)], "gram in parts, two stages": [(1000, 4000)],
         "gram in parts, four stages": [(1000, 1300)], "tall, mixed": [(60, 150, 130), (4, 600, 260), (30, 90, 70)]}


@pytest.mark.parametrize("plan", PLANS)
def test_every_form_of_the_products(plan):
    """A step from zeros is -O."""
    grads = [_gradient(*s, seed=43 + i) for i, s in enumerate(PLANS[plan])]
    params, momenta = ([torch.zeros(s, device=DEV) for s in PLANS[plan]] for _ in range(2))
    ops.muon_step_(params, [g.to(DEV) for g in grads], momenta, lr=1.0, adjust="none", nesterov=False)
    for p, g in zip(params, grads):
        _check_halves(-p, g)
    if len(grads) == 1:
        assert torch.equal(ops.orthogonalize(grads[0].to(DEV)), -params[0])


@pytest.mark.parametrize("shape", [(128, 2048), (1600, 113), (116, 2635), (129, 2048), (112, 2048)])
def test_a_hundred_rows_and_long(shape):
    """Eight blocks of 16 rows, whose sums would leave a slab no room for a line."""
    g = _gradient(*shape, seed=44)
    _check_halves(ops.orthogonalize(g.to(DEV)), g)
    _check_step(*_triples([shape, (2, *shape)], F32, BF16, seed=45), lr=0.1)
