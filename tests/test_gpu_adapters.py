"""``ops.low_rank_adapters`` and its gradients against float64 (``oracle/train.py``): FP32 sums of each product, the middle kept
in two 16-bit numbers, one rounding of the result."""

import math

import pytest
import torch

from flashim_amd import ops
from oracle import train as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0**-8, F16: 2.0**-11}
TINY = {BF16: 2.0**-134, F16: 2.0**-25}


def _inputs(lead, k, n, r, j, dtype, seed=0, index=None, d=1.0):
    g = torch.Generator().manual_seed(seed)
    spread = torch.exp(torch.empty(k).uniform_(-1, 1, generator=g))
    x = (torch.randn(*lead, k, generator=g) * spread).to(dtype)
    base = torch.randn(*lead, n, generator=g).to(dtype)
    a = (torch.randn(j, r, k, generator=g) * k**-0.5).to(dtype)
    b = (torch.randn(j, n, r, generator=g) * 0.5 * r**-0.5).to(dtype)
    d_out = (torch.randn(*lead, n, generator=g) * d).to(dtype)
    return base, x, a, b, d_out


def _close(name, got, want, error):
    dtype = got.dtype
    got = got.detach().double().cpu()
    bound = error + HALF_STEP[dtype] * (want.abs() + error) + TINY[dtype]
    off = (got - want).abs()
    # a value past the type's range rounds to infinity: 65520 and more in FP16, its largest 65504 and half of its last step 32
    most = torch.finfo(dtype).max * (1 + HALF_STEP[dtype] / 2)
    off[torch.isinf(got) & (got.sign() == want.sign()) & (want.abs() + bound >= most)] = 0
    assert (off <= bound).all(), (name, (off / bound).max().item(), (off > bound).sum().item(), off.numel())


def _run(base, x, a, b, index, scale, d_out=None):
    dev = [None if t is None else t.to(DEV) for t in (base, x, a, b, index, scale if isinstance(scale, torch.Tensor) else None)]
    leaves = [None if t is None else t.detach().requires_grad_(d_out is not None) for t in dev[:4]]
    out = ops.low_rank_adapters(*leaves, dev[4], scale=dev[5] if dev[5] is not None else scale)
    if d_out is None:
        return out, None
    wanted = [t for t in leaves if t is not None]
    return out, dict(zip(("base", "x", "a", "b")[4 - len(wanted):], torch.autograd.grad(out, wanted, d_out.to(DEV))))


def _check(base, x, a, b, index, scale, d_out=None):
    out, grads = _run(base, x, a, b, index, scale, d_out)
    want = ref.low_rank_adapters(base, x, a, b, index, scale, d_out)
    assert out.shape == (*x.shape[:-1], b.shape[1]) and out.dtype == x.dtype
    _close("out", out, want["out"], want["out_error"])
    if d_out is not None:
        if base is not None:
            assert torch.equal(grads["base"].cpu(), d_out)
        for name in ("x", "a", "b"):
            _close(name, grads[name], want[name], want[name + "_error"])
    return out, grads


def _index(kind, lead, j, seed=0):
    g = torch.Generator().manual_seed(seed + 1)
    if kind == "all":
        return torch.tensor(j - 1)
    if kind == "image":
        return torch.randint(-1, j, lead[:1], generator=g)
    if kind == "row":  # any order
        return torch.randint(-1, j, lead, generator=g).to(torch.int32)
    m = math.prod(lead)  # runs
    ends = torch.sort(torch.randint(0, m, (3 * j,), generator=g)).values
    return torch.randint(-1, j, (3 * j + 1,), generator=g)[torch.searchsorted(ends, torch.arange(m))].reshape(lead)


SIZES = [((1,), 512, 2048, 8, 4), ((1, 1), 8, 8, 1, 1), ((3, 5), 7, 3, 3, 2), ((17,), 33, 31, 5, 3), ((64,), 1024, 520, 16, 9),
         ((2, 20, 16), 64, 256, 8, 2), ((2, 700), 196, 523, 12, 6), ((5, 130), 96, 100, 17, 3), ((600,), 40, 72, 33, 4),
         ((3, 200), 130, 65, 64, 2), ((2, 300), 48, 40, 100, 3), ((2, 2600), 32, 64, 4, 3), ((4000,), 20, 24, 16, 40)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", ["all", "image", "row", "runs"])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(size, kind, dtype):
    lead, k, n, r, j = size
    base, x, a, b, d_out = _inputs(lead, k, n, r, j, dtype, seed=k + n + r)
    scale = torch.exp(torch.empty(j).uniform_(-1, 1, generator=torch.Generator().manual_seed(r)))
    _check(base, x, a, b, _index(kind, lead, j), scale, d_out)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_without_a_base_and_with_a_number_for_a_scale(dtype):
    _, x, a, b, d_out = _inputs((3, 40), 50, 70, 6, 4, dtype, seed=2)
    _check(None, x, a, b, torch.tensor([2, -1, 0]), 0.75, d_out)


def test_values_that_name_no_adapter():
    """Rows of those keep the base's bits and have no gradient, whatever x holds there."""
    base, x, a, b, d_out = _inputs((6, 30), 64, 48, 8, 3, BF16, seed=3)
    for wide in (torch.int32, torch.int64):
        index = torch.tensor([0, -1, 3, 2, -(2**31), 2**31 - 1], dtype=wide)
        bad = x.clone()
        bad[[1, 2, 4, 5]] = float("nan")
        out, grads = _run(base, bad, a, b, index, 1.0, d_out)
        assert torch.equal(out[[1, 2, 4, 5]].cpu(), base[[1, 2, 4, 5]])
        assert (grads["x"][[1, 2, 4, 5]] == 0).all()
        want = ref.low_rank_adapters(base, x, a, b, index, 1.0, d_out)
        for name in ("a", "b"):
            _close(name, grads[name], want[name], want[name + "_error"])
        assert (grads["a"][1] == 0).all() and (grads["b"][1] == 0).all()
    index = torch.tensor([2**32, -(2**32), 2**32 + 1, 2**40, 3, -1])  # whose low halves would name one
    out, grads = _run(base, x, a, b, index, 1.0, d_out)
    assert torch.equal(out.cpu(), base) and all((grads[n] == 0).all() for n in ("x", "a", "b"))


def test_gradients_against_differences():
    """Directional differences of the float64 forward, and the kernel's gradients: second-order terms vanish (each input enters
    linearly), so the two agree to the gradient's own error."""
    base, x, a, b, d_out = _inputs((4, 25), 48, 40, 8, 3, BF16, seed=4)
    index = torch.tensor([2, 0, 2, -1])
    _, grads = _run(base, x, a, b, index, 0.5, d_out)
    want = ref.low_rank_adapters(base, x, a, b, index, 0.5, d_out)
    g = torch.Generator().manual_seed(5)

    def value(x, a, b):
        return (ref.low_rank_adapters(base, x, a, b, index, 0.5)["out"] * d_out.double()).sum()

    for i, name in enumerate(("x", "a", "b")):
        at = [t.double() for t in (x, a, b)]
        v = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        plus, minus = ([t + s * v if k == i else t for k, t in enumerate(at)] for s in (0.5, -0.5))
        difference = value(*plus) - value(*minus)
        bound = ((want[name + "_error"] + HALF_STEP[BF16] * want[name].abs() * 1.01) * v.abs()).sum()
        assert (grads[name].double().cpu() * v).sum().sub(difference).abs() <= bound, name


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("width", [(64, 256), (200, 520)])
def test_small_and_large_values(width, dtype):
    """Gradients of 1e-6 and activations of 1e3: FP16 holds neither x A^T nor d_out B as they are."""
    k, n = width
    for d, up in ((1e-6, 1.0), (1.0, 1e3)):
        base, x, a, b, d_out = _inputs((2, 300), k, n, 8, 3, dtype, seed=6, d=d)
        x = (x.float() * up).to(dtype)
        a = (a.float() * (30.0 if up > 1 else 1.0)).to(dtype)
        b = (b.float() * (1e-3 if up > 1 else 1.0)).to(dtype)
        _check(base, x, a, b, torch.tensor([1, 2]), 1.0, d_out)


@pytest.mark.parametrize("kind", ["image", "row"])
def test_infinite_and_nan_rows_stay_alone(kind):
    base, x, a, b, _ = _inputs((6, 40), 64, 96, 8, 3, BF16, seed=7)
    index = _index(kind, (6, 40), 3, seed=7)
    want = _run(base, x, a, b, index, 1.0)[0]
    bad = x.clone()
    bad[2, 5, 3], bad[4, 39, 60], bad[0, 0, 0] = math.nan, math.inf, -math.inf
    got = _run(base, bad, a, b, index, 1.0)[0]
    rows = torch.ones(6, 40, dtype=torch.bool)
    rows[2, 5] = rows[4, 39] = rows[0, 0] = False
    assert torch.equal(got.cpu()[rows], want.cpu()[rows])
    for at in ((2, 5), (4, 39), (0, 0)):
        j = index[at] if kind == "row" else index[at[0]]
        if j >= 0:
            exact = base[at].double() + (bad[at].double() @ a[j].double().t()) @ b[j].double().t()
            assert torch.equal(torch.isfinite(got[at].cpu()), torch.isfinite(exact))


def test_layouts():
    """Rows apart in memory, leading dimensions that do not merge, expanded bases and gradients, transposed adapters."""
    base, x, a, b, d_out = _inputs((3, 30), 64, 96, 8, 4, BF16, seed=8)
    index = torch.tensor([3, 1, 0])
    want, want_grads = _run(base, x, a, b, index, 0.5, d_out)

    def apart(t):
        return torch.cat([t, t + 1], -1)[..., :t.shape[-1]]

    def turned(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    for view in (apart, turned, lambda t: torch.cat([t[..., :1], t], -1)[..., 1:]):
        dev = [view(t.to(DEV)) for t in (base, x, a, b)]
        leaves = [t.detach().requires_grad_() for t in dev]
        out = ops.low_rank_adapters(*leaves, index.to(DEV), scale=0.5)
        assert torch.equal(out, want)
        for g, name in zip(torch.autograd.grad(out, leaves, view(d_out.to(DEV))), ("base", "x", "a", "b")):
            assert torch.equal(g, want_grads[name]), name
    one = base[:1, :1].to(DEV)
    expanded = ops.low_rank_adapters(one.expand(3, 30, 96), x.to(DEV), a.to(DEV), b.to(DEV), index.to(DEV), scale=0.5)
    assert torch.equal(expanded, ops.low_rank_adapters(one.expand(3, 30, 96).contiguous(), x.to(DEV), a.to(DEV), b.to(DEV),
                                                       index.to(DEV), scale=0.5))
    leaf = one.clone().requires_grad_()
    out = ops.low_rank_adapters(leaf.expand(3, 30, 96), x.to(DEV), a.to(DEV), b.to(DEV), index.to(DEV), scale=0.5)
    torch.testing.assert_close(torch.autograd.grad(out, leaf, torch.ones_like(out))[0], torch.full_like(leaf, 90.0))


@pytest.mark.parametrize("wanted", ["x", "a", "b", "base", "xa", "ab"])
@pytest.mark.parametrize("width", [(64, 96), (300, 260)])
def test_gradients_wanted_alone(width, wanted):
    k, n = width
    base, x, a, b, d_out = _inputs((2, 350), k, n, 8, 3, BF16, seed=9)
    index = torch.tensor([1, 2], device=DEV)
    names = ["base", "x", "a", "b"]
    every = dict(zip(names, (t.to(DEV) for t in (base, x, a, b))))
    whole = {m: t.clone().requires_grad_() for m, t in every.items()}
    want = dict(zip(names, torch.autograd.grad(ops.low_rank_adapters(*whole.values(), index), list(whole.values()), d_out.to(DEV))))
    chosen = ["base"] if wanted == "base" else list(wanted)
    some = {m: t.clone().requires_grad_(m in chosen) for m, t in every.items()}
    got = torch.autograd.grad(ops.low_rank_adapters(*some.values(), index), [some[m] for m in chosen], d_out.to(DEV))
    assert all(torch.equal(g, want[m]) for g, m in zip(got, chosen))


def test_no_rows():
    base, x, a, b, _ = (t.to(DEV) for t in _inputs((0, 5), 16, 24, 4, 3, BF16))
    leaves = [t.requires_grad_() for t in (base, x, a, b)]
    out = ops.low_rank_adapters(*leaves, torch.zeros(0, dtype=torch.int64, device=DEV))
    assert out.shape == (0, 5, 24)
    grads = torch.autograd.grad(out, leaves, torch.zeros_like(out))
    assert all((g == 0).all() and g.shape == t.shape for g, t in zip(grads, leaves))


def test_rows_past_32_bit_offsets():
    """600 rows 2^22 elements apart (5 GB): forward and both forms of the backward pass."""
    for k, n in ((64, 96), (200, 520)):
        base, x, a, b, d_out = _inputs((600,), k, n, 8, 3, BF16, seed=10)
        index = torch.arange(600) % 4 - 1
        memory = torch.empty(600, 1 << 22, dtype=BF16, device=DEV)
        far = memory[:, 5:5 + k]
        far.copy_(x)
        memory[:, 5000:5000 + n].copy_(base)
        memory[:, 10000:10000 + n].copy_(d_out)
        want, want_grads = _run(base, x, a, b, index, 1.0, d_out)
        leaves = [t.to(DEV).requires_grad_() for t in (a, b)]
        x_leaf = far.detach().requires_grad_()
        out = ops.low_rank_adapters(memory[:, 5000:5000 + n], x_leaf, *leaves, index.to(DEV))
        assert torch.equal(out, want)
        d = memory[:, 10000:10000 + n]
        for g, name in zip(torch.autograd.grad(out, [x_leaf, *leaves], d), ("x", "a", "b")):
            assert torch.equal(g, want_grads[name]), name
        del memory, far, x_leaf, d, out


def test_more_adapters_than_rows_and_many_chunks():
    base, x, a, b, d_out = _inputs((40,), 96, 64, 4, 300, BF16, seed=11)
    _check(base, x, a, b, torch.randint(0, 300, (40,), generator=torch.Generator().manual_seed(0)), 1.0, d_out)
    base, x, a, b, d_out = _inputs((9000,), 40, 500, 4, 2, BF16, seed=12)
    _check(base, x, a, b, (torch.arange(9000) // 5000), 1.0, d_out)


@pytest.mark.parametrize("size", [((2, 20000), 96, 160, 24, 400), ((20000,), 300, 340, 100, 400)])
def test_chunks_of_several_lists(size):
    """So many adapters that the partial sums of all take few, long chunks: their rows are listed in pieces."""
    lead, k, n, r, j = size
    base, x, a, b, d_out = _inputs(lead, k, n, r, j, BF16, seed=21)
    index = _index("row", lead, j, seed=22)
    index[..., : lead[-1] // 3] = 7  # one adapter's rows fill lists
    _check(base, x, a, b, index, 0.5, d_out)


@pytest.mark.parametrize("width", [(64, 256), (200, 520)])
def test_rows_of_different_magnitude_in_fp16(width):
    """A row's dx keeps its precision beside rows of 2^20 times its gradient."""
    k, n = width
    base, x, a, b, d_out = _inputs((300,), k, n, 8, 2, F16, seed=23)
    d_out = (d_out.double() * 2.0 ** (-20 * (torch.arange(300) % 3 == 0).double())[:, None] * 16).to(F16)
    _check(base, x, (a * 64).to(F16), b, _index("row", (300,), 2, seed=24), 1.0, d_out)


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_an_infinite_row_leaves_the_others_their_precision(bad):
    """FP16 gradients of 1e-6 beside one that is not finite."""
    base, x, a, b, d_out = _inputs((200,), 64, 256, 8, 1, F16, seed=25, d=1e-6)
    index, a = torch.tensor(0), (a * 64).to(F16)
    d_out[77, 3] = bad
    _, grads = _run(base, x, a, b, index, 1.0, d_out)
    keep = torch.arange(200) != 77
    want = ref.low_rank_adapters(base[keep], x[keep], a, b, index, 1.0, d_out[keep])
    _close("x", grads["x"][keep.to(DEV)], want["x"], want["x_error"])
    assert not torch.isfinite(grads["x"][77]).any()


def test_same_bits_on_any_stream():
    base, x, a, b, d_out = _inputs((3, 3000), 64, 256, 8, 3, BF16, seed=13)
    index = torch.tensor([0, 2, 0])
    want, want_grads = _run(base, x, a, b, index, 1.0, d_out)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out, grads = _run(base, x, a, b, index, 1.0, d_out)
        side.synchronize()
        assert torch.equal(out, want) and all(torch.equal(grads[m], want_grads[m]) for m in grads)


@pytest.mark.parametrize("width", [(64, 256), (300, 260)])
def test_graph_capture(width):
    k, n = width
    base, x, a, b, d_out = (t.to(DEV) for t in _inputs((3, 500), k, n, 8, 4, BF16, seed=14))
    index = torch.tensor([0, 3, -1], device=DEV)
    leaves = [t.requires_grad_() for t in (base, x, a, b)]

    def both():
        out = ops.low_rank_adapters(*leaves, index, scale=0.5)
        return out.detach(), *torch.autograd.grad(out, leaves, d_out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    for seed in range(3):
        with torch.no_grad():
            leaves[1].copy_(_inputs((3, 500), k, n, 8, 4, BF16, seed=20 + seed)[1])
            index.copy_(torch.tensor([seed, -1, 3 - seed]))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(c, e) for c, e in zip(captured, both()))


def test_refusals():
    base, x, a, b, _ = (t.to(DEV) for t in _inputs((2, 10), 64, 48, 8, 3, BF16))
    index = torch.tensor([0, 1], device=DEV)
    wide = torch.zeros(3, 129, 64, device=DEV, dtype=BF16), torch.zeros(3, 48, 129, device=DEV, dtype=BF16)
    bad = [(base.float(), x.float(), a.float(), b.float(), index), (base, x, a.to(F16), b, index), (base.to(F16), x, a, b, index),
           (base[..., :40], x, a, b, index), (base, x, a[:, :, :32], b, index), (base, x, a[:2], b, index), (base, x, a, b[..., :4], index),
           (base, x, a, b, index[:1]), (base, x, a, b, index.float()), (base, x, a, b, index.cpu()), (base, x, a, b, index[:, None]),
           (base, x, a[0], b[0], index), (base, x, *wide, index), (base, x, a[:0], b[:0], index), (base, x.cpu(), a, b, index),
           (base, x, a, b, torch.zeros(2, 10, 64, dtype=torch.int32, device=DEV))]
    for args in bad:
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.low_rank_adapters(*args)
    for scale in (torch.ones(2, device=DEV), torch.ones(3, device=DEV, dtype=BF16), torch.ones(3)):
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.low_rank_adapters(base, x, a, b, index, scale=scale)
    with pytest.raises((TypeError, ValueError)):
        torch.ops.flashim_amd.low_rank_adapters(base, x, a.to(F16), b, index, None, 1.0, False)
    with pytest.raises(ValueError):
        torch.ops.flashim_amd.low_rank_adapters(base, x, a, b, index[:1], None, 1.0, False)
    with pytest.raises(NotImplementedError, match="scales"):
        ops.low_rank_adapters(base, x, a, b, index, scale=torch.ones(3, device=DEV, requires_grad=True))
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(ops.low_rank_adapters(base, leaf, a, b, index).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        g.sum().backward()


def _positive(lead, k, n, r, j, dtype, seed):
    """Inputs above zero, so that an infinity meets no other of its sign's opposite: what it reaches is +infinity."""
    base, x, a, b, d_out = ((t.float().abs() + 0.125).to(dtype) for t in _inputs(lead, k, n, r, j, dtype, seed=seed))
    return base, x, a, b, d_out / 16  # (sums within FP16)


def _infinite_as_defined(bad, width, r, dtype, names, lead=(70,)):
    """An infinity in one operand, and the named results against float64's: infinities, NaN and finite values where it has them."""
    k, n = width
    base, x, a, b, d_out = _positive(lead, k, n, r, 3, dtype, seed=26)
    {"x": x, "d": d_out, "a": a[1], "b": b[1]}[bad].view(-1)[5 % min(k, n)] = math.inf
    index = torch.arange(lead[0]) % 3
    index[0] = 1 if bad in "ab" else index[0]
    out, grads = _run(base, x, a, b, index, 0.5, d_out)
    want = ref.low_rank_adapters(base, x, a, b, index, 0.5, d_out)
    for name, got in {"out": out, **grads}.items():
        if name in names:
            w, g = want[name], got.double().cpu()
            assert torch.equal(torch.isposinf(g), torch.isposinf(w)) and torch.equal(torch.isnan(g), torch.isnan(w)), (name, bad)
            assert not torch.isneginf(g).any()
            at = torch.isfinite(w) & torch.isfinite(want[name + "_error"])
            _close(name, got.cpu()[at], w[at], want[name + "_error"][at])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("r", [1, 5, 8, 24])
@pytest.mark.parametrize("bad, names", [("d", ("x", "a")), ("a", ("b",)), ("b", ("a",))])
def test_infinities_beside_padding(bad, names, r, dtype):
    """Ranks past R and rows past a turn's last are no part of the narrow backward pass: infinities there are the definition's."""
    _infinite_as_defined(bad, (64, 96), r, dtype, names)
    _infinite_as_defined(bad, (41, 50), r, dtype, names)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("width, r", [((64, 96), 1), ((64, 96), 8), ((41, 50), 5), ((64, 96), 24), ((200, 520), 5), ((200, 520), 8),
                                      ((200, 520), 24), ((200, 523), 40), ((96, 200), 100)])
@pytest.mark.parametrize("bad", ["x", "d", "a", "b"])
def test_infinities_meet_both_halves(bad, width, r, dtype):
    """h and t go into products as two numbers of 16 bits, whose second may be zero or negative: an infinity on the other side
    stays the one that it makes with the first."""
    for lead in ((70,), (600,), (9, 40)):
        _infinite_as_defined(bad, width, r, dtype, ("out", "x", "a", "b"), lead)


@pytest.mark.parametrize("wanted", ["x", "a"])
def test_what_the_backward_pass_cannot_hold_is_refused_by_the_forward_pass(wanted):
    """Adapters of 2^32 elements and more (their transposes' launch): served, but not trained or trained through."""
    from flashim_amd._lib import UnsupportedShape

    j, r, k, n = 1024, 128, 32768 - 32, 64
    a, b = torch.empty(j, r, k, dtype=BF16, device=DEV), torch.zeros(j, n, r, dtype=BF16, device=DEV)
    x, index = torch.zeros(3, k, dtype=BF16, device=DEV), torch.tensor([5, -1, 1023], device=DEV)
    a[[5, 1023]] = 1.0
    assert (ops.low_rank_adapters(None, x, a, b, index) == 0).all()
    (x if wanted == "x" else a).requires_grad_()
    with pytest.raises(UnsupportedShape, match="backward"):
        ops.low_rank_adapters(None, x, a, b, index)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("size", [((2100,), 200, 523, 24, 3), ((2100,), 200, 523, 100, 3), ((17000,), 72, 520, 40, 3),
                                  ((17000,), 196, 300, 64, 5), ((33000,), 64, 256, 8, 4), ((33000,), 41, 50, 5, 4),
                                  ((33000,), 64, 100, 24, 3), ((33000,), 64, 100, 40, 3), ((33000,), 72, 100, 100, 3),
                                  ((33000,), 130, 520, 12, 3)])
def test_every_form_of_the_tiles(size, dtype):
    """Two sets of 16 rows at any rank, and a wavefront a tile, on the other side of the rows they begin at (8, 64 and 128 a CU)."""
    lead, k, n, r, j = size
    base, x, a, b, d_out = _inputs(lead, k, n, r, j, dtype, seed=27, d=0.125)
    _check(base, x, a, b, _index("runs", lead, j, seed=28), 0.5, d_out)
