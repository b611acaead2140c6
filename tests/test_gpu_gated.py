"""``ops.gated_linear`` against its definition in float64 (``oracle/train.py``), forward and gradients.

Bounds, with ``u`` half a unit of the type's last place (2^-8, 2^-11): an FP32 sum of n exact products is within
n 2^-24 of its terms' magnitudes at worst, and 2^-18 of them covers every length here; an output is that, through the
activation (slope below 1.13), rounded once. The backward pass rounds each pre-activation's gradient to 16 bits before the
next product: independent errors of at most u of a term, so a sum of them stays within 6 u / sqrt(3) of the root of its
terms' squares (six standard deviations), beside the FP32 sum and the final rounding. Bias gradients are sums of unrounded
values."""

import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

from flashim_amd import _lib, ops
from oracle import train as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ACTS = {"none": lambda z: z, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh")}
U = {BF16: 2.0**-8, F16: 2.0**-11, F32: 2.0**-24}
TINY = {BF16: 1e-38, F16: 2.0**-25, F32: 1e-38}
SUM = 2.0**-18


def _inputs(m, k, h, dtype, bias=None, seed=0, strong=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    wg, wu = ((torch.randn(h, k, generator=g) * strong * k**-0.5).to(dtype) for _ in range(2))
    bg, bu = ((0.5 * torch.randn(h, generator=g)).to(bias) if bias is not None else None for _ in range(2))
    return x, wg, wu, bg, bu, (0.25 * torch.randn(m, h, generator=g)).to(dtype)


def _dev(*tensors):
    return [None if t is None else t.to(DEV) for t in tensors]


def _check(what, got, want, bound):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = (got.double().cpu() - want).abs() - bound
    assert not (over > 0).any(), f"{what}: {int((over > 0).sum())} of {over.numel()} off, by up to {over.max().item():.3g}"
    assert torch.isfinite(got).all(), what


def _forward(x, wg, wu, bg, bu, act):
    out = ops.gated_linear(*_dev(x, wg, wu, bg, bu), activation=act)
    assert out.dtype == x.dtype
    want, reach = ref.gated_linear(x, wg, wu, bg, bu, act)
    _check("out", out, want, U[x.dtype] * want.abs() + SUM * (reach + want.abs()) + TINY[x.dtype])


def _backward(x, wg, wu, bg, bu, act, d_out):
    names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    leaves = [None if t is None else t.requires_grad_() for t in _dev(x, wg, wu, bg, bu)]
    wanted = [(n, t) for n, t in zip(names, leaves) if t is not None]
    grads = torch.autograd.grad(ops.gated_linear(*leaves, activation=act), [t for _, t in wanted], d_out.to(DEV))
    want = ref.gated_linear_gradients(d_out, x, wg, wu, bg, bu, act)
    # the pre-activations' own errors: SUM of their terms, which are a few times their deviation in these inputs
    pre = SUM * (4 * x.shape[1] ** 0.5 + 4)
    for (name, leaf), got in zip(wanted, grads):
        assert got.dtype == leaf.dtype, name
        bound = U[leaf.dtype] * want[name].abs() + (SUM + pre) * want[name + "_terms"] + TINY[leaf.dtype]
        if name + "_squares" in want:
            u = U[x.dtype]
            scale = {"x": wg.double().abs().amax(), "w_gate": x.double().abs().amax(), "w_up": x.double().abs().amax()}[name]
            n = x.shape[0] if name != "x" else 2 * wg.shape[0]
            bound = bound + 6 / math.sqrt(3) * (u * want[name + "_squares"] + TINY[x.dtype] * scale * n**0.5)
        _check(name, got, want[name], bound)


FEW, ROWS, TILES = range(3)  # forms of the forward pass


def plan(m, k, h):
    """Form of the forward pass, blocks of its tile, backward in one pass, blocks of dx's tile, its splits, blocks of the
    weights' tile, its splits."""
    out = (ctypes.c_int * 7)()
    _lib.probe_call("fim_test_gated_plan", m, k, h, ctypes.addressof(out))
    return tuple(out)


SHAPES = [  # rows, channels, hidden: single values, one row, odd and prime sizes, tile edges, several tiles each way
    (1, 1, 1), (1, 64, 256), (2, 8, 8), (3, 7, 5), (16, 512, 2048), (17, 196, 523), (64, 64, 64), (65, 72, 130),
    (100, 33, 257), (127, 128, 129), (128, 64, 128), (129, 1000, 40), (300, 320, 853), (257, 264, 264), (1000, 16, 24),
    (513, 520, 1032), (2049, 96, 192), (33, 2056, 72),
]


@pytest.mark.parametrize("m,k,h", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_forward_and_gradients(m, k, h, dtype):
    act = ("silu", "gelu", "gelu_tanh")[(m + k + h) % 3]
    x, wg, wu, bg, bu, d_out = _inputs(m, k, h, dtype, bias=(None, F32, dtype)[(m + h) % 3], seed=m + k + h)
    _forward(x, wg, wu, bg, bu, act)
    _backward(x, wg, wu, bg, bu, act, d_out)


NARROW = [  # backward in one pass: channels up to 64, hidden up to 256; one or two row blocks a step, steps past the last row
    (1, 64, 256), (31, 64, 256), (32, 63, 255), (33, 64, 128), (63, 8, 129), (64, 64, 160), (65, 57, 31), (127, 64, 256),
    (1000, 64, 96), (4097, 24, 200), (9000, 40, 128), (20011, 64, 256), (8191, 64, 64), (8300, 5, 33),
]


@pytest.mark.parametrize("m,k,h", NARROW)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_narrow_layers(m, k, h, dtype):
    act = ("silu", "gelu", "gelu_tanh")[(m + k + h) % 3]
    x, wg, wu, bg, bu, d_out = _inputs(m, k, h, dtype, bias=(None, F32, dtype)[(m + h) % 3], seed=m + k + h)
    _forward(x, wg, wu, bg, bu, act)
    _backward(x, wg, wu, bg, bu, act, d_out)


@pytest.mark.parametrize("m,k,h", [(500, 64, 256), (500, 40, 100), (500, 72, 300)])
@pytest.mark.parametrize("wanted", [(0,), (1, 2), (3, 4), (0, 3), (2,)])
def test_wanted_gradients_alone_are_those_of_all(m, k, h, wanted):
    tensors = [t.to(DEV) for t in _inputs(m, k, h, BF16, bias=F32, seed=9)]
    d_out = tensors.pop()

    def grads(which):
        leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate(tensors)]
        return torch.autograd.grad(ops.gated_linear(*leaves), [leaves[i] for i in which], d_out)

    every = grads(range(5))
    for i, got in zip(wanted, grads(wanted)):
        assert torch.equal(got, every[i])


LONG = [  # many rows of few channels: a last block of one row, odd widths, several hidden blocks, channels up to 128
    (32800, 64, 256), (32769, 33, 77), (33333, 8, 256), (40001, 40, 104), (36000, 64, 264), (33000, 100, 300),
    (32768, 128, 136), (35001, 127, 131),
]


@pytest.mark.parametrize("m,k,h", LONG)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_many_rows_of_few_channels(m, k, h, dtype):
    act = ("silu", "gelu", "gelu_tanh")[(m + k + h) % 3]
    x, wg, wu, bg, bu, d_out = _inputs(m, k, h, dtype, bias=(None, F32, dtype)[(m + h) % 3], seed=m + k + h)
    _forward(x, wg, wu, bg, bu, act)
    _backward(x, wg, wu, bg, bu, act, d_out)


ROWS_SHAPES = [  # the forward pass by rows: a last block of one row, odd widths, hidden blocks that end inside, few rows of many
    (40001, 64, 256), (40003, 33, 77), (41000, 8, 255), (20100, 40, 520), (8300, 64, 1240), (160001, 100, 60), (80100, 128, 264),
    (9100, 127, 2300),
]


@pytest.mark.parametrize("m,k,h", ROWS_SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_forward_by_rows(m, k, h, dtype):
    assert plan(m, k, h)[0] == ROWS
    x, wg, wu, bg, bu, _ = _inputs(m, k, h, dtype, bias=(None, F32, dtype)[(m + h) % 3], seed=m + k + h)
    _forward(x, wg, wu, bg, bu, ("silu", "gelu", "gelu_tanh")[(m + k + h) % 3])


LARGE_TILES = {  # 256 x 256 tiles, by what takes them (the plan's fields): odd sizes and sizes of whole 16-byte rows
    (3001, 1031, 2053): {1: 4, 5: 4, 6: 3},        # forward; weights in three splits
    (3000, 776, 2056): {1: 4},
    (4101, 1031, 2051): {3: 4, 4: 3, 5: 4, 6: 3},  # dx and weights in three splits
    (4100, 1032, 2056): {3: 4, 4: 3, 5: 4, 6: 3},
    (8201, 1541, 523): {3: 4, 4: 1},               # dx whole
    (8200, 1544, 520): {3: 4, 4: 1},
}


@pytest.mark.parametrize("m,k,h", LARGE_TILES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_tiles(m, k, h, dtype):
    chosen = plan(m, k, h)
    assert chosen[0] == TILES and all(chosen[i] == v for i, v in LARGE_TILES[m, k, h].items())
    act = ("silu", "gelu", "gelu_tanh")[(m + k + h) % 3]
    x, wg, wu, bg, bu, d_out = _inputs(m, k, h, dtype, bias=(None, F32, dtype)[(m + h) % 3], seed=m + k + h)
    _forward(x, wg, wu, bg, bu, act)
    _backward(x, wg, wu, bg, bu, act, d_out)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_large_tiles_of_every_activation(act):
    x, wg, wu, bg, bu, _ = _inputs(3001, 777, 2053, BF16, bias=BF16, seed=17)
    assert plan(3001, 777, 2053)[1] == 4
    _forward(x, wg, wu, bg, bu, act)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("bias", [None, "gate", "up", BF16, F32])
@pytest.mark.parametrize("m", [5, 200])
def test_activations_and_biases(act, bias, m):
    x, wg, wu, bg, bu, d_out = _inputs(m, 72, 136, BF16, bias=F32 if isinstance(bias, str) else bias, seed=1)
    bg, bu = None if bias == "up" else bg, None if bias == "gate" else bu
    _forward(x, wg, wu, bg, bu, act)
    if act != "relu":  # (its derivative jumps where the gate is zero up to rounding)
        _backward(x, wg, wu, bg, bu, act, d_out)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_saturated_gates(act):
    """Gates far into both tails of the activation."""
    x, wg, wu, bg, bu, d_out = _inputs(150, 64, 72, BF16, seed=2, strong=30.0)
    _forward(x, wg, wu, bg, bu, act)


@pytest.mark.parametrize("m", [1, 8, 77, 300])
def test_leading_dimensions_and_single_rows_agree(m):
    x, wg, wu, bg, bu, _ = _dev(*_inputs(m * 6, 64, 96, BF16, bias=F32, seed=3))
    flat = ops.gated_linear(x, wg, wu, bg, bu)
    assert torch.equal(ops.gated_linear(x.view(2, 3, m, 64), wg, wu, bg, bu).view(-1, 96), flat)
    one = ops.gated_linear(x[0], wg, wu, bg, bu)
    assert one.shape == (96,)
    want, reach = ref.gated_linear(x[:1].cpu(), *(t.cpu() for t in (wg, wu, bg, bu)), "silu")
    _check("row", one[None], want, U[BF16] * want.abs() + SUM * (reach + want.abs()))


@pytest.mark.parametrize("m", [9, 250])
def test_views(m):
    """Row strides, channel slices at aligned and odd offsets, transposed and broadcast operands: the values of their
    packed copies."""
    x, wg, wu, bg, bu, d_out = _dev(*_inputs(m, 72, 88, BF16, bias=BF16, seed=4))
    g = torch.Generator(device=DEV).manual_seed(0)

    def strided(t, left, right):
        wide = torch.randn(t.shape[0], left + t.shape[1] + right, generator=g, device=DEV).to(t.dtype)
        wide[:, left:left + t.shape[1]] = t
        return wide[:, left:left + t.shape[1]]

    def results(x, wg, wu, d):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        out = ops.gated_linear(*leaves, bg, bu, activation="gelu")
        return [out, *torch.autograd.grad(out, leaves, d)]

    want = results(x, wg, wu, d_out)
    for xs in (strided(x, 0, 8), strided(x, 8, 16), strided(x, 3, 2), strided(x, 1, 0), x.t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(results(xs, wg, wu, d_out), want))
    for ws in (lambda t: strided(t, 16, 0), lambda t: strided(t, 5, 1), lambda t: t.t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(results(x, ws(wg), wu, d_out), want))
        assert all(torch.equal(a, b) for a, b in zip(results(x, wg, ws(wu), d_out), want))
    for ds in (strided(d_out, 8, 0), strided(d_out, 1, 6), d_out.t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(results(x, wg, wu, ds), want))
    rows = x[:1].expand(m, -1)  # a row stride of 0
    assert torch.equal(ops.gated_linear(rows, wg, wu, bg, bu), ops.gated_linear(rows.contiguous(), wg, wu, bg, bu))
    ones = torch.ones((), device=DEV, dtype=BF16).expand(m, 88)
    assert all(torch.equal(a, b) for a, b in zip(results(x, wg, wu, ones), results(x, wg, wu, ones.contiguous())))


def test_gradients_only_where_wanted():
    x, wg, wu, bg, bu, d_out = _dev(*_inputs(130, 64, 96, BF16, bias=F32, seed=5))
    every = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    want = torch.autograd.grad(ops.gated_linear(*every), every, d_out)
    for i in range(5):
        leaves = [t.clone().requires_grad_(k == i) for k, t in enumerate((x, wg, wu, bg, bu))]
        ops.gated_linear(*leaves).backward(d_out)
        assert torch.equal(leaves[i].grad, want[i])
        assert all(t.grad is None for k, t in enumerate(leaves) if k != i)


def test_shared_operands_and_broadcast_inputs():
    """One weight for both projections, and an input that several rows share: gradients add up."""
    x, w, _, b, _, d_out = _dev(*_inputs(96, 64, 80, F16, bias=F32, seed=6))
    leaf, bias, row = w.clone().requires_grad_(), b.clone().requires_grad_(), x[:1].clone().requires_grad_()
    rows = row.expand(96, -1)
    got = torch.autograd.grad(ops.gated_linear(rows, leaf, leaf, bias, bias), (row, leaf, bias), d_out)
    parts = [t.clone().requires_grad_() for t in (rows.detach().contiguous(), w, w, b, b)]
    dx, dwg, dwu, dbg, dbu = torch.autograd.grad(ops.gated_linear(*parts), parts, d_out)
    assert torch.equal(got[1], dwg + dwu) and torch.equal(got[2], dbg + dbu)
    want = dx.double().sum(0, keepdim=True)
    assert ((got[0].double() - want).abs() <= 8 * U[F16] * dx.double().abs().sum(0, keepdim=True)).all()


def test_empty_batch():
    x = torch.empty(0, 64, device=DEV, dtype=BF16, requires_grad=True)
    w = torch.randn(48, 64, device=DEV).to(BF16).requires_grad_()
    out = ops.gated_linear(x, w, w)
    assert out.shape == (0, 48)
    dx, dw = torch.autograd.grad(out, (x, w), torch.empty_like(out))
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("m", [12, 200])
def test_nonfinite_rows_stay_in_their_row(m):
    x, wg, wu, bg, bu, d_out = _dev(*_inputs(m, 72, 88, BF16, bias=F32, seed=7))
    clean = ops.gated_linear(x, wg, wu, bg, bu)
    broken = x.clone()
    broken[5, 3] = math.nan
    leaf = broken.requires_grad_()
    out = ops.gated_linear(leaf, wg, wu, bg, bu)
    keep = torch.arange(m, device=DEV) != 5
    assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[5]).all()
    (dx,) = torch.autograd.grad(out, leaf, d_out)
    assert torch.isfinite(dx[keep]).all() and torch.isnan(dx[5]).all()


@pytest.mark.parametrize("k,h", [(64, 96), (72, 87)])  # backward in one pass, on tiles
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_nan_biases_reach_their_gradients(act, k, h):
    """A NaN in one gate's bias: NaN where autograd of the same formulas has it, ReLU's slope of 1 there included."""
    x, wg, wu, bg, bu, d_out = _inputs(70, k, h, F16, bias=F32, seed=15)
    bg[11] = math.nan
    leaves = [t.double().requires_grad_() for t in (x, wg, wu, bg, bu)]
    want = torch.autograd.grad(ACTS[act](F.linear(leaves[0], leaves[1], leaves[3])) * F.linear(leaves[0], leaves[2], leaves[4]),
                               leaves, d_out.double())
    leaves = [t.requires_grad_() for t in _dev(x, wg, wu, bg, bu)]
    got = torch.autograd.grad(ops.gated_linear(*leaves, activation=act), leaves, d_out.to(DEV))
    for name, t, v in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), got, want):
        assert torch.equal(t.isnan().cpu(), v.isnan()), name
    # sums of 70 terms of about 0.25, each good to 2^-13 (the bound of _backward)
    torch.testing.assert_close(got[3].double().cpu(), want[3], rtol=2e-3, atol=1e-2, equal_nan=True)


@pytest.mark.parametrize("k,h", [(64, 129), (72, 87), (200, 523)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_an_infinite_bias_of_the_last_column(k, h, dtype):
    """dx is infinite with its sign, as the definition has it: the columns that pad the hidden width have no bias."""
    x, wg, wu, bg, bu, d_out = _inputs(70, k, h, dtype, bias=F32, seed=16)
    bu[-1] = math.inf
    want = ref.gated_linear_gradients(d_out, x, wg, wu, bg, bu, "silu")["x"]
    leaves = [t.requires_grad_() for t in _dev(x, wg, wu, bg, bu)]
    (dx,) = torch.autograd.grad(ops.gated_linear(*leaves), leaves[:1], d_out.to(DEV))
    sure = want.isinf()
    assert sure.float().mean() > 0.9 and torch.equal(dx.double().cpu()[sure], want[sure])


def test_nonfinite_values_beside_a_view_are_not_read_into_it():
    """The memory between a view's rows, and past its last one, holds NaN."""
    for k, h in ((72, 88), (71, 87)):
        x, wg, wu, _, _, d_out = _dev(*_inputs(100, k, h, BF16, seed=8))

        def framed(t):
            wide = torch.full((t.shape[0] + 3, t.shape[1] + 9), math.nan, dtype=t.dtype, device=DEV)
            wide[:t.shape[0], :t.shape[1]] = t
            return wide[:t.shape[0], :t.shape[1]]

        leaves = [framed(t).requires_grad_() for t in (x, wg, wu)]
        out = ops.gated_linear(*leaves)
        packed = [t.clone().requires_grad_() for t in (x, wg, wu)]
        want = ops.gated_linear(*packed)
        assert torch.equal(out, want)
        for a, b in zip(torch.autograd.grad(out, leaves, framed(d_out)), torch.autograd.grad(want, packed, d_out)):
            assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """Rows of x, and of the incoming gradient, more than 2^31 elements apart."""
    far = 2**31 // 2 + 64
    memory = torch.empty(2 * far + 4096, dtype=BF16, device=DEV)
    x, wg, wu, bg, bu, d_out = _dev(*_inputs(3, 64, 96, BF16, seed=9))
    xs = torch.as_strided(memory, (3, 64), (far, 1))
    ds = torch.as_strided(memory, (3, 96), (far, 1), 1024)
    xs.copy_(x)
    ds.copy_(d_out)
    leaves = [t.detach().requires_grad_() for t in (xs, wg, wu)]
    out = ops.gated_linear(*leaves)
    packed = [t.detach().requires_grad_() for t in (x, wg, wu)]
    want = ops.gated_linear(*packed)
    assert torch.equal(out, want)
    for a, b in zip(torch.autograd.grad(out, leaves, ds), torch.autograd.grad(want, packed, d_out)):
        assert torch.equal(a, b)


def test_many_rows():
    """More rows than one 32-bit product of rows and padded hidden width holds at 2 bytes; spot rows against float64."""
    m, k, h = 2**23 + 77, 16, 136
    g = torch.Generator(device=DEV).manual_seed(10)
    x = torch.randn(m, k, generator=g, device=DEV).to(BF16).requires_grad_()
    wg, wu = ((torch.randn(h, k, generator=g, device=DEV) * 0.25).to(BF16) for _ in range(2))
    d_out = torch.randn(m, h, generator=g, device=DEV, dtype=BF16)
    out = ops.gated_linear(x, wg, wu)
    (dx,) = torch.autograd.grad(out, x, d_out)
    rows = torch.tensor([0, 1, 4096, 2**22 + 5, 2**23 - 1, 2**23, m - 2, m - 1])
    xr, dr, w1, w2 = x.detach()[rows.to(DEV)].cpu(), d_out[rows.to(DEV)].cpu(), wg.cpu(), wu.cpu()
    want, reach = ref.gated_linear(xr, w1, w2, None, None, "silu")
    _check("out", out[rows.to(DEV)], want, U[BF16] * want.abs() + SUM * (reach + want.abs()))
    grads = ref.gated_linear_gradients(dr, xr, w1, w2, None, None, "silu")
    _check("dx", dx[rows.to(DEV)], grads["x"], U[BF16] * grads["x"].abs() + 32 * SUM * grads["x_terms"]
           + 6 / math.sqrt(3) * U[BF16] * grads["x_squares"])


def test_many_rows_on_tiles():
    """Backward on tiles with dg and du of more than 4 GB each: spot rows of dx, and the gradients over all rows against
    float64 on the GPU, in parts."""
    m, k, h, part = 5_700_001, 72, 264, 300_000
    assert not plan(m, k, h)[2] and 2 * m * h > 2**31
    g = torch.Generator(device=DEV).manual_seed(18)
    x = torch.randn(m, k, generator=g, device=DEV, dtype=BF16)
    wg, wu = ((torch.randn(h, k, generator=g, device=DEV) * k**-0.5).to(BF16) for _ in range(2))
    bg, bu = (0.5 * torch.randn(h, generator=g, device=DEV) for _ in range(2))
    d_out = torch.randn(m, h, generator=g, device=DEV, dtype=BF16)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    names = ("x", "w_gate", "w_up", "b_gate", "b_up")
    got = dict(zip(names, torch.autograd.grad(ops.gated_linear(*leaves), leaves, d_out)))
    tensors = [t.detach() for t in leaves]
    pre = SUM * (4 * k**0.5 + 4)
    at = torch.tensor([0, 127, 128, 2**21 + 5, 2**22 - 1, 2**22, 5_592_405, 5_592_406, m - 2, m - 1], device=DEV)
    want = ref.gated_linear_gradients(d_out[at].cpu(), x.detach()[at].cpu(), *(t.cpu() for t in tensors[1:]), "silu")
    _check("dx", got["x"][at], want["x"], U[BF16] * want["x"].abs() + (SUM + pre) * want["x_terms"]
           + 6 / math.sqrt(3) * U[BF16] * want["x_squares"])
    sums = {}
    for i in range(0, m, part):
        r = ref.gated_linear_gradients(d_out[i:i + part], tensors[0][i:i + part], *tensors[1:], "silu")
        for name, v in r.items():
            if name[0] != "x":
                v = v.square() if name.endswith("squares") else v
                sums[name] = v if i == 0 else sums[name] + v
    for name in names[1:]:
        want, terms = sums[name].cpu(), sums[name + "_terms"].cpu()
        bound = U[got[name].dtype] * want.abs() + (SUM + pre) * terms
        if name[0] == "w":
            bound = bound + 6 / math.sqrt(3) * U[BF16] * sums[name + "_squares"].sqrt().cpu()
        _check(name, got[name], want, bound)


def test_same_bits_every_time_and_on_another_stream():
    x, wg, wu, bg, bu, d_out = _dev(*_inputs(3000, 200, 264, BF16, bias=F32, seed=11))
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]

    def both():
        out = ops.gated_linear(*leaves)
        return out.detach(), *torch.autograd.grad(out, leaves, d_out)

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            again = both()
        side.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(first, again))


def test_gradient_against_differences():
    """The float64 definition's central differences along random directions against the kernel's FP16 gradients, which
    are good to 2^-9 of the direction's terms (two roundings of 2^-11, added up at worst)."""
    x, wg, wu, bg, bu, d_out = _inputs(40, 24, 32, F16, bias=F32, seed=12)
    leaves = [t.requires_grad_() for t in _dev(x, wg, wu, bg, bu)]
    grads = torch.autograd.grad(ops.gated_linear(*leaves, activation="gelu"), leaves, d_out.to(DEV))
    base, g, step = [t.double() for t in (x, wg, wu, bg, bu)], torch.Generator().manual_seed(13), 1e-4
    for i in range(5):
        v = torch.randn(base[i].shape, generator=g).double()
        moved = [[t + s * step * v if k == i else t for k, t in enumerate(base)] for s in (1, -1)]
        loss = [(ref.gated_linear(*p, "gelu")[0] * d_out.double()).sum().item() for p in moved]
        slope, dot = (loss[0] - loss[1]) / (2 * step), (grads[i].double().cpu() * v).sum().item()
        assert abs(slope - dot) <= 2.0**-9 * (grads[i].double().cpu() * v).abs().sum().item(), (i, slope, dot)


@pytest.mark.parametrize("m", [4, 700])
def test_graph_capture(m):
    x, wg, wu, bg, bu, d_out = _dev(*_inputs(m, 100, 264, BF16, bias=F32, seed=14))
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]

    def both():
        out = ops.gated_linear(*leaves)
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
            leaves[0].copy_(_inputs(m, 100, 264, BF16, seed=20 + seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(captured, both()))


def test_refusals():
    x, wg, wu, bg, bu, _ = _dev(*_inputs(10, 64, 48, BF16, bias=F32))
    bad = [(x.float(), wg.float(), wu.float()), (x, wg, wu.to(F16)), (x, wg[:, :32], wu), (x, wg, wu[:40]),
           (x, wg, wu, bg[:40]), (x, wg, wu, bg, bu.to(BF16)), (x, wg, wu, bg.to(F16), bu.to(F16)), (x, wg.cpu(), wu)]
    for args in bad:
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.gated_linear(*args)
    with pytest.raises(NotImplementedError, match="no HIP impl"):
        ops.gated_linear(x, wg, wu, activation="softmax")
    with pytest.raises((TypeError, ValueError)):
        torch.ops.flashim_amd.gated_linear(x, wg, wu.to(F16), None, None, 2)
    with pytest.raises(ValueError):
        torch.ops.flashim_amd.gated_linear(x, wg[:, :32], wu[:, :32], None, None, 2)
    with pytest.raises(RuntimeError):
        torch.ops.flashim_amd.gated_linear(x, wg, wu, None, None, 7)
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(ops.gated_linear(leaf, wg, wu).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):
        g.sum().backward()
