"""``ops.group_norm_act`` against its definition in float64 (``oracle/train.py``), forward and gradients.

Bounds, with ``u`` half a unit of the output type's last place (2^-8, 2^-11, 2^-24, relative): an output is the float64
value rounded once, after an FP32 chain. The statistics carry at most 2^-20 of the group's magnitude (sums of a few hundred
FP32 terms, merged), which reaches z as 2^-20 |w| (|x| + |mean|) rstd, and every activation here has a slope below 1.13;
its own FP32 steps stay below 2^-21 (1 + |z|). Gradients are sums: 2^-19 of the sum of their terms' magnitudes on top of
the rounding."""

import math

import pytest
import torch
import torch.nn.functional as F

from flashim_amd import ops
from oracle import train as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0**-25, torch.float32: 1e-38}  # half the smallest step of all
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ACTS = {"none": lambda z: z, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh")}


def _inputs(shape, dtype, param=F32, seed=0, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    c = shape[-1]
    x = (torch.randn(*shape, generator=g) * (torch.rand(c, generator=g) + 0.3) + mean * torch.randn(c, generator=g)).to(dtype)
    w, b = (1 + 0.3 * torch.randn(c, generator=g)).to(param), (0.3 * torch.randn(c, generator=g)).to(param)
    return x, w, b, torch.randn(*shape, generator=g).to(dtype)


def _forward_bound(x, groups, w, b, eps, want):
    xhat, mean, rstd = ref.normalized(x, groups, eps)
    w = torch.ones(x.shape[-1]) if w is None else w
    v = x.double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    reach = ((v.abs() + mean.abs()) * rstd).reshape(x.shape) * w.double().abs()
    z = xhat.abs() * w.double().abs() + (0 if b is None else b.double().abs())
    return U[x.dtype] * want.abs() + 1.13 * 2.0**-20 * reach + 2.0**-21 * (1 + z) + TINY[x.dtype]


def _check(got, want, bound):
    assert got.shape == want.shape
    over = (got.double().cpu() - want).abs() - bound
    assert not (over > 0).any(), f"{int((over > 0).sum())} of {over.numel()} off, by up to {over.max().item():.3g}"
    assert torch.isfinite(got).all()


def _forward(x, groups, w, b, eps, act):
    out = ops.group_norm_act(x.to(DEV), groups, None if w is None else w.to(DEV), None if b is None else b.to(DEV),
                             eps=eps, activation=act)
    assert out.dtype == x.dtype
    want = ref.group_norm_act(x, groups, w, b, eps, act)
    _check(out, want, _forward_bound(x, groups, w, b, eps, want))
    return out


def _backward(x, groups, w, b, eps, act, d_out):
    leaves = [t.to(DEV).requires_grad_() if t is not None else None for t in (x, w, b)]
    out = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], eps=eps, activation=act)
    wanted = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("x", "weight", "bias"), leaves) if t is not None],
                     torch.autograd.grad(out, wanted, d_out.to(DEV))))
    _check_gradients(grads, x, groups, w, b, eps, act, d_out)


def _check_gradients(grads, x, groups, w, b, eps, act, d_out):
    want = ref.group_norm_act_gradients(d_out, x, groups, w, b, eps, act)
    # z's own error moves dz by the activation's second derivative (below 1.2) of it
    xhat, mean, rstd = ref.normalized(x, groups, eps)
    v = x.double().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    ww = torch.ones(x.shape[-1]) if w is None else w
    moved = 2.0**-19 * (1 + ((v.abs() + mean.abs()) * rstd).reshape(x.shape) * ww.double().abs())
    d = d_out.double().abs() * moved
    extra = {"x": (rstd * (d * ww.double().abs()).reshape(v.shape)).reshape(x.shape)
             + 2.0**-19 * (want["x_terms"] + ((v.abs() + mean.abs()) * rstd**2).reshape(x.shape) * d_out.double().abs().mean()),
             "weight": (d * (xhat.abs() + 1)).reshape(-1, x.shape[-1]).sum(0) + 2.0**-19 * want["weight_terms"],
             "bias": d.reshape(-1, x.shape[-1]).sum(0) + 2.0**-19 * want["bias_terms"]}
    for name, got in grads.items():
        leaf = dict(zip(("x", "weight", "bias"), (x, w, b)))[name]
        assert got.dtype == leaf.dtype
        _check(got, want[name], U[leaf.dtype] * want[name].abs() + extra[name] + TINY[leaf.dtype])


SHAPES = [  # (shape, groups): one pixel, one channel a group, one group, odd channel counts, several workgroups an image
    ((1, 1, 64), 8), ((2, 1, 8), 8), ((3, 5, 7, 32), 4), ((1, 33, 35, 64), 32), ((2, 40, 41, 196), 14), ((2, 17, 3), 1),
    ((1, 300, 5), 5), ((4, 64), 4), ((2, 9, 11, 999), 9), ((1, 3, 8192), 16), ((1, 3, 4099), 1), ((5, 130, 128), 32),
    ((1, 121, 61, 512), 32), ((2, 90, 90, 64), 1), ((1, 20, 1028), 4),
]


@pytest.mark.parametrize("shape,groups", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_forward_and_gradients(shape, groups, dtype):
    x, w, b, d_out = _inputs(shape, dtype, seed=len(shape) + groups)
    act = ("silu", "gelu", "gelu_tanh", "none")[shape[-1] % 4]
    _forward(x, groups, w, b, 1e-5, act)
    _backward(x, groups, w, b, 1e-5, act, d_out)


SPLIT = [  # more than a workgroup's registers hold: groups of odd widths, one group, wide maps, a group that crosses loads
    ((2, 70, 71, 12), 3), ((1, 9000, 5), 5), ((1, 5000, 3), 1), ((1, 1300, 999), 9), ((1, 900, 4099), 1), ((1, 330, 8192), 16),
    ((3, 2100, 196), 14), ((1, 130, 131, 64), 32), ((17, 1023, 196), 14),
]


@pytest.mark.parametrize("shape,groups", SPLIT)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_split_maps(shape, groups, dtype):
    x, w, b, d_out = _inputs(shape, dtype, seed=len(shape) + groups)
    act = ("silu", "gelu", "gelu_tanh", "none")[shape[-1] % 4]
    _forward(x, groups, w, b, 1e-5, act)
    _backward(x, groups, w, b, 1e-5, act, d_out)


@pytest.mark.parametrize("param", [BF16, F16, F32])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_activations_and_parameter_types_of_split_maps(act, param):
    x, w, b, _ = _inputs((2, 5003, 48), BF16, param=param, seed=3)
    _forward(x, 6, w, b, 1e-3, act)
    _forward(x, 6, None, b, 1e-3, act)


def test_split_maps_of_a_large_mean_and_of_single_nonfinite_values():
    g = torch.Generator().manual_seed(10)
    x = 100.0 + 0.1 * torch.randn(2, 20000, 32, generator=g)
    _, w, b, _ = _inputs((1, 1, 32), F32)
    _forward(x, 4, w, b, 1e-5, "none")
    x = torch.randn(2, 20000, 32, generator=g)
    clean = ops.group_norm_act(x.to(DEV), 4)
    for bad in (math.nan, math.inf):
        x[1, 19999, 9] = bad  # the second of four groups
        got = ops.group_norm_act(x.to(DEV), 4)
        assert got[1, :, 8:16].isnan().all()
        got[1, :, 8:16] = clean[1, :, 8:16]
        assert torch.equal(got, clean)


@pytest.mark.parametrize("groups", [8, 32])  # the second pass adds up the partials, and a launch of its own does
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
def test_nonfinite_values_anywhere_in_a_thread_s_pixels(act, bad, groups):
    """Ten pixels a thread, of which the first four give the shift: a first one, one past the fourth, in the first, the last
    but one and the last chunk. An infinity leaves no variance, whatever the mean: NaN in the whole group."""
    g = torch.Generator(device=DEV).manual_seed(17)
    x = torch.randn(2, 160000, 64, generator=g, device=DEV).to(BF16)
    w, b = (t.to(DEV) for t in _inputs((1, 1, 64), F32)[1:3])
    d = 64 // groups
    clean = ops.group_norm_act(x, groups, w, b, activation=act)
    for pixel in (0, 3 + 5 * 64, 254 * 625 + 1 + 7 * 64, 159999):
        broken = x.clone()
        broken[1, pixel, 2 * d + 1] = bad
        got = ops.group_norm_act(broken, groups, w, b, activation=act)
        assert got[1, :, 2 * d:3 * d].isnan().all(), pixel
        got[1, :, 2 * d:3 * d] = clean[1, :, 2 * d:3 * d]
        assert torch.equal(got, clean), pixel


@pytest.mark.parametrize("pixels", [40, 20000])  # one launch, two
@pytest.mark.parametrize("act", ["none", "silu"])
def test_a_variance_past_fp32_is_infinite(act, pixels):
    """Deviations of 1e25, whose squares FP32 does not hold: the normalized values are 0 at every map size."""
    x, w, b, _ = (t.to(DEV) for t in _inputs((2, pixels, 32), F32, seed=18))
    clean = ops.group_norm_act(x, 4, w, b, activation=act)
    x[1, :, 8:16] *= 1e25
    got = ops.group_norm_act(x, 4, w, b, activation=act)
    flat = ops.group_norm_act(torch.zeros(1, 1, 32, device=DEV), 4, w, b, activation=act)  # a constant map: act(bias)
    assert torch.equal(got[1, :, 8:16], flat[0, :, 8:16].expand(pixels, 8))
    got[1, :, 8:16] = clean[1, :, 8:16]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("params", ["both", "weight", "bias", "neither"])
def test_activations_and_missing_parameters(act, params):
    x, w, b, d_out = _inputs((2, 23, 19, 48), BF16, param=BF16, seed=3)
    w, b = w if params in ("both", "weight") else None, b if params in ("both", "bias") else None
    _forward(x, 6, w, b, 1e-3, act)
    if act != "relu":  # (its derivative jumps where z is zero up to rounding)
        _backward(x, 6, w, b, 1e-3, act, d_out)


def test_relu_gradient_away_from_its_corner():
    x, w, b, d_out = _inputs((2, 23, 19, 48), F32, seed=4)
    xhat = ref.normalized(x, 6, 1e-5)[0]
    d_out = torch.where((xhat * w + b).abs() > 1e-3, d_out, torch.zeros_like(d_out))
    _backward(x, 6, w, b, 1e-5, "relu", d_out)


@pytest.mark.parametrize("param", [BF16, F16, F32])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_parameter_types(dtype, param):
    x, w, b, d_out = _inputs((2, 31, 64), dtype, param=param, seed=5)
    _forward(x, 8, w, b, 1e-5, "silu")
    _backward(x, 8, w, b.to(F32), 1e-5, "silu", d_out)


def _views():
    """Views of one map: an aligned and an unaligned channel slice, NHWC of NCHW memory, a cropped image, every second
    pixel, a broadcast image."""
    g = torch.Generator().manual_seed(6)
    big = torch.randn(2, 12, 14, 96, generator=g)
    yield "channels 32 to 96", big, lambda t: t[..., 32:]
    yield "channels 3 to 67", big, lambda t: t[..., 3:67]
    yield "nchw memory", big.permute(0, 3, 1, 2).contiguous(), lambda t: t.permute(0, 2, 3, 1)
    yield "crop", big, lambda t: t[:, 1:9, 2:11]
    yield "every second column", big, lambda t: t[:, :, ::2]
    yield "broadcast", big[:1], lambda t: t.expand(3, -1, -1, -1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("name", [v[0] for v in _views()])
def test_views(name, dtype):
    base, view = next((b, f) for n, b, f in _views() if n == name)
    base = base.to(dtype)
    x = view(base)
    c = x.shape[-1]
    _, w, b, _ = _inputs((1, 1, c), dtype, seed=7)
    d_out = torch.randn(x.shape, generator=torch.Generator().manual_seed(8)).to(dtype)
    leaf, wd, bd = base.to(DEV).requires_grad_(), w.to(DEV), b.to(DEV)
    out = ops.group_norm_act(view(leaf), 8, wd, bd, activation="silu")
    want = ref.group_norm_act(x, 8, w, b, 1e-5, "silu")
    _check(out, want, _forward_bound(x, 8, w, b, 1e-5, want))
    out.backward(d_out.to(DEV))
    dense = x.contiguous().to(DEV).requires_grad_()
    ops.group_norm_act(dense, 8, wd, bd, activation="silu").backward(d_out.to(DEV))
    if name != "broadcast":  # in their places (sums in another order where the view's alignment takes other loads)
        _check_gradients({"x": view(leaf.grad)}, x, 8, w, b, 1e-5, "silu", d_out)
    else:
        want = dense.grad.double().sum(0, keepdim=True)
        assert ((leaf.grad.double() - want).abs() <= 3 * U[dtype] * dense.grad.double().abs().sum(0, keepdim=True)).all()


def test_gradient_of_another_layout():
    x, w, b, d_out = _inputs((2, 8, 9, 32), BF16, seed=9)
    leaf = x.to(DEV).requires_grad_()
    out = ops.group_norm_act(leaf, 4, w.to(DEV), b.to(DEV), activation="gelu")
    d = d_out.to(DEV)
    want = torch.autograd.grad(out, leaf, d, retain_graph=True)[0]
    for other in (d.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1), torch.cat([d, d], -1)[..., 32:],
                  torch.cat([d[..., :3], d], -1)[..., 3:]):
        assert torch.equal(torch.autograd.grad(out, leaf, other, retain_graph=True)[0], want)
    (total,) = torch.autograd.grad(out.sum(), leaf)  # a broadcast gradient: stride 0
    assert torch.equal(total, torch.autograd.grad(ops.group_norm_act(leaf, 4, w.to(DEV), b.to(DEV), activation="gelu"),
                                                  leaf, torch.ones_like(d))[0])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_mean(dtype):
    """A mean 1000 times the deviation: sums about zero would leave no digits of the variance in FP32."""
    g = torch.Generator().manual_seed(10)
    x = (100.0 + 0.1 * torch.randn(2, 400, 32, generator=g)).to(dtype)
    _, w, b, _ = _inputs((1, 1, 32), dtype)
    _forward(x, 4, w, b, 1e-5, "none")


def test_constant_groups_and_single_values():
    x = torch.full((2, 6, 16), 3.0, dtype=F32, device=DEV)
    b = torch.randn(16, generator=torch.Generator().manual_seed(0)).to(DEV)
    out = ops.group_norm_act(x, 4, None, b)
    assert torch.equal(out, b.expand_as(out))
    one = torch.randn(3, 1, 8, device=DEV, requires_grad=True)  # one value a group: xhat 0, no gradient
    y = ops.group_norm_act(one, 8)
    assert torch.equal(y, torch.zeros_like(y))
    assert torch.equal(torch.autograd.grad(y, one, torch.randn_like(y))[0], torch.zeros_like(one))


@pytest.mark.parametrize("shape", [(0, 5, 16), (2, 0, 16), (2, 0, 3, 16)])
def test_empty_maps(shape):
    x = torch.empty(shape, device=DEV, requires_grad=True)
    w = torch.randn(16, device=DEV, requires_grad=True)
    out = ops.group_norm_act(x, 4, w, activation="silu")
    assert out.shape == x.shape
    dx, dw = torch.autograd.grad(out, (x, w), torch.empty_like(out))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nonfinite_values_stay_in_their_group(bad):
    x, w, b, d_out = _inputs((2, 40, 32), BF16, seed=11)
    clean = ops.group_norm_act(x.to(DEV), 4, w.to(DEV), b.to(DEV), activation="silu")
    x[1, 7, 9] = bad
    leaf = x.to(DEV).requires_grad_()
    out = ops.group_norm_act(leaf, 4, w.to(DEV), b.to(DEV), activation="silu")
    hit = torch.zeros(2, 40, 4, 8, dtype=torch.bool, device=DEV)
    hit[1, :, 1] = True
    hit = hit.reshape(2, 40, 32)
    assert torch.equal(out[~hit], clean[~hit]) and not torch.isfinite(out[hit]).any()
    (dx,) = torch.autograd.grad(out, leaf, d_out.to(DEV))
    assert torch.isfinite(dx[~hit]).all() and torch.isnan(dx[hit]).all()


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_nan_parameters_reach_their_gradients(act):
    """A NaN in one channel's bias: NaN where autograd of the same formulas has it, ReLU's slope of 1 there included."""
    x, w, b, d_out = _inputs((2, 40, 32), F32, seed=19)
    b[9] = math.nan
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    rows = torch.group_norm(leaves[0].transpose(1, 2), 4, leaves[1], leaves[2]).transpose(1, 2)
    want = torch.autograd.grad(ACTS[act](rows), leaves, d_out.double())
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(ops.group_norm_act(leaves[0], 4, leaves[1], leaves[2], activation=act), leaves, d_out.to(DEV))
    assert act in ("none", "relu") or want[2].isnan().any()
    for name, t, v in zip(("x", "weight", "bias"), got, want):
        assert torch.equal(t.isnan().cpu(), v.isnan()), name
        torch.testing.assert_close(t.double().cpu(), v, rtol=1e-4, atol=1e-4, equal_nan=True)


def test_offsets_past_32_bits():
    """Two images and a pixel stride that put elements more than 2^31 apart."""
    far = 2**31 + 64
    memory = torch.empty(far + 4096, dtype=BF16, device=DEV)
    x, w, b, d_out = _inputs((2, 9, 64), BF16, seed=12)
    view = torch.as_strided(memory, (2, 9, 64), (far, 128, 1))
    d = torch.as_strided(memory, (2, 9, 64), (far, 128, 1), 1152)
    view.copy_(x.to(DEV))
    d.copy_(d_out.to(DEV))
    leaf = view.detach().requires_grad_()
    out = ops.group_norm_act(leaf, 8, w.to(DEV), b.to(DEV), activation="gelu")
    dense = x.to(DEV).requires_grad_()
    want = ops.group_norm_act(dense, 8, w.to(DEV), b.to(DEV), activation="gelu")
    assert torch.equal(out, want)
    assert torch.equal(torch.autograd.grad(out, leaf, d)[0], torch.autograd.grad(want, dense, d_out.to(DEV))[0])


def test_more_images_than_a_launch_has_workgroups():
    """2^23 images and some: a workgroup each, and their partials' merge, take several launches. Spot images; the parameters'
    gradients over all of them."""
    n, w, b = 2**23 + 5, *_inputs((1, 1, 8), F32, seed=20)[1:3]
    g = torch.Generator(device=DEV).manual_seed(21)
    x, d_out = (torch.randn(n, 2, 8, generator=g, device=DEV, dtype=BF16) for _ in range(2))
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    out = ops.group_norm_act(leaves[0], 4, leaves[1], leaves[2], eps=0.01)
    dx, dw, db = torch.autograd.grad(out, leaves, d_out)
    at = torch.tensor([0, 1, 2**22 - 1, 2**22, 2**22 + 1, 2**23 - 1, 2**23, n - 1])
    xs, ds = x[at.to(DEV)].cpu(), d_out[at.to(DEV)].cpu()
    want = ref.group_norm_act(xs, 4, w, b, 0.01, "none")
    _check(out[at.to(DEV)], want, _forward_bound(xs, 4, w, b, 0.01, want))
    _check_gradients({"x": dx[at.to(DEV)]}, xs, 4, w, b, 0.01, "none", ds)
    v = x.view(n, 2, 4, 2).double()
    mean = v.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(dim=(1, 3), keepdim=True) + 0.01)
    hat, d = ((v - mean) * rstd).view(-1, 8), d_out.view(-1, 8).double()
    off = 2.0**-20 * ((v.abs() + mean.abs()) * rstd).view(-1, 8)  # of xhat
    for got, terms, moved in ((dw, d * hat, d.abs() * off), (db, d, 0 * d)):
        _check(got, terms.sum(0).cpu(), (moved.sum(0) + 2.0**-19 * terms.abs().sum(0)).cpu())


@pytest.mark.parametrize("shape,groups", [((2, 700, 1024), 1024), ((3, 130, 1040), 520), ((1, 9000, 640), 640)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_than_512_groups(shape, groups, dtype):
    """Their partials are merged by a launch of their own, in either direction."""
    x, w, b, d_out = _inputs(shape, dtype, seed=groups)
    _forward(x, groups, w, b, 1e-5, "silu")
    _backward(x, groups, w, b, 1e-5, "silu", d_out)


def test_same_bits_every_time_and_on_another_stream():
    x, w, b, d_out = (t.to(DEV) for t in _inputs((2, 100, 90, 64), BF16, seed=13))
    leaf = x.requires_grad_()

    def both():
        out = ops.group_norm_act(leaf, 8, w, b, activation="gelu")
        return out.detach(), torch.autograd.grad(out, leaf, d_out)[0]

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            again = both()
        side.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(first, again))


def test_gradient_against_differences():
    """The float64 definition's central differences along random directions against the kernel's FP32 gradients: the
    gradients are good to 2^-15 of the terms' magnitudes, the differences to their step's square."""
    x, w, b, d_out = _inputs((2, 30, 24), F32, seed=14)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.group_norm_act(leaves[0], 3, leaves[1], leaves[2], activation="gelu"), leaves,
                                d_out.to(DEV))

    def loss(x, w, b):
        return (ref.group_norm_act(x, 3, w, b, 1e-5, "gelu") * d_out.double()).sum().item()

    g, step = torch.Generator().manual_seed(15), 1e-4
    base = [t.double() for t in (x, w, b)]
    for i in range(3):
        v = torch.randn(base[i].shape, generator=g).double()
        moved = [[t + s * step * v if k == i else t for k, t in enumerate(base)] for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        dot = (grads[i].double().cpu() * v).sum().item()
        scale = (grads[i].double().cpu() * v).abs().sum().item()
        assert abs(slope - dot) <= 2.0**-15 * scale + 10 * step**2 * scale, (i, slope, dot)


def test_graph_capture():
    x, w, b, d_out = (t.to(DEV) for t in _inputs((2, 50, 60, 64), BF16, seed=16))
    leaf = x.requires_grad_()

    def both():
        out = ops.group_norm_act(leaf, 8, w, b, activation="silu")
        return out.detach(), torch.autograd.grad(out, leaf, d_out)[0]

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
            leaf.copy_(_inputs((2, 50, 60, 64), BF16, seed=20 + seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(captured, both()))


def test_refusals():
    x = torch.randn(2, 5, 48, device=DEV)
    for args, kwargs in [((x, 5), {}), ((x, 0), {}), ((x, 4, torch.ones(47, device=DEV)), {}), ((x, 4), {"activation": "tanh"}),
                         ((x.double(), 4), {}), ((x, 4, torch.ones(48)), {}), ((torch.randn(1, 2, 8200, device=DEV), 8), {}),
                         ((torch.randn(8, device=DEV), 4), {})]:
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.group_norm_act(*args, **kwargs)
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(ops.group_norm_act(leaf, 4).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="not implemented"):  # no second derivative
        g.sum().backward()
    with pytest.raises(ValueError):
        torch.ops.flashim_amd.group_norm_act(x, 5, None, None, 1e-5, 0)
    with pytest.raises(RuntimeError):
        torch.ops.flashim_amd.group_norm_act(x, 4, None, None, 1e-5, 9)
