"""The training-step operators without a GPU: the float64 oracle against torch's own autograd, the torch operators' fakes
(forward and backward), their refusals, version counters, and the C ABI's argument checks."""

import ctypes
import math

import pytest
import torch
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

from flashim_amd import _lib, gated, library, ops
from flashim_amd.backends.hip import train as ht
from oracle import train as ref

ACTS = {"none": lambda z: z, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh")}


# -- the oracle ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape,groups", [((2, 5, 7, 12), 3), ((1, 1, 8), 8), ((3, 11, 6), 1)])
def test_oracle_group_norm_matches_torch(act, shape, groups):
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(s, generator=g, dtype=torch.float64).requires_grad_() for s in (shape, shape[-1:], shape[-1:]))
    d = torch.randn(shape, generator=g, dtype=torch.float64)
    rows = x.reshape(shape[0], -1, shape[-1]).transpose(1, 2)
    want = ACTS[act](torch.group_norm(rows, groups, w, b, 1e-3).transpose(1, 2).reshape(shape))
    got = ref.group_norm_act(x.detach(), groups, w.detach(), b.detach(), 1e-3, act)
    torch.testing.assert_close(got, want.detach(), rtol=1e-11, atol=1e-11)
    grads = ref.group_norm_act_gradients(d, x.detach(), groups, w.detach(), b.detach(), 1e-3, act)
    for name, v in zip(("x", "weight", "bias"), torch.autograd.grad(want, (x, w, b), d)):
        torch.testing.assert_close(grads[name], v, rtol=1e-9, atol=1e-9)


@pytest.mark.parametrize("act", ACTS)
def test_oracle_gated_linear_matches_torch(act):
    g = torch.Generator().manual_seed(1)
    x, wg, wu, bg, bu = (torch.randn(s, generator=g, dtype=torch.float64).requires_grad_()
                         for s in ((9, 6), (7, 6), (7, 6), (7,), (7,)))
    d = torch.randn(9, 7, generator=g, dtype=torch.float64)
    want = ACTS[act](F.linear(x, wg, bg)) * F.linear(x, wu, bu)
    args = [t.detach() for t in (x, wg, wu, bg, bu)]
    torch.testing.assert_close(ref.gated_linear(*args, act)[0], want.detach(), rtol=1e-11, atol=1e-11)
    grads = ref.gated_linear_gradients(d, *args, act)
    for name, v in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), torch.autograd.grad(want, (x, wg, wu, bg, bu), d)):
        torch.testing.assert_close(grads[name], v, rtol=1e-9, atol=1e-9)


def test_oracle_clip_matches_torch():
    g = torch.Generator().manual_seed(2)
    params = [torch.nn.Parameter(torch.zeros(n, dtype=torch.float64)) for n in (5, 60)]
    for norm in (2.0, math.inf):
        for p in params:
            p.grad = torch.randn(p.shape, generator=g, dtype=torch.float64)
        grads = [p.grad.clone() for p in params]
        total = torch.nn.utils.clip_grad_norm_(params, 0.7, norm_type=norm)
        torch.testing.assert_close(ref.grad_norm(grads, norm), total)
        scale = ref.clip_scale(total, 0.7)
        for p, q in zip(params, grads):
            torch.testing.assert_close(q * scale, p.grad)


# -- fakes ---------------------------------------------------------------------------------------------------------------


def _fake(*tensors):
    mode = FakeTensorMode(allow_non_fake_inputs=False)
    return mode, [mode.from_tensor(t).to("meta") for t in tensors]  # autograd of a fake cuda tensor asks for a stream


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_norm_fakes(dtype):
    mode, (x, w, b) = _fake(torch.randn(2, 3, 5, 32).to(dtype), torch.randn(32), torch.randn(32).to(dtype))
    with mode:
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        out = ht.group_norm_act(leaves[0], 4, leaves[1], leaves[2], activation="gelu")
        assert out.shape == x.shape and out.dtype == dtype and out.requires_grad
        for t, g in zip(leaves, torch.autograd.grad(out, leaves, torch.empty_like(out))):
            assert g.shape == t.shape and g.dtype == t.dtype
        stats = library.group_norm_act(x, 4, None, None, 1e-5, 0)[1]
        assert stats.shape == (2, 4, 2) and stats.dtype == torch.float32
        dx, dw, db = library.group_norm_act_backward(x, x, stats, 4, None, b, 0)
        assert dx.shape == x.shape and dw.shape == (0,) and db.shape == (32,) and db.dtype == dtype


def test_gated_linear_fakes():
    half = torch.bfloat16
    mode, (x, wg, wu, bg, bu) = _fake(torch.randn(2, 3, 16).to(half), torch.randn(24, 16).to(half),
                                      torch.randn(24, 16).to(half), torch.randn(24), torch.randn(24))
    with mode:
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, bg, bu)]
        out = ht.gated_linear(*leaves, activation="silu")
        assert out.shape == (2, 3, 24) and out.dtype == half
        for t, g in zip(leaves, torch.autograd.grad(out, leaves, torch.empty_like(out))):
            assert g.shape == t.shape and g.dtype == t.dtype
        only = wu.detach().requires_grad_()
        out = ht.gated_linear(x, wg, only)
        assert torch.autograd.grad(out, only, torch.empty_like(out))[0].shape == (24, 16)


def test_clip_fakes():
    mode, grads = _fake(torch.randn(5), torch.randn(7).to(torch.bfloat16))
    with mode:
        assert ht.grad_norm(grads).shape == () and ht.grad_norm(grads).dtype == torch.float32
        assert ht.clip_grad_norm_(grads, 1.0, norm_type=math.inf).shape == ()
        assert ht.clip_grad_norm_(grads, 1.0, out=[g.float() for g in grads]).dtype == torch.float32


def test_clip_counts_its_writes():
    """Autograd finds a saved tensor that was clipped since by its version counter."""
    grads = [torch.empty(5, device="meta"), torch.empty(7, device="meta")]
    out = [torch.empty(5, device="meta"), torch.empty(7, device="meta")]
    ht.clip_grad_norm_(grads, 1.0)
    assert [g._version for g in grads] == [1, 1]
    ht.clip_grad_norm_(grads, 1.0, out=out)
    assert [g._version for g in grads] == [1, 1] and [o._version for o in out] == [1, 1]
    x = torch.empty(5, device="meta", requires_grad=True)
    y = x * grads[0]
    ht.clip_grad_norm_(grads, 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(NotImplementedError):  # no derivative through the clip
        torch.ops.flashim_amd.clip_grad_norm_([x], 1.0, 2.0)


@pytest.mark.parametrize("grads", [True, False])
def test_forward_mode_is_refused(grads):
    """A tangent raises, under ``no_grad`` too: that ends the recording of gradients, not forward mode."""
    x, w = torch.empty(3, 16, device="meta", dtype=torch.bfloat16), torch.empty(8, 16, device="meta", dtype=torch.bfloat16)
    b = torch.empty(16, device="meta")
    calls = [(lambda t: ht.group_norm_act(t, 4), x), (lambda t: ht.group_norm_act(x, 4, None, t), b),
             (lambda t: ht.gated_linear(t, w, w), x), (lambda t: ht.gated_linear(x, w, t), w)]
    with torch.set_grad_enabled(grads):
        for call, t in calls:
            with pytest.raises(RuntimeError):
                torch.func.jvp(call, (t,), (torch.empty_like(t),))
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="jvp is not implemented"):
                call(forward_ad.make_dual(t, torch.empty_like(t)))
            assert not call(t).requires_grad


@pytest.mark.parametrize("create_graph", [False, True])
def test_a_tangent_of_the_incoming_gradient_is_refused(create_graph):
    """The backward passes have no forward-mode derivatives either: a tangent raises there, it is not dropped."""
    x = torch.empty(3, 16, device="meta", dtype=torch.bfloat16, requires_grad=True)
    w = torch.empty(8, 16, device="meta", dtype=torch.bfloat16)
    for out in (ht.group_norm_act(x, 4), ht.gated_linear(x, w, w)):
        d = torch.empty_like(out)
        assert torch.autograd.grad(out, x, d, retain_graph=True)[0].shape == x.shape
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, x, forward_ad.make_dual(d, torch.empty_like(d)), create_graph=create_graph)


def test_clip_refuses_tangents():
    """In place, a clipped gradient would keep its unclipped tangent."""
    with forward_ad.dual_level():
        plain = torch.empty(5, device="meta")
        dual = forward_ad.make_dual(torch.empty(5, device="meta"), torch.empty(5, device="meta"))
        for grads, out in (([plain, dual], None), ([dual], [torch.empty(5, device="meta")]), ([plain], [dual])):
            for mode in (True, False):
                with torch.set_grad_enabled(mode), pytest.raises(NotImplementedError, match="has a tangent"):
                    ht.clip_grad_norm_(grads, 1.0, out=out)
        assert plain._version == 0 and dual._version == 0


def test_train_step_of_a_module_without_gradients():
    """Frozen, beside a parameter that the loss also has: nothing to clip, and the other one still steps."""
    module, other = torch.nn.Linear(3, 2).requires_grad_(False), torch.nn.Parameter(torch.ones(2))
    loss, norm = gated.train_step(module, torch.optim.SGD([other], lr=0.5), lambda: (module(torch.ones(3)) * 0 + other).sum(), 1.0)
    assert loss.item() == 2.0 and norm.shape == () and norm.dtype == torch.float32 and norm.item() == 0.0
    assert torch.equal(other.detach(), torch.full((2,), 0.5))


# -- refusals ------------------------------------------------------------------------------------------------------------


def test_no_cpu_fallback():
    x, w = torch.randn(4, 16), torch.randn(8, 16)
    for call in (lambda: ops.group_norm_act(x, 4), lambda: ops.gated_linear(x.bfloat16(), w.bfloat16(), w.bfloat16()),
                 lambda: ops.grad_norm([x]), lambda: ops.clip_grad_norm_([x], 1.0), lambda: ops.grad_norm([]),
                 lambda: ops.grad_norm(x)):
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            call()


def test_c_abi_checks_its_arguments():
    lib = _lib.load()
    fake, out = 1 << 20, ctypes.c_int64()  # stand-ins: the calls return before touching memory
    at = ctypes.byref(out)
    assert lib.fim_group_norm_workspace(2, 100, 64, 8, 0, at) == 0 and out.value > 0
    assert lib.fim_group_norm_workspace(2, 100, 64, 7, 0, at) == _lib.FIM_ERR_INVALID
    assert lib.fim_group_norm_workspace(2, 100, 8200, 8, 0, at) == _lib.FIM_ERR_UNSUPPORTED
    assert lib.fim_group_norm_workspace(2, 100, 64, 8, 0, None) == _lib.FIM_ERR_INVALID

    def norm(dtype=1, groups=8, act=0, x=fake, stats=fake):
        return lib.fim_group_norm(x, dtype, 1, 10, 64, 640, 64, groups, None, 0, None, 0, 1e-5, act, fake, stats, fake, None)

    assert norm(dtype=3) == norm(groups=0) == norm(act=5) == norm(x=None) == norm(stats=None) == _lib.FIM_ERR_INVALID
    assert lib.fim_gated_linear_workspace(fake, 100, 64, 64, fake, 64, fake, 64, 128, 1, at) == 0 and out.value > 0
    assert lib.fim_gated_linear_workspace(fake, 100, 64, 64, fake, 64, fake, 64, 128, 0, at) == 0 and out.value == 0
    assert lib.fim_gated_linear_workspace(fake, 100, 63, 63, fake, 63, fake, 63, 128, 0, at) == 0 and out.value > 0

    def gated(dtype=1, k=64, act=0, bias_dtype=0, x=fake, workspace=None, size=0, stride=64):
        return lib.fim_gated_linear(x, dtype, 100, k, stride, fake, stride, fake, stride, 128, None, None, bias_dtype, act, fake,
                                    workspace, size, None)

    assert gated(dtype=0) == _lib.FIM_ERR_UNSUPPORTED
    assert gated(k=0) == gated(act=-1) == gated(bias_dtype=2) == gated(x=None) == _lib.FIM_ERR_INVALID
    assert gated(k=63, stride=63) == gated(k=63, stride=63, workspace=fake, size=16) == _lib.FIM_ERR_INVALID
    assert lib.fim_gated_linear_backward(fake, 1, 100, 64, 64, fake, 64, fake, 64, 128, None, None, 0, 0, fake, 1 << 22, fake,
                                         None, None, None, None, fake, 1 << 40, None) == _lib.FIM_ERR_UNSUPPORTED
    sizes = (ctypes.c_int64 * 2)(10, -1)
    assert lib.fim_grad_norm_workspace(2, sizes, at) == _lib.FIM_ERR_INVALID
    assert lib.fim_grad_norm_workspace(1, sizes, at) == 0 and out.value == 1
    ptrs, types = (ctypes.c_void_p * 1)(fake), (ctypes.c_int * 1)(0)
    assert lib.fim_grad_norm(1, ptrs, types, sizes, 1, fake, fake, None) == _lib.FIM_ERR_INVALID  # norm 1
    assert lib.fim_grad_norm(1, ptrs, (ctypes.c_int * 1)(5), sizes, 2, fake, fake, None) == _lib.FIM_ERR_INVALID
    assert lib.fim_grad_norm(1, (ctypes.c_void_p * 1)(fake + 2), types, sizes, 2, fake, fake, None) == _lib.FIM_ERR_INVALID
    assert lib.fim_grad_norm(1, ptrs, types, sizes, 2, None, fake, None) == _lib.FIM_ERR_INVALID
    assert lib.fim_clip_grad_norm(1, ptrs, types, None, types, sizes, 1.0, 2, fake, fake, None) == _lib.FIM_ERR_INVALID


def test_c_abi_refuses_a_misaligned_workspace():
    """The gated product's workspace holds operands of 16-byte loads; both calls return before touching memory."""
    lib = _lib.load()
    fake, size = 1 << 20, 1 << 40
    for off in (2, 8, 16, 128):
        assert lib.fim_gated_linear(fake, 1, 100, 63, 63, fake, 63, fake, 63, 128, None, None, 0, 0, fake, fake + off, size,
                                    None) == _lib.FIM_ERR_INVALID
        assert lib.fim_gated_linear_backward(fake, 1, 100, 64, 64, fake, 64, fake, 64, 128, None, None, 0, 0, fake, 128, fake,
                                             None, None, None, None, fake + off, size, None) == _lib.FIM_ERR_INVALID
