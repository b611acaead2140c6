"""Orthogonalization, the optimizer step made of it and the low-rank adapters without a GPU: the float64 oracle against torch, the
torch operators' fakes (forward and backward), their refusals, version counters, and the C ABI's argument checks."""

import ctypes
import math

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

from flashim_amd import _lib, library, ops, optim
from flashim_amd.backends.hip import train as ht
from oracle import train as ref

BF16 = torch.bfloat16


# -- the oracle ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("shape", [(6, 9), (9, 6), (5, 5)])
def test_oracle_orthogonalize_is_the_polynomial_of_the_singular_values(shape):
    g = torch.randn(shape, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    u, s, v = torch.linalg.svd(g, full_matrices=False)
    s = s / (g.norm() + 1e-7)
    a, b, c = ref.NEWTON_SCHULZ
    for _ in range(5):
        s = a * s + b * s**3 + c * s**5
    torch.testing.assert_close(ref.orthogonalize(g), u @ torch.diag(s) @ v, rtol=1e-10, atol=1e-10)


def test_oracle_bound_covers_a_perturbed_iteration():
    """Steps rounded to 20 bits instead of 22 and FP32 sums end within 2^2 of the bound."""
    g = torch.randn(12, 30, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    a, b, c = ref.NEWTON_SCHULZ

    def rounded(t):
        m, e = torch.frexp(t)
        return torch.ldexp(torch.round(m * 2**20) / 2**20, e)

    x = rounded(g / (g.norm() + 1e-7))
    for _ in range(5):
        gram = rounded(x @ x.t())
        x = rounded(rounded(a * torch.eye(12, dtype=torch.float64) + b * gram + c * gram @ gram) @ x)
    assert (x - ref.orthogonalize(g)).norm().item() <= 4 * ref.schulz_bound(g)


@pytest.mark.parametrize("base", [True, False])
def test_oracle_adapters_match_torch(base):
    g = torch.Generator().manual_seed(2)
    x, a, b, z = (torch.randn(s, generator=g, dtype=torch.float64).requires_grad_() for s in ((4, 3, 6), (3, 2, 6), (3, 5, 2), (4, 3, 5)))
    index, scale = torch.tensor([2, -1, 0, 2]), torch.tensor([0.5, 2.0, 1.5])
    d = torch.randn(4, 3, 5, generator=g, dtype=torch.float64)
    rows = [scale[j].double() * x[i] @ a[j].t() @ b[j].t() if j >= 0 else x[i] @ torch.zeros(6, 5, dtype=torch.float64)
            for i, j in enumerate(index.tolist())]
    want = torch.stack(rows) + (z if base else 0)
    got = ref.low_rank_adapters(z.detach() if base else None, x.detach(), a.detach(), b.detach(), index, scale, d)
    torch.testing.assert_close(got["out"], want.detach(), rtol=1e-11, atol=1e-11)
    for name, v in zip("xab", torch.autograd.grad(want, (x, a, b), d)):
        torch.testing.assert_close(got[name], v, rtol=1e-11, atol=1e-11)


# -- fakes ---------------------------------------------------------------------------------------------------------------


def _fake(*tensors):
    mode = FakeTensorMode(allow_non_fake_inputs=False)
    return mode, [mode.from_tensor(t).to("meta") for t in tensors]


def test_orthogonalize_and_step_fakes():
    mode, (g, p, m) = _fake(torch.randn(3, 8, 5).to(BF16), torch.randn(3, 8, 5), torch.randn(3, 8, 5))
    with mode:
        out = ht.orthogonalize(g)
        assert out.shape == g.shape and out.dtype == BF16
        assert ht.orthogonalize(g, out_dtype=torch.float32).dtype == torch.float32
        assert ht.muon_step_([p], [g], [m], lr=0.1) is None


@pytest.mark.parametrize("k, n, rank, columns", [(16, 24, 4, 0), (16, 24, 32, 0), (16, 24, 33, 64), (200, 300, 4, 16), (200, 300, 100, 128)])
def test_adapters_fakes(k, n, rank, columns):
    """Also: the columns of h that a fake forward saves are those that the library asks for."""
    saved = ctypes.c_int64()
    assert _lib.load().fim_low_rank_adapters_saved(k, n, rank, ctypes.byref(saved)) == 0 and saved.value == columns
    mode, (base, x, a, b, index) = _fake(torch.randn(2, 7, n).to(BF16), torch.randn(2, 7, k).to(BF16), torch.randn(3, rank, k).to(BF16),
                                         torch.randn(3, n, rank).to(BF16), torch.zeros(2, dtype=torch.int64))
    with mode:
        leaves = [t.detach().requires_grad_() for t in (base, x, a, b)]
        out = ht.low_rank_adapters(*leaves, index, scale=0.5)
        assert out.shape == base.shape and out.dtype == BF16
        for t, g in zip(leaves, torch.autograd.grad(out, leaves, torch.empty_like(out))):
            assert g.shape == t.shape and g.dtype == t.dtype
        assert library.low_rank_adapters(base, x, a, b, index, None, 1.0, True)[1].shape == (14, columns)
        only = a.detach().requires_grad_()
        out = ht.low_rank_adapters(None, x, only, b, index)
        assert torch.autograd.grad(out, only, torch.empty_like(out))[0].shape == a.shape


# -- autograd ------------------------------------------------------------------------------------------------------------


def test_a_step_counts_its_writes():
    p, g, m = (torch.empty(4, 5, device="meta") for _ in range(3))
    x = torch.empty(4, 5, device="meta", requires_grad=True)
    y = x * p
    ht.muon_step_([p], [g], [m], lr=0.1)
    assert (p._version, g._version, m._version) == (1, 0, 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(NotImplementedError, match="no derivative"):
        torch.ops.flashim_amd.muon_step_([x], [g], [m], 0.1, 0.9, True, 0.0, 0, 5, 3.0, -3.0, 1.0, 1e-7)


@pytest.mark.parametrize("grads", [True, False])
def test_forward_mode_is_refused(grads):
    x, a, b = (torch.empty(s, device="meta", dtype=BF16) for s in ((2, 3, 16), (4, 2, 16), (4, 8, 2)))
    base, index = torch.empty(2, 3, 8, device="meta", dtype=BF16), torch.empty(2, device="meta", dtype=torch.int64)
    p, m = torch.empty(4, 5, device="meta"), torch.empty(4, 5, device="meta")
    calls = [(lambda t: ht.low_rank_adapters(base, t, a, b, index), x), (lambda t: ht.low_rank_adapters(t, x, a, b, index), base),
             (lambda t: ht.low_rank_adapters(base, x, a, t, index), b)]
    with torch.set_grad_enabled(grads), forward_ad.dual_level():
        for call, t in calls:
            with pytest.raises(RuntimeError, match="jvp is not implemented"):
                call(forward_ad.make_dual(t, torch.empty_like(t)))
        for lists in (([p], [forward_ad.make_dual(p.clone(), p.clone())], [m]), ([forward_ad.make_dual(p.clone(), p.clone())], [p], [m])):
            with pytest.raises(NotImplementedError, match="has a tangent"):
                ht.muon_step_(*lists, lr=0.1)


@pytest.mark.parametrize("create_graph", [False, True])
def test_a_tangent_of_the_incoming_gradient_is_refused(create_graph):
    x = torch.empty(2, 3, 16, device="meta", dtype=BF16, requires_grad=True)
    a, b = (torch.empty(s, device="meta", dtype=BF16) for s in ((4, 2, 16), (4, 8, 2)))
    out = ht.low_rank_adapters(None, x, a, b, torch.empty(2, device="meta", dtype=torch.int64))
    d = torch.empty_like(out)
    assert torch.autograd.grad(out, x, d, retain_graph=True)[0].shape == x.shape
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        torch.autograd.grad(out, x, forward_ad.make_dual(d, torch.empty_like(d)), create_graph=create_graph)


# -- the optimizer -------------------------------------------------------------------------------------------------------


def test_optimizer_sorts_its_parameters(monkeypatch):
    calls = []
    monkeypatch.setattr(optim.ops, "muon_step_", lambda p, g, m, **kw: calls.append((p, g, m, kw)))
    matrix, stack, vector, still = (torch.nn.Parameter(torch.ones(s)) for s in ((3, 4), (2, 3, 4), (5,), (3, 4)))
    opt = optim.Muon([{"params": [matrix, vector, still]}, {"params": [stack], "lr": 0.5, "steps": 3}], lr=0.1, adam_lr=0.01)
    for p in (matrix, stack, vector):
        p.grad = torch.full_like(p, 2.0)
    assert opt.step(lambda: 7.0) == 7.0
    assert [c[0] for c in calls] == [[matrix], [stack]] and [c[3]["lr"] for c in calls] == [0.1, 0.5] and calls[1][3]["steps"] == 3
    assert calls[0][1] == [matrix.grad] and calls[0][2][0].dtype == torch.float32 and (calls[0][2][0] == 0).all()
    torch.testing.assert_close(vector.detach(), torch.full((5,), 0.99))  # Adam's first step: its learning rate
    assert (still == 1).all() and still not in opt.state
    opt.step()
    assert calls[2][2][0] is calls[0][2][0] and opt.state[vector]["step"] == 2


def test_optimizer_keeps_fp32_momenta_through_a_state_dict(monkeypatch):
    monkeypatch.setattr(optim.ops, "muon_step_", lambda p, g, m, **kw: [t.add_(1 + 2.0**-20) for t in m])
    first, second = (torch.nn.Parameter(torch.ones(3, 4, dtype=BF16)) for _ in range(2))
    a, b = optim.Muon([first]), optim.Muon([second])
    first.grad = torch.ones_like(first)
    a.step()
    b.load_state_dict(a.state_dict())
    assert b.state[second]["momentum"].dtype == torch.float32
    assert torch.equal(b.state[second]["momentum"], a.state[first]["momentum"])
    assert b.state[second]["momentum"] is not a.state[first]["momentum"]
    with pytest.raises(ValueError):
        optim.Muon([first], lr=-1.0)


# -- refusals ------------------------------------------------------------------------------------------------------------


def test_no_cpu_fallback():
    g, x = torch.randn(4, 5), torch.randn(2, 8).to(BF16)
    a, b = torch.randn(3, 2, 8).to(BF16), torch.randn(3, 6, 2).to(BF16)
    for call in (lambda: ops.orthogonalize(g), lambda: ops.muon_step_([g], [g], [g], lr=0.1),
                 lambda: ops.muon_step_([], [], [], lr=0.1), lambda: ops.low_rank_adapters(None, x, a, b, torch.zeros(2).long())):
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            call()


def test_c_abi_checks_its_arguments():
    lib = _lib.load()
    fake, out = 1 << 20, ctypes.c_int64()  # stand-ins: the calls return before touching memory
    at, big = ctypes.byref(out), 1 << 40
    bad, no = _lib.FIM_ERR_INVALID, _lib.FIM_ERR_UNSUPPORTED
    assert lib.fim_orthogonalize_workspace(2, 100, 300, at) == 0 and out.value > 2 * 100 * 300 * 8
    assert lib.fim_orthogonalize_workspace(2, 100, 300, None) == bad
    assert lib.fim_orthogonalize_workspace(-1, 100, 300, at) == bad
    assert lib.fim_orthogonalize_workspace(1, 1 << 15, 1 << 15, at) == no

    def orthogonalize(g=fake, dtype=0, steps=5, a=3.4445, b=-4.7750, c=2.0315, eps=1e-7, to=fake, to_dtype=0, ws=fake, size=big):
        return lib.fim_orthogonalize(g, dtype, 1, 100, 300, steps, a, b, c, eps, to, to_dtype, ws, size, None)

    assert orthogonalize(g=None) == orthogonalize(dtype=3) == orthogonalize(steps=0) == orthogonalize(steps=101) == bad
    assert orthogonalize(eps=-1.0) == orthogonalize(eps=math.nan) == orthogonalize(to=None) == orthogonalize(to_dtype=-1) == bad
    assert orthogonalize(g=fake + 2) == orthogonalize(ws=None) == orthogonalize(ws=fake + 128) == orthogonalize(size=1000) == bad
    assert orthogonalize(a=10.0) == orthogonalize(c=math.nan) == orthogonalize(b=math.inf) == orthogonalize(c=200.0) == no
    one = (ctypes.c_int64 * 1)
    ptrs, types, factors = (ctypes.c_void_p * 1)(fake), (ctypes.c_int * 1)(0), (ctypes.c_float * 1)(1.0)

    def step(params=ptrs, types=types, momenta=ptrs, factors=factors, rows=100, ws=fake):
        return lib.fim_muon_step(1, params, types, ptrs, types, momenta, one(1), one(rows), one(300), factors, 0.9, 1, 1.0, 5, 3.4445,
                                 -4.7750, 2.0315, 1e-7, ws, big, None)

    assert lib.fim_muon_step_workspace(1, one(2), one(100), one(300), at) == 0 and out.value > 0
    assert lib.fim_muon_step_workspace(1, one(2), one(-1), one(300), at) == bad
    assert step(params=None) == step(momenta=None) == step(factors=None) == step(rows=-1) == step(ws=None) == bad
    assert step(types=(ctypes.c_int * 1)(7)) == step(momenta=(ctypes.c_void_p * 1)(fake + 2)) == bad
    assert lib.fim_low_rank_adapters_saved(8, 8, 0, at) == lib.fim_low_rank_adapters_saved(8, 8, 4, None) == bad
    assert lib.fim_low_rank_adapters_saved(8, 8, 129, at) == no

    def adapt(x=fake, dtype=1, m=100, k=64, n=48, j=3, r=8, index=fake, wide=1, entries=10, to=fake, h=None):
        return lib.fim_low_rank_adapters(fake, n, x, k, dtype, m, k, n, fake, fake, j, r, index, wide, entries, None, 1.0, to, h, None)

    assert adapt(x=None) == adapt(dtype=3) == adapt(m=-1) == adapt(k=0) == adapt(j=0) == adapt(r=0) == adapt(wide=2) == bad
    assert adapt(entries=7) == adapt(entries=0) == adapt(index=None) == adapt(index=fake + 4) == adapt(to=None) == adapt(h=fake + 4) == bad
    assert adapt(x=fake + 1) == bad
    assert adapt(dtype=0) == adapt(r=129) == adapt(m=1 << 31, entries=1) == adapt(j=1 << 20) == no
    assert lib.fim_low_rank_adapters_backward_workspace(100, 600, 48, 3, 8, at) == 0 and out.value > 0
    assert lib.fim_low_rank_adapters_backward_workspace(100, 64, 48, 3, 8, None) == bad

    def backward(k=600, h=fake, dx=fake, da=fake, db=fake, ws=fake, size=big, m=100):
        return lib.fim_low_rank_adapters_backward(fake, 48, fake, k, 1, m, k, 48, fake, fake, 3, 8, fake, 1, 10, None, 1.0, h, dx, da, db,
                                                  ws, size, None)

    assert backward(h=None) == backward(da=None) == backward(db=None) == backward(ws=None) == backward(ws=fake + 8) == backward(size=0) == bad
    assert backward(m=0) == bad
    assert backward(dx=None, da=None, db=None) == 0  # nothing to do


def test_c_abi_refuses_what_one_launch_cannot_hold():
    lib = _lib.load()
    fake, out = 1 << 20, ctypes.c_int64()
    at, no = ctypes.byref(out), _lib.FIM_ERR_UNSUPPORTED
    assert lib.fim_orthogonalize_workspace(1 << 22, 16, 16, at) == no
    assert lib.fim_orthogonalize_workspace(1 << 20, 16, 16, at) == 0
    assert lib.fim_low_rank_adapters(fake, 8, fake, 8, 1, 1 << 28, 8, 8, fake, fake, 1, 4, fake, 1, 1, None, 1.0, fake, None, None) == no
    assert lib.fim_low_rank_adapters_backward(fake, 600, fake, 600, 1, 64, 600, 1 << 23, fake, fake, 100, 128, fake, 1, 1, None, 1.0,
                                              fake, fake, fake, fake, fake, 1 << 50, None) == no


def test_partial_sums_of_many_adapters_stay_small():
    """However long the input: chunks are fewer and longer, so that all adapters' sums take at most 256 MB."""
    lib, out = _lib.load(), ctypes.c_int64()
    for m, k, n, j, r in ((1 << 20, 64, 256, 1000, 8), (1 << 21, 128, 256, 100, 32), (1 << 24, 64, 64, 2000, 16)):
        assert lib.fim_low_rank_adapters_backward_workspace(m, k, n, j, r, ctypes.byref(out)) == 0
        assert out.value <= (256 << 20) + j * 1024 * 4 + 4096


# -- memory of a step's tensors --------------------------------------------------------------------------------------------


def _apart(tensors):
    """``fim_host_apart`` of ``(address, element bytes, written, [(stride in bytes, size)])``."""
    fn, i64 = _lib.load_host().fim_host_apart, ctypes.c_int64

    def array(kind, values):
        return (kind * max(1, len(values)))(*values)

    dims = [d for t in tensors for d in t[3]]
    return fn(i64(len(tensors)), array(i64, [t[0] for t in tensors]), array(i64, [t[1] for t in tensors]),
              array(ctypes.c_uint8, [t[2] for t in tensors]), array(i64, [len(t[3]) for t in tensors]),
              array(i64, [d[0] for d in dims]), array(i64, [d[1] for d in dims])) == 1


def _apart_by_bytes(tensors):
    """The same, byte by byte."""
    seen, read = set(), set()
    for address, size, written, dims in tensors:
        at = [address]
        for stride, n in dims:
            at = [x + stride * i for x in at for i in range(n)]
        own = [x + i for x in at for i in range(size)]
        if written and (len(set(own)) < len(own) or not read.isdisjoint(own)) or not seen.isdisjoint(own):
            return False
        (seen if written else read).update(own)
    return True


def test_overlaps_of_strided_tensors_are_found_exactly():
    """Two or three tensors of up to three dimensions, random and nested strides: byte by byte the same answer, both often."""
    g = torch.Generator().manual_seed(0)

    def pick(*values):
        return values[torch.randint(0, len(values), (), generator=g).item()]

    answers = [0, 0]
    for trial in range(4000):
        tensors = []
        row = pick(24, 40, 64)  # bytes of a row of a shared buffer
        for _ in range(pick(2, 2, 3)):
            es = pick(2, 4)
            if trial % 2:  # views of rows
                step, cols = es * pick(1, 1, 2, 3), pick(1, 2, 3, 5)
                dims = [(row * pick(1, 2), pick(1, 3, 4)), (step, cols)]
                dims = dims[::-1] if pick(0, 1) else dims
                address = row * pick(0, 0, 1) + es * pick(0, 1, 2, 4, 6, 8)
            else:
                dims = [(es * pick(0, 1, 2, 3, 5, 7, 11, 13), pick(1, 2, 3, 4)) for _ in range(pick(0, 1, 2, 3))]
                address = es * torch.randint(0, 60, (), generator=g).item()
            tensors.append((address, es, pick(0, 1, 1), dims))
        want = _apart_by_bytes(tensors)
        answers[want] += 1
        assert _apart(tensors) == want, tensors
    assert min(answers) > 800, answers


def test_overlaps_of_large_tensors_are_found_in_few_steps():
    """Halves of a matrix's columns, its transposes and interleaved slices at full size; strides that do not nest count as overlapping
    once the search grows long."""
    n = 1 << 20
    left, right = (0, 4, 1, [(8 * n, n), (4, n)]), (4 * n, 4, 1, [(4, n), (8 * n, n)])
    assert _apart([left, right]) and not _apart([left, (4 * n - 4, 4, 1, right[3])])
    assert _apart([(0, 4, 1, [(8, n)]), (4, 4, 1, [(8, n)]), (8 * n, 2, 0, [(0, n), (2, n)])])
    assert not _apart([(0, 4, 1, [(8, n)]), (4 * n, 2, 0, [(4, n)])])
    assert not _apart([(0, 4, 1, [(12, n), (8, n)])])
    assert not _apart([(0, 2, 1, [(10**6 + 2, 1000), (10**6 - 2, 999), (10**6 + 6, 998)]),
                       (2, 2, 1, [(10**6 + 4, 1000), (10**6 - 8, 999), (10**6 + 14, 998)])])


def test_adapters_whose_gradients_one_launch_cannot_hold_are_refused_by_the_workspace():
    lib, out = _lib.load(), ctypes.c_int64()
    at, no = ctypes.byref(out), _lib.FIM_ERR_UNSUPPORTED

    def workspace(m, k, n, j, r):
        return lib.fim_low_rank_adapters_backward_workspace(m, k, n, j, r, at)

    assert workspace(3, 32768 - 64, 64, 1024, 128) == no  # 2^32 elements of adapters
    assert workspace(3, 32768 - 65, 64, 1024, 128) == 0
    assert workspace(3, 1 << 23, 1, 1, 128) == no  # 2^30 of one
    # many tiny adapters: fewer chunks, not more workgroups than a launch has
    for j in (1 << 15, 1 << 17, (1 << 20) - 1):
        assert workspace(1 << 20, 1, 1, j, 1) == 0 and workspace(1 << 20, 8, 400, j, 1) == 0


def test_optimizer_refuses_what_is_neither_a_matrix_nor_a_stack():
    """A convolution's weight, of which the stack would be its kernels; a group that is refused leaves the optimizer as it was."""
    conv = torch.nn.Conv2d(3, 4, 3)
    with pytest.raises(ValueError, match="neither a matrix"):
        optim.Muon(conv.parameters())
    opt = optim.Muon([conv.bias])
    with pytest.raises(ValueError, match="neither a matrix"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(2, 3)), conv.weight]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": torch.nn.Parameter(conv.weight.detach().flatten(1))})
    assert len(opt.param_groups) == 2


@pytest.mark.parametrize("shape", [(16, 512), (64, 256), (48, 100), (40, 1500), (7, 3696), (96, 96), (65, 65), (100, 200), (130, 150)])
def test_oracle_tells_a_product_without_its_low_halves(shape):
    """Of matrices as gradients are: an iteration that drops the low halves of one of its products ends at least twice as far from
    the exact result as 4 times one that keeps them, the tolerance of the tests that hold the kernels to it."""
    g = torch.Generator().manual_seed(3)
    few = min(6, *shape)
    strong = torch.randn(shape[0], few, generator=g) * torch.exp(-0.5 * torch.arange(few))
    u = strong @ torch.randn(few, shape[1], generator=g) + 0.05 * torch.randn(shape, generator=g)
    want = ref.orthogonalize(u)
    off = {name: (ref.schulz_halves(u, leave_out=name) - want).norm() for name in ("", "gram", "square", "apply")}
    assert off[""] <= 1e-5 * want.norm()
    for name in ("gram", "square", "apply"):
        assert off[name] >= 8 * off[""], (name, off)
    if shape[0] != shape[1]:  # (a tall one's is the other's; a square one's sums run otherwise)
        torch.testing.assert_close(ref.schulz_halves(u.t()), ref.schulz_halves(u).t())


def test_workspaces_of_every_shape_are_found():
    """Each number of rows past and below what a workgroup holds, beside lengths on both sides of every rule (128 x 2048, say)."""
    lib, out = _lib.load(), ctypes.c_int64()
    for rows in range(1, 700):
        for cols in (1, 31, 33, 64, 100, 512, 1000, 1537, 1568, 1569, 2048, 4096, 10000, 65536, 131072):
            for shape in ((rows, cols), (cols, rows)):
                assert lib.fim_orthogonalize_workspace(3, *shape, ctypes.byref(out)) == 0
                m, n = (-(-x // 32) * 32 for x in sorted(shape))
                # halves of X twice, A and P, but for matrices that stay in a workgroup and, once, in slabs' ones
                least = 0 if min(shape) <= 64 else 3 * 4 * (2 * m * n + 2 * m * m)
                assert least <= out.value <= 3 * 4 * (2 * m * n + 2 * m * m) + 3 * (4 << 20) + (1 << 28), shape


def test_coefficients_that_diverge_between_common_points_are_refused():
    """Singular values in a window of 1e-4 pass 6 in ten steps of this polynomial; its neighbour keeps all of them below 2."""
    lib, fake = _lib.load(), 1 << 20

    def call(a, b, c, steps):
        return lib.fim_orthogonalize(fake, 0, 1, 0, 300, steps, a, b, c, 1e-7, fake, 0, None, 0, None)  # (no rows: nothing is launched)

    x = torch.linspace(0, 1, 2_000_001, dtype=torch.float64)
    for (a, b, c), refused in (((2.3763397567, -4.95683002527, 1.579664002893), True), ((2.3763397567, -4.5, 1.579664002893), False)):
        v, most = x, 0.0
        for _ in range(10):
            v = v * (a + b * v**2 + c * v**4)
            most = max(most, v.abs().max().item())
        assert (most > 6) == refused
        assert call(a, b, c, 10) == (_lib.FIM_ERR_UNSUPPORTED if refused else 0)
    for coefficients, steps in ((ref.NEWTON_SCHULZ, 5), (ref.NEWTON_SCHULZ, 100), ((1.5, -0.5, 0.0), 12), ((0.0, 0.0, 1.0), 3),
                                ((1.0, 0.0, 0.0), 1), ((-1.5, 0.5, 0.0), 4)):
        assert call(*coefficients, steps) == 0
