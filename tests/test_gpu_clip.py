"""``ops.grad_norm`` and ``ops.clip_grad_norm_`` against float64 (``oracle/train.py``). The norm's squares are summed in 64
bits: its error is the final FP32 rounding (2^-24 relative; 2^-23 with the root's own). A scaled element carries the
scale's few FP32 roundings (2^-22) and the output's own."""

import math

import pytest
import torch

from flashim_amd import ops
from oracle import train as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF16: 2.0**-8, F16: 2.0**-11, F32: 2.0**-24}
TINY = {BF16: 2.0**-134, F16: 2.0**-25, F32: 2.0**-150}


def _grads(sizes, dtypes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * math.exp(-(i % 7))).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def _check(grads, max_norm, norm_type, total, out):
    want = ref.grad_norm(grads, norm_type)
    assert total.dtype == F32 and total.ndim == 0
    assert abs(total.item() - want.item()) <= 2.0**-23 * want.item()
    scale = ref.clip_scale(want, max_norm)
    for g, o in zip(grads, out):
        exact = g.double() * scale
        bound = (U[o.dtype] + 2.0**-22) * exact.abs() + TINY[o.dtype]
        assert ((o.double().cpu() - exact).abs() <= bound).all()


SIZES = {
    "one value": [1], "one vector": [5000], "odd": [1, 2, 3, 7, 8, 9, 15, 17, 2047, 2048, 2049, 4100, 1],
    "many small": [5 + i % 60 for i in range(700)], "large": [3_000_001, 64, 1_000_000],
    "with empty": [0, 10, 0, 0, 300, 0],
}


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)])
@pytest.mark.parametrize("sizes", SIZES)
def test_norm_and_clip(sizes, dtypes, norm_type):
    grads = _grads(SIZES[sizes], dtypes)
    dev = [g.to(DEV) for g in grads]
    want = ref.grad_norm(grads, norm_type)
    total = ops.grad_norm(dev, norm_type=norm_type)
    assert abs(total.item() - want.item()) <= 2.0**-23 * want.item()
    for max_norm in (want.item() * 0.25, want.item() * 2):
        inplace = [g.clone() for g in dev]
        total = ops.clip_grad_norm_(inplace, max_norm, norm_type=norm_type)
        _check(grads, max_norm, norm_type, total, inplace)
        out = [torch.full_like(g, 7.0, dtype=F32) for g in dev]
        total = ops.clip_grad_norm_(dev, max_norm, norm_type=norm_type, out=out)
        _check(grads, max_norm, norm_type, total, out)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, grads)), "out of place leaves the gradients"


@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_packed_views_at_odd_offsets(dtype, out_dtype):
    """Gradients that lie packed behind each other, at any element offset, and outputs at other offsets."""
    sizes = [3, 1000, 5, 4096, 1, 2500, 64]
    bucket = torch.cat(_grads(sizes, (dtype,), seed=1)).to(DEV)
    grads = list(bucket.split(sizes))
    memory = torch.full((sum(sizes) + 16,), 9.0, dtype=out_dtype, device=DEV)
    for shift in (0, 1, 4, 7):
        memory.fill_(9.0)
        out = list(memory[shift:shift + sum(sizes)].split(sizes))
        total = ops.clip_grad_norm_(grads, 0.5, out=out)
        _check([g.cpu() for g in grads], 0.5, 2.0, total, out)
        assert (memory[:shift] == 9).all() and (memory[shift + sum(sizes):] == 9).all()
    before = bucket.cpu()
    total = ops.clip_grad_norm_(grads, 0.5)
    _check(list(before.split(sizes)), 0.5, 2.0, total, grads)


@pytest.mark.parametrize("dtype, out_dtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F32, BF16)])
def test_more_than_the_caches_hold(dtype, out_dtype):
    """134 million bytes of gradients and outputs and more, in two launches' tables, packed at odd offsets."""
    sizes = [1 + 2 * i for i in range(170)] + [9_000_001, 31, 5_500_007] + [17] * 40 + [8_000_003]
    sizes += [13_000_009] if dtype != F32 or out_dtype != F32 else []
    if dtype != F32 and out_dtype != F32:
        sizes.append(9_000_013)
    assert sum(sizes) * (dtype.itemsize + out_dtype.itemsize) > 1 << 27
    bucket = torch.cat(_grads(sizes, (dtype,), seed=9)).to(DEV)
    grads, cpu = list(bucket.split(sizes)), list(bucket.cpu().split(sizes))
    memory = torch.full((sum(sizes) + 16,), 9.0, dtype=out_dtype, device=DEV)
    out = list(memory[3:3 + sum(sizes)].split(sizes))
    _check(cpu, 0.5, 2.0, ops.clip_grad_norm_(grads, 0.5, out=out), out)
    assert (memory[:3] == 9).all() and (memory[3 + sum(sizes):] == 9).all()
    assert torch.equal(bucket.cpu(), torch.cat(cpu))
    aligned = list(memory[:sum(sizes)].split(sizes))
    _check(cpu, 0.5, 2.0, ops.clip_grad_norm_(grads, 0.5, out=aligned), aligned)
    _check(cpu, 0.5, 2.0, ops.clip_grad_norm_(grads, 0.5), grads)


def test_layouts():
    """Dense tensors of any order are scaled in place; gaps of strided ones stay as they are."""
    g = torch.Generator().manual_seed(2)
    a = torch.randn(4, 8, 6, 10, generator=g)
    for view in (lambda t: t, lambda t: t.permute(0, 2, 3, 1), lambda t: t.to(memory_format=torch.channels_last),
                 lambda t: t[:, ::2], lambda t: t[..., 1:7], lambda t: t[0, 0, 0, 0]):
        base = a.clone().to(DEV)
        grad = view(base)
        before = grad.cpu().clone()
        rest = base.clone()
        total = ops.clip_grad_norm_([grad, torch.ones(3, device=DEV)], 0.25)
        _check([before.reshape(-1), torch.ones(3)], 0.25, 2.0, total, [grad.reshape(-1).cpu(), torch.ones(3) * float(
            ref.clip_scale(ref.grad_norm([before, torch.ones(3)]), 0.25))])
        if grad.numel() < base.numel() and grad.data_ptr() >= base.data_ptr() and view(rest).data_ptr() != rest.data_ptr():
            keep = torch.ones_like(base, dtype=torch.bool)
            view(keep)[...] = False
            assert torch.equal(base[keep], rest[keep])
        out = torch.empty_like(before, device=DEV).t() if before.ndim == 2 else torch.empty(before.shape, device=DEV)
        ops.clip_grad_norm_([view(rest)], 0.25, out=[out])
        scale = ref.clip_scale(ref.grad_norm([before]), 0.25)
        assert ((out.double().cpu() - before.double() * scale).abs() <= 2.0**-21 * before.double().abs()).all()


def test_unclipped_gradients_keep_their_bits():
    grads = [g.to(DEV) for g in _grads([1000, 33], (F32, BF16), seed=3)]
    before = [g.clone() for g in grads]
    ops.clip_grad_norm_(grads, 1e6)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_zero_gradients():
    grads = [torch.zeros(100, device=DEV), torch.zeros(7, device=DEV, dtype=BF16)]
    assert ops.clip_grad_norm_(grads, 1.0).item() == 0.0
    assert all((g == 0).all() for g in grads)


def test_extreme_magnitudes():
    """Squares past FP32's range at both ends."""
    for value in (1e30, 1e-30):
        grads = [torch.full((1000,), value, device=DEV), torch.full((24,), -value, device=DEV)]
        total = ops.grad_norm(grads)
        assert abs(total.item() / (value * 32) - 1) < 1e-6
    grads = [torch.full((1000,), 1e30, device=DEV)]
    ops.clip_grad_norm_(grads, 1.0)
    assert abs(grads[0].double().norm().item() - 1) < 1e-6


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nonfinite_gradients(bad, norm_type):
    for at in (0, 5, 2999):
        grads = [g.to(DEV) for g in _grads([3000, 40], (F32, BF16), seed=4)]
        grads[0][at] = bad
        before = [g.clone() for g in grads]
        with pytest.raises(RuntimeError, match="not finite"):
            ops.clip_grad_norm_(grads, 1.0, norm_type=norm_type, error_if_nonfinite=True)
        assert all(torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)) for a, b in zip(grads, before))
        total = ops.clip_grad_norm_(grads, 1.0, norm_type=norm_type)
        if math.isnan(bad):
            assert math.isnan(total.item()) and all(torch.isnan(g).all() for g in grads)
        else:
            assert total.item() == math.inf
            assert torch.isnan(grads[0][at]) and (grads[1] == 0).all()
            grads[0][at] = 0
            assert (grads[0] == 0).all()


def test_matches_torch():
    params = [torch.nn.Parameter(g.to(DEV)) for g in _grads([100, 3000, 7], (F32,), seed=5)]
    for p in params:
        p.grad = torch.randn_like(p)
    copies = [p.grad.clone() for p in params]
    want = torch.nn.utils.clip_grad_norm_(params, 1.0)
    got = ops.clip_grad_norm_(copies, 1.0)
    assert abs(got.item() - want.item()) <= 2.0**-20 * want.item()
    for c, p in zip(copies, params):
        assert ((c - p.grad).abs() <= 2.0**-20 * p.grad.abs()).all()


def test_a_tensor_past_32_bit_offsets():
    """One BF16 gradient of more than 2^31 bytes, in pieces of 2^30 elements, and a value in its last one."""
    n = 2**30 + 12345
    big = torch.zeros(n, dtype=BF16, device=DEV)
    big[3], big[2**30 - 1], big[2**30], big[n - 1] = 3.0, 4.0, 12.0, 84.0
    total = ops.clip_grad_norm_([big, torch.zeros(5, device=DEV)], 8.5)
    assert total.item() == 85.0
    got = big[[3, 2**30 - 1, 2**30, n - 1]].float().cpu()
    assert ((got - torch.tensor([0.3, 0.4, 1.2, 8.4])).abs() <= got * 2.0**-8).all()
    assert big.count_nonzero().item() == 4


def test_same_bits_every_time_and_versions():
    grads = [g.to(DEV) for g in _grads([100_000] * 30 + [7], (F32, BF16), seed=6)]
    first = ops.grad_norm(grads)
    out = [torch.empty_like(g) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            total = ops.clip_grad_norm_(grads, 0.5, out=out)
        side.synchronize()
        assert torch.equal(total, first)
    versions = [g._version for g in grads]
    ops.clip_grad_norm_(grads, 0.5)
    assert all(g._version == v + 1 for g, v in zip(grads, versions))
    assert all(torch.equal(a, b) for a, b in zip(grads, out))


def test_graph_capture():
    grads = [g.to(DEV) for g in _grads([5000, 64, 300_000], (F32,), seed=7)]
    out = [torch.empty_like(g) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.clip_grad_norm_(grads, 0.5, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = ops.clip_grad_norm_(grads, 0.5, out=out)
    for seed in range(3):
        for g, new in zip(grads, _grads([5000, 64, 300_000], (F32,), seed=20 + seed)):
            g.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.empty_like(g) for g in grads]
        assert torch.equal(total, ops.clip_grad_norm_(grads, 0.5, out=eager))
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals():
    g = torch.ones(10, device=DEV)
    for args, kwargs in [(([],), {}), (([g.double()],), {}), (([torch.ones(3)],), {}), (([g, torch.ones(3)],), {}),
                         (([g],), {"norm_type": 1.0})]:
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.grad_norm(*args, **kwargs)
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.clip_grad_norm_(*args, 1.0, **kwargs)
    for out in ([], [g, g], [torch.ones(11, device=DEV)], [torch.ones(10)], [g.long()]):
        with pytest.raises(NotImplementedError, match="no HIP impl"):
            ops.clip_grad_norm_([g], 1.0, out=out)
    with pytest.raises(ValueError):
        torch.ops.flashim_amd.grad_norm([g], 3.0)
    with pytest.raises(ValueError):
        torch.ops.flashim_amd.clip_grad_norm_out([g], [g, g], 1.0, 2.0)
