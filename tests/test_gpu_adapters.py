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
