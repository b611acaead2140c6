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
