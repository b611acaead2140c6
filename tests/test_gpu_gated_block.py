"""The gated block (``flashim_amd.gated``) end to end: gradients and a training step against float64 autograd of the same
block, torch.compile, and the quantized block against the float one.

The block rounds to BF16 (half a unit 2^-8) at six places a pass; independent roundings of 2^-8 / sqrt(3) each add up to
2^-8 sqrt(6 / 3) relative to the tensor's norm, and the bounds below allow four times that, 0.022."""

import pytest
import torch
import torch.nn.functional as F

from flashim_amd import gated, ops
from oracle import reference, train as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOUND = 0.022


def _block(channels=64, hidden=160, groups=8, seed=0):
    return gated.GatedBlock(channels, hidden, groups, generator=torch.Generator().manual_seed(seed))


def _data(shape, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(torch.bfloat16), torch.randn(shape, generator=g)


def _float64(block, x):
    p = {n: v.detach().cpu().double().requires_grad_() for n, v in block.named_parameters()}
    c = x.shape[-1]
    rows = x.double().reshape(x.shape[0], -1, c).transpose(1, 2)
    n = F.group_norm(rows, block.groups, p["norm_weight"], p["norm_bias"], 1e-5).transpose(1, 2).reshape(x.shape)
    h = F.silu(F.linear(n, p["w_gate"], p["b_gate"])) * F.linear(n, p["w_up"], p["b_up"])
    return p, x.double() + F.linear(h, p["w_down"], p["b_down"])


def _rel(a, b):
    return ((a.double().cpu() - b).norm() / b.norm()).item()


def test_gradients_and_clip_of_a_training_step():
    block = _block()
    x, target = _data((2, 30, 37, 64))
    params = {n: v.detach().cpu().double().clone() for n, v in block.named_parameters()}
    p, y = _float64(block, x)
    ((y - target.double()) ** 2).mean().backward()
    norm = ref.grad_norm([v.grad for v in p.values()])
    optimizer = torch.optim.SGD(block.parameters(), lr=1.0)
    value, got = gated.train_step(block, optimizer, lambda: F.mse_loss(block(x.to(DEV)).float(), target.to(DEV)),
                                  max_norm=norm.item() / 3)
    assert abs(got.item() / norm.item() - 1) < BOUND
    assert abs(value.item() / ((y - target.double()) ** 2).mean().item() - 1) < BOUND
    for n, v in block.named_parameters():
        assert _rel(v.grad, p[n].grad / 3) < BOUND, n
        step = p[n].grad / 3  # the parameter's own rounding on top
        moved = (v.detach().cpu().double() - (params[n] - step)).norm()
        assert moved < BOUND * step.norm() + 2.0**-8 * params[n].norm(), n


def test_training_lowers_the_loss():
    block = _block(seed=2)
    x, _ = _data((2, 24, 24, 64), seed=3)
    teacher = _block(seed=4)
    with torch.no_grad():
        target = teacher(x.to(DEV)).float()
    optimizer = torch.optim.AdamW(block.parameters(), lr=5e-3)
    losses = [gated.train_step(block, optimizer, lambda: F.mse_loss(block(x.to(DEV)).float(), target), 1.0)[0].item()
              for _ in range(60)]
    assert losses[-1] < 0.5 * losses[0], losses[::10]


@pytest.mark.parametrize("preset", ["int8", "mxfp8"])
def test_quantized_block(preset):
    """INT8: bit-exact with the oracle's convolution of the hidden map's codes. MXFP8: the float64 product of the codes; a sum
    of 512 FP32 products and the bias lie within 513 FP32 units (2^-24) of their terms' magnitudes, the contraction and the
    sum with the residual are then each rounded to BF16 (2^-8, half a unit in the last of 8 bits)."""
    block = _block(channels=128, hidden=512, groups=32, seed=5)
    x = _data((1, 40, 50, 128), seed=6)[0].to(DEV)
    quantized = gated.QuantizedGatedBlock(block, preset, x)
    with torch.no_grad():
        hidden, scale = block.hidden(x).cpu().float(), quantized.scale.cpu()
    got, bias = quantized(x).cpu(), block.b_down.detach().cpu()
    if preset == "int8":
        codes, w_scale = (t.cpu() for t in quantized.weight)
        want = reference.int8_conv2d(reference.quantize_int8(hidden, scale), codes, scale, w_scale.reshape(-1), bias,
                                     1, 1, 1, 1, 0, 0, 1, 1, residual=x.cpu())
        assert torch.equal(got, want)
        return

    def blocks(codes, exponent):
        return torch.ldexp(codes.double().reshape(-1, 512 // 32, 32), exponent.int()[..., None]).reshape(-1, 512)

    a = blocks(reference.quantize_mxfp8(hidden, scale), scale)
    weight = blocks(quantized.weight.values.cpu(), quantized.weight.scale_exponent.cpu())
    bias, rows = bias.double(), x.cpu().double().reshape(-1, 128)
    conv, terms = a @ weight.t() + bias, a.abs() @ weight.abs().t() + bias.abs()
    error = (got.double().reshape(-1, 128) - (conv + rows)).abs()
    bound = 2.0**-8 * (1 + 2.0**-7) * (conv.abs() + (conv + rows).abs()) + 1.01 * 513 * 2.0**-24 * terms
    assert (error <= bound).all(), (error / bound).max()


def test_compiled_block_equals_eager():
    block = _block(seed=7)
    x = _data((2, 20, 21, 64), seed=8)[0].to(DEV)
    torch._dynamo.reset()
    compiled = torch.compile(block.hidden, fullgraph=True)
    d_hidden = torch.randn(2, 20, 21, 160, device=DEV, generator=torch.Generator(device=DEV).manual_seed(0)).to(torch.bfloat16)
    leaves = [p for n, p in block.named_parameters() if "down" not in n]
    want_out = block.hidden(x)
    want = torch.autograd.grad(want_out, leaves, d_hidden)
    got_out = compiled(x)
    got = torch.autograd.grad(got_out, leaves, d_hidden)
    assert torch.equal(got_out, want_out)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_compiled_clip_equals_eager():
    grads = [torch.randn(n, device=DEV) for n in (100, 4097, 3)]
    for out in (False, True):
        def clip(tensors, to):
            return ops.clip_grad_norm_(tensors, 0.5, out=to) if out else ops.clip_grad_norm_(tensors, 0.5)

        a, b = [g.clone() for g in grads], [g.clone() for g in grads]
        ta, tb = [torch.zeros_like(g) for g in grads], [torch.zeros_like(g) for g in grads]
        torch._dynamo.reset()
        want, got = clip(a, ta), torch.compile(clip, fullgraph=True)(b, tb)
        assert torch.equal(want, got)
        assert all(torch.equal(x, y) for x, y in zip(a + ta, b + tb))
