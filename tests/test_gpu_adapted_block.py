"""Adapters of a gated block, trained beside the frozen block with ``optim.Muon`` through ``gated.train_step`` and then served for
many requests beside the quantized contraction."""

import pytest
import torch
import torch.nn.functional as F

from flashim_amd import gated, ops, optim
from oracle import train as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16
HALF_STEP = 2.0**-8


def _block(channels=64, hidden=160, groups=8, seed=0):
    return gated.GatedBlock(channels, hidden, groups, generator=torch.Generator().manual_seed(seed))


def _adapters(block, count=3, rank=8, seed=1, random_b=False):
    g = torch.Generator().manual_seed(seed)
    adapters = gated.Adapters(block, count, rank, scale=0.5, generator=g)
    if random_b:
        with torch.no_grad():
            adapters.b.copy_((torch.randn(adapters.b.shape, generator=g) * 0.2).to(BF16))
    return adapters


def _images(n, h=12, w=10, c=64, seed=2):
    return torch.randn(n, h, w, c, generator=torch.Generator().manual_seed(seed)).to(BF16).to(DEV)


def test_adapters_start_without_a_change():
    block = _block()
    x = _images(4)
    index = torch.tensor([0, 2, -1, 1], device=DEV)
    with torch.no_grad():
        want = block(x)
        assert torch.equal(gated.AdaptedGatedBlock(block, _adapters(block))(x, index), want)


def test_a_training_step_of_the_adapters_alone():
    """Gradients of the adapters against the formulas, the optimizer's step against the definition, the block untouched."""
    block = _block(seed=3)
    adapted = gated.AdaptedGatedBlock(block, _adapters(block, random_b=True))
    before = {n: p.detach().clone() for n, p in adapted.named_parameters()}
    x, index = _images(5, seed=4), torch.tensor([1, 1, 2, -1, 1], device=DEV)
    optimizer = optim.Muon(adapted.adapters.parameters(), lr=0.05, momentum=0.9, weight_decay=0.1)
    weight = torch.randn(x.shape, generator=torch.Generator().manual_seed(5)).to(BF16).to(DEV)
    loss, norm = gated.train_step(adapted, optimizer, lambda: (adapted(x, index).float() * weight.float()).sum(), max_norm=1e9)
    with torch.no_grad():
        hidden = block.hidden(x)
        base = x + F.linear(hidden, block.w_down, block.b_down)
    a, b = (before["adapters." + n].cpu() for n in "ab")
    want = ref.low_rank_adapters(base.cpu(), hidden.cpu(), a, b, index.cpu(), 0.5, weight.cpu())
    for name, p in (("a", adapted.adapters.a), ("b", adapted.adapters.b)):
        off = (p.grad.double().cpu() - want[name]).abs()
        assert (off <= want[name + "_error"] + HALF_STEP * (want[name].abs() + want[name + "_error"])).all(), name
        assert (p.grad[0] == 0).all()  # no image has adapter 0
        g = p.grad.cpu().double()  # the first step's update direction is (1 + momentum) times the gradient
        old, bounds = before["adapters." + name].cpu().double(), []
        step, factor = ref.orthogonalize(1.9 * g), 0.05 * max(1.0, p.shape[-2] / p.shape[-1]) ** 0.5
        bounds = torch.stack([torch.full(m.shape, ref.schulz_bound(1.9 * m)) for m in g])
        expect = old * (1 - 0.05 * 0.1) - factor * step
        off = (p.detach().double().cpu() - expect).abs()
        assert (off <= factor * bounds + HALF_STEP * expect.abs() + 2.0**-22 * old.abs()).all(), name
        torch.testing.assert_close(optimizer.state[p]["momentum"].cpu(), p.grad.cpu().float(), rtol=0, atol=0)
    for n, p in block.named_parameters():
        assert p.grad is None and torch.equal(p, before["block." + n]), n


def test_block_and_adapters_train_on():
    """Several steps of a whole block with Muon (matrices and vectors): finite, every parameter moves."""
    block = _block(seed=6)
    x, target = _images(2, seed=7), _images(2, seed=8).float()
    optimizer = optim.Muon(block.parameters(), lr=0.02, weight_decay=0.01)
    before = {n: p.detach().clone() for n, p in block.named_parameters()}
    losses = [gated.train_step(block, optimizer, lambda: F.mse_loss(block(x).float(), target), 1.0)[0] for _ in range(4)]
    assert all(torch.isfinite(v) for v in losses)
    for n, p in block.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n


@pytest.mark.parametrize("preset", ["int8", "mxfp8"])
def test_many_requests_beside_the_quantized_contraction(preset):
    block = _block(channels=128, hidden=512, groups=32, seed=9)
    x = _images(6, 9, 11, 128, seed=10)
    adapters = _adapters(block, count=4, rank=16, random_b=True)
    index = torch.tensor([3, 0, -1, 2, 0, 3], device=DEV, dtype=torch.int32)
    quantized = gated.QuantizedGatedBlock(block, preset, x)
    with torch.no_grad():
        plain, hidden = quantized(x), block.hidden(x)
    got = quantized(x, adapters, index)
    want = ref.low_rank_adapters(plain.cpu(), hidden.cpu(), adapters.a.detach().cpu(), adapters.b.detach().cpu(), index.cpu(), 0.5)
    off = (got.double().cpu() - want["out"]).abs()
    assert (off <= want["out_error"] + HALF_STEP * (want["out"].abs() + want["out_error"])).all()
    assert torch.equal(got[2], plain[2])
    with pytest.raises(ValueError):
        quantized(x, adapters)
    # one request at a time, as a server would without batching, gives the same values
    for i in range(6):
        one = adapters(plain[i:i + 1], hidden[i:i + 1], index[i:i + 1])
        assert torch.equal(one[0], got[i]), i


def test_optimizer_state_is_saved_and_loaded():
    block, other = _block(seed=11), _block(seed=11)
    x, target = _images(2, seed=12), _images(2, seed=13).float()
    first, second = (optim.Muon(b.parameters(), lr=0.03) for b in (block, other))
    gated.train_step(block, first, lambda: F.mse_loss(block(x).float(), target), 1.0)
    other.load_state_dict(block.state_dict())
    second.load_state_dict(first.state_dict())
    for p, q in zip(block.parameters(), other.parameters()):
        for key, value in first.state[p].items():
            assert second.state[q][key].dtype == value.dtype and torch.equal(second.state[q][key], value)
            assert second.state[q][key].data_ptr() != value.data_ptr()
    for b, o in ((block, first), (other, second)):
        gated.train_step(b, o, lambda: F.mse_loss(b(x).float(), target), 1.0)
    assert all(torch.equal(p, q) for p, q in zip(block.parameters(), other.parameters()))


def test_compiled_adapted_block_equals_eager():
    block = _block(seed=14)
    adapted = gated.AdaptedGatedBlock(block, _adapters(block, random_b=True))
    x, index = _images(3, seed=15), torch.tensor([2, -1, 0], device=DEV)
    d = torch.randn(3, 12, 10, 64, generator=torch.Generator().manual_seed(16)).to(BF16).to(DEV)
    torch._dynamo.reset()

    def run(base, hidden):
        return ops.low_rank_adapters(base, hidden, adapted.adapters.a, adapted.adapters.b, index, scale=0.5)

    with torch.no_grad():
        hidden = block.hidden(x)
    leaves = [adapted.adapters.a, adapted.adapters.b]
    want = run(x, hidden)
    got = torch.compile(run, fullgraph=True)(x, hidden)
    assert torch.equal(got, want)
    for u, v in zip(torch.autograd.grad(got, leaves, d), torch.autograd.grad(want, leaves, d)):
        assert torch.equal(u, v)


def test_compiled_step_equals_eager():
    g = torch.Generator().manual_seed(17)
    tensors = [[torch.randn(s, generator=g).to(DEV) for s in ((64, 160), (200, 70))] for _ in range(3)]

    def step(params, grads, momenta):
        ops.muon_step_(params, grads, momenta, lr=0.1, weight_decay=0.1)
        return ops.orthogonalize(grads[0])

    copies = [[[t.clone() for t in ts] for ts in tensors] for _ in range(2)]
    torch._dynamo.reset()
    want, got = step(*copies[0]), torch.compile(step, fullgraph=True)(*copies[1])
    assert torch.equal(want, got)
    for a, b in zip(copies[0], copies[1]):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    assert not torch.equal(copies[0][0][0], tensors[0][0])


def test_captured_optimizer_steps_equal_eager_ones():
    """Matrices and vectors: replays count AdamW's steps, and start from no zeros."""
    block, other = _block(seed=17), _block(seed=17)
    captured, eager = (optim.Muon(b.parameters(), lr=0.03, weight_decay=0.1, capturable=True) for b in (block, other))

    def gradients(seed):
        g = torch.Generator().manual_seed(seed)
        for p, q in zip(block.parameters(), other.parameters()):
            new = torch.randn(p.shape, generator=g).to(p)
            for t in (p, q):
                if t.grad is None:
                    t.grad = torch.empty_like(t)
                t.grad.copy_(new)

    gradients(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured.step()
    torch.cuda.current_stream().wait_stream(side)
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for seed in range(1, 4):
        gradients(seed)
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        for p, q in zip(block.parameters(), other.parameters()):
            assert torch.equal(p, q)
            assert all(torch.equal(captured.state[p][k], v) for k, v in eager.state[q].items())


@pytest.mark.parametrize("state", [False, True])
def test_captures_that_would_replay_wrong_steps_are_refused(state):
    block = _block(seed=18)
    optimizer = optim.Muon(block.parameters())
    for p in block.parameters():
        p.grad = torch.ones_like(p)
    if state:
        optimizer.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable" if state else "first step"), torch.cuda.graph(graph):
        optimizer.step()
    optimizer.step()
    assert all(torch.isfinite(p).all() for p in block.parameters())
