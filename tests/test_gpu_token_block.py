"""The block: a training step against the same block in 64 bits, 8-bit
checkpoints against the step without them, autocast, and answers token by token
against whole prompts, in the parameters' type and in 8-bit integers."""
from __future__ import annotations

import copy

import pytest
import torch

from oracle import block as ref
from oracle import tokens as attention_ref

pytestmark = pytest.mark.gpu

ARGS = (48, 4, 2, 32, (4, 6, 6), 88)


def randomise(block, seed):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n, p in block.named_parameters():
            if p.dim() == 1:
                p.copy_(1 + 0.3 * torch.randn(p.shape, generator=g))
    return block


def plain(block, x, positions, starts, causal, gates):
    """The block in 64 bits on the CPU, from the definitions; differentiable."""
    w = {n: p.detach().cpu().double().requires_grad_(True) for n, p in block.named_parameters()}
    a = block.attention
    hq, hk, d = a.q_heads, a.k_heads, a.head_dim

    def norm(t, name):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + block.eps) * w[name]

    rows = (norm(x, 'attention_norm') @ w['attention.qkv.weight'].T).unflatten(-1, (-1, d))
    q, k, v = rows.split((hq, hk, hk), -2)
    freq = a.frequencies.cpu()
    q, _ = attention_ref.norm_rotate(q, positions, freq, a.pairs, w['attention.q_norm'], a.eps)
    k, _ = attention_ref.norm_rotate(k, positions, freq, a.pairs, w['attention.k_norm'], a.eps)
    out = []
    for i, j in zip(starts[:-1], starts[1:]):
        limits = [t + 1 if causal else j - i for t in range(j - i)]
        out.append(torch.stack([attention_ref.attend_rows(
            q[i:j, h], k[i:j, h // (hq // hk)], v[i:j, h // (hq // hk)], limits,
            d ** -0.5)[0] @ v[i:j, h // (hq // hk)] for h in range(hq)], 1))
    y = torch.cat(out).flatten(1) @ w['attention.out.weight'].T
    x = x + gates[0] * w['attention_scale'] * norm(y, 'attention_out_norm')
    y = ref.gated(norm(x, 'gated_norm') @ w['up.weight'].T, block.activation) @ w['down.weight'].T
    return x + gates[1] * w['gated_scale'] * norm(y, 'gated_out_norm'), w


@pytest.mark.parametrize('activation', ['silu', 'gelu'])
def test_training_step(pkg, cuda, activation):
    torch.manual_seed(1)
    block = randomise(pkg.TokenBlock(*ARGS, activation=activation, device=cuda), 1)
    x, goal = torch.randn(75, 48), torch.randn(75, 48)
    positions, starts = torch.randint(0, 30, (75, 3)), [0, 31, 31, 75]
    gates = [torch.randn(3, 48), torch.randn(75, 48)]
    leaves = [t.to(cuda).requires_grad_(True) for t in (x, *gates)]
    y = block(leaves[0], positions.to(cuda), torch.tensor(starts, device=cuda), causal=True,
              gates=leaves[1:])
    (y * goal.to(cuda)).sum().backward()
    doubles = [t.double().requires_grad_(True) for t in (x, *gates)]
    want, w = plain(block, doubles[0], positions, starts, True,
                    (doubles[1].repeat_interleave(25, 0), doubles[2]))
    (want * goal.double()).sum().backward()
    # fp32 through four products of up to 128 terms and the operators between
    assert torch.allclose(y.detach().cpu().double(), want.detach(), rtol=1e-4, atol=1e-4)
    for n, p, g in [(n, p, w[n].grad) for n, p in block.named_parameters()] + [
            (i, a, b.grad) for i, (a, b) in enumerate(zip(leaves, doubles))]:
        scale = g.abs().max().item()
        assert torch.allclose(p.grad.cpu().double(), g, rtol=2e-3, atol=2e-4 * scale), n


def test_checkpoints_change_the_gradients_little(pkg, cuda):
    """The same results; gradients off by what the copies are: 2^-7 of a block's
    largest magnitude at most, in a few places on the way."""
    torch.manual_seed(2)
    block = randomise(pkg.TokenBlock(*ARGS, device=cuda), 2)
    packed = pkg.TokenBlock(*ARGS, checkpoint=8, device=cuda)
    packed.load_state_dict(block.state_dict())
    x, goal = torch.randn(90, 48, device=cuda), torch.randn(90, 48, device=cuda)
    positions = torch.randint(0, 30, (90, 3), device=cuda)
    starts = torch.tensor([0, 40, 90], device=cuda)
    results = []
    for b in (block, packed):
        leaf = x.clone().requires_grad_(True)
        y = b(leaf, positions, starts)
        y.backward(goal)
        results.append((y, {'x': leaf.grad, **{n: p.grad for n, p in b.named_parameters()}}))
    assert torch.equal(results[0][0], results[1][0])
    for n, g in results[0][1].items():
        off = (results[1][1][n] - g).norm() / g.norm()
        # normal values are off by 0.7% of their deviation; each gradient is a product of at most
        # a handful of such factors
        assert 0 < off < 0.05, (n, off.item())


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('checkpoint', [None, 8])
def test_autocast(pkg, cuda, dtype, checkpoint):
    """fp32 parameters and stream under autocast: the step of a block in 16 bits
    with the same values on an fp32 stream, gradients in fp32."""
    torch.manual_seed(3)
    block = randomise(pkg.TokenBlock(*ARGS, checkpoint=checkpoint, device=cuda), 3)
    with torch.no_grad():
        for p in block.parameters():
            p.copy_(p.to(dtype))
    half = pkg.TokenBlock(*ARGS, checkpoint=checkpoint, device=cuda, dtype=dtype)
    half.load_state_dict(block.state_dict())
    x, positions = torch.randn(60, 48, device=cuda), torch.randint(0, 30, (60, 3), device=cuda)
    starts = torch.tensor([0, 31, 60], device=cuda)
    with torch.autocast('cuda', dtype):
        y = block(x, positions, starts)
    want = half(x, positions, starts)
    assert y.dtype == want.dtype == torch.float32
    assert torch.equal(y, want)
    y.backward(torch.ones_like(y))
    for n, p in block.named_parameters():
        assert p.grad.dtype == torch.float32 and p.grad.isfinite().all(), n
    z = half(x.to(dtype), positions, starts)
    assert z.dtype == dtype and torch.allclose(z.float(), want, rtol=0.1, atol=0.1)


@pytest.mark.parametrize('new', [1, 3])
def test_steps_are_the_prompts_rows(pkg, cuda, new):
    """Each answer over a shared scene and its own cache is the end of a causal
    prompt of scene and answer, gates and all."""
    torch.manual_seed(4)
    block = randomise(pkg.TokenBlock(*ARGS, device=cuda), 4)
    scene, places = torch.randn(100, 48, device=cuda), torch.randint(0, 20, (100, 3), device=cuda)
    B, total = 3, 6
    x = torch.randn(B, total, 48, device=cuda)
    at = torch.arange(20, 20 + total, device=cuda)[None, :, None].expand(B, total, 3)
    gates = torch.randn(2, B, 48, device=cuda)
    cache = [torch.full((B, 9, 2, 32), float('nan'), device=cuda) for _ in range(2)]
    lengths = torch.zeros(B, dtype=torch.int32, device=cuda)
    prefix = block.scene(scene, places)
    got = torch.cat([block.step(x[:, i:i + new], at[:, i:i + new], *cache, lengths, prefix,
                                gates=gates) for i in range(0, total, new)], 1)
    for b in range(B):
        rows = [torch.cat((torch.ones(100, 48, device=cuda), g[b].expand(total, 48))) for g in gates]
        with torch.no_grad():
            whole = block(torch.cat((scene, x[b])), torch.cat((places, at[b])),
                          torch.tensor([0, 106], device=cuda), causal=True, gates=rows)
        # two fp32 results of the same sums in another order
        assert torch.allclose(got[b], whole[100:], rtol=1e-4, atol=1e-4)


def test_quantized(pkg, cuda):
    """8-bit products: near the block they are made of; steps are still the rows
    of prompts, bit for bit where tokens' codes are the same; no gradient."""
    torch.manual_seed(5)
    block = randomise(pkg.TokenBlock(*ARGS, device=cuda, dtype=torch.bfloat16), 5)
    served = copy.deepcopy(block).quantize()
    assert served.quantize() is served and isinstance(served.up, pkg.Int8Linear)
    x, positions = torch.randn(70, 48, device=cuda), torch.randint(0, 30, (70, 3), device=cuda)
    starts = torch.tensor([0, 70], device=cuda)
    with torch.no_grad():
        want, got = block(x, positions, starts), served(x, positions, starts)
    off = (got - want).norm() / (want - x).norm()
    # operands of every product off by 1 / 254 of their largest magnitude at most, evenly
    # distributed: under 1% of their deviations; four products and two norms
    assert 0 < off < 0.05, off.item()
    with pytest.raises(RuntimeError, match='no gradient'):
        served(x, positions, starts)
    cache = [torch.zeros((2, 5, 2, 32), device=cuda, dtype=torch.bfloat16) for _ in range(2)]
    lengths = torch.zeros(2, dtype=torch.int32, device=cuda)
    y = served.step(x[:2, None], positions[:2, None], *cache, lengths)
    for b in range(2):
        with torch.no_grad():
            one = served(x[b:b + 1], positions[b:b + 1], torch.tensor([0, 1], device=cuda))
        # (one token alone: the same codes; attention over one key in another kernel)
        assert torch.allclose(y[b], one, rtol=2 ** -6, atol=2 ** -6)


def test_graph_of_a_step(pkg, cuda):
    """A captured serving step, replayed between eager ones."""
    torch.manual_seed(6)
    block = pkg.TokenBlock(*ARGS, device=cuda, dtype=torch.bfloat16).quantize()
    x, at = torch.randn(3, 1, 48, device=cuda), torch.zeros((3, 1, 3), dtype=torch.int64, device=cuda)

    def fresh():
        return ([torch.zeros((3, 9, 2, 32), device=cuda, dtype=torch.bfloat16) for _ in range(2)],
                torch.zeros(3, dtype=torch.int32, device=cuda))

    (a, b), (c, d) = fresh(), fresh()
    block.step(x, at, *fresh()[0], fresh()[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = block.step(x, at, *a, b)
    for i in range(4):
        x.copy_(torch.randn_like(x))
        at.fill_(i)
        graph.replay()
        want = block.step(x, at, *c, d)
        assert torch.equal(y, want) and torch.equal(b, d), i
    assert b.tolist() == [4, 4, 4]
