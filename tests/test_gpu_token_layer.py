"""The token operators together: the layer's training step against the same
layer in 64 bits, and answers token by token over a shared scene against whole
causal prompts."""
from __future__ import annotations

import importlib.util

import pytest
import torch

from conftest import ROOT
from oracle import tokens as ref

pytestmark = pytest.mark.gpu


def _plain(layer, x, positions, starts, causal):
    """The layer in 64 bits on the CPU, from the definitions; differentiable."""
    w = {n: p.detach().cpu().double().requires_grad_(True) for n, p in layer.named_parameters()}
    hq, hk, d = layer.q_heads, layer.k_heads, layer.head_dim
    rows = (x @ w['qkv.weight'].T).unflatten(-1, (-1, d))
    q, k, v = rows.split((hq, hk, hk), -2)
    freq = layer.frequencies.cpu()
    q, _ = ref.norm_rotate(q, positions, freq, layer.pairs, w['q_norm'], layer.eps)
    k, _ = ref.norm_rotate(k, positions, freq, layer.pairs, w['k_norm'], layer.eps)
    out = []
    for a, b in zip(starts[:-1], starts[1:]):
        limits = [i + 1 if causal else b - a for i in range(b - a)]
        heads = [ref.attend_rows(q[a:b, h], k[a:b, h // (hq // hk)], v[a:b, h // (hq // hk)],
                                 limits, d ** -0.5)[0] @ v[a:b, h // (hq // hk)]
                 for h in range(hq)]
        out.append(torch.stack(heads, 1))
    return torch.cat(out).flatten(1) @ w['out.weight'].T, w


@pytest.mark.parametrize('causal', [False, True])
def test_training_step(pkg, cuda, causal):
    torch.manual_seed(1)
    layer = pkg.TokenAttention(40, 4, 2, 32, (4, 6, 6), device=cuda)
    x = torch.randn(75, 40)
    positions, starts = torch.randint(0, 30, (75, 3)), [0, 31, 31, 75]
    y = layer(x.to(cuda), positions.to(cuda), torch.tensor(starts, device=cuda), causal=causal)
    goal = torch.randn(75, 40)
    (y * goal.to(cuda)).sum().backward()
    want, w = _plain(layer, x.double(), positions, starts, causal)
    (want * goal.double()).sum().backward()
    # fp32 through two products of 40 and 128 terms and the operators between
    assert torch.allclose(y.detach().cpu().double(), want.detach(), rtol=1e-4, atol=1e-5)
    for n, p in layer.named_parameters():
        scale = w[n].grad.abs().max().item()
        assert torch.allclose(p.grad.cpu().double(), w[n].grad, rtol=1e-3, atol=1e-4 * scale), n


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_autocast(pkg, cuda, dtype):
    """fp32 parameters under autocast: the training step of a layer in 16 bits
    with the same values, its gradients in fp32; and single tokens."""
    torch.manual_seed(3)
    layer = pkg.TokenAttention(32, 4, 2, 32, (4, 6, 6), device=cuda)
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_((p * 1.25 + 0.01).to(dtype))
    half = pkg.TokenAttention(32, 4, 2, 32, (4, 6, 6), device=cuda, dtype=dtype)
    half.load_state_dict(layer.state_dict())
    x, positions = torch.randn(75, 32, device=cuda), torch.randint(0, 30, (75, 3), device=cuda)
    starts = torch.tensor([0, 31, 75], device=cuda)
    with torch.autocast('cuda', dtype):
        y = layer(x, positions, starts, causal=True)
    want = half(x.to(dtype), positions, starts, causal=True)
    assert y.dtype == dtype and torch.equal(y, want)
    goal = torch.randn_like(want)
    y.backward(goal)
    want.backward(goal)
    for (n, p), h in zip(layer.named_parameters(), half.parameters()):
        assert p.grad.dtype == torch.float32 and torch.equal(p.grad, h.grad.float()), n
    cache = [torch.zeros((2, 5, 2, 32), device=cuda, dtype=dtype) for _ in range(4)]
    lengths = torch.zeros((2, 2), dtype=torch.int32, device=cuda)
    with torch.autocast('cuda', dtype):
        y = layer.step(x[:2, None], positions[:2, None], *cache[:2], lengths[0])
    assert torch.equal(y, half.step(x[:2, None].to(dtype), positions[:2, None], *cache[2:],
                                    lengths[1]))


@pytest.mark.parametrize('new', [1, 3])
def test_steps_are_the_prompts_rows(pkg, cuda, new):
    """Each answer, `new` tokens at a time over the shared scene and its own
    cache, is the end of a causal prompt of scene and answer."""
    torch.manual_seed(2)
    layer = pkg.TokenAttention(32, 4, 2, 64, (8, 12, 12), device=cuda)
    scene, places = torch.randn(150, 32, device=cuda), torch.randint(0, 20, (150, 3), device=cuda)
    B, total = 3, 6
    x = torch.randn(B, total, 32, device=cuda)
    at = torch.arange(20, 20 + total, device=cuda)[None, :, None].expand(B, total, 3)
    cache = [torch.full((B, 9, 2, 64), float('nan'), device=cuda) for _ in range(2)]
    lengths = torch.zeros(B, dtype=torch.int32, device=cuda)
    prefix = layer.scene(scene, places)
    got = torch.cat([layer.step(x[:, i:i + new], at[:, i:i + new], *cache, lengths, prefix)
                     for i in range(0, total, new)], 1)
    assert lengths.tolist() == [total] * B
    for b in range(B):
        with torch.no_grad():
            whole = layer(torch.cat((scene, x[b])), torch.cat((places, at[b])),
                          torch.tensor([0, 156], device=cuda), causal=True)
        # two fp32 results of the same sums in another order
        assert torch.allclose(got[b], whole[150:], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize('kind', [torch.int32, torch.int64])
def test_steps_past_the_capacity_stay_in_the_cache(pkg, cuda, kind):
    """A full cache takes new tokens in its last slots and no others."""
    torch.manual_seed(4)
    layer = pkg.TokenAttention(32, 4, 2, 64, (8, 12, 12), device=cuda)
    x, at = torch.randn(3, 2, 32, device=cuda), torch.full((3, 2, 3), 7, device=cuda)
    wide = [torch.zeros((3, 9, 2, 64), device=cuda) for _ in range(2)]
    cache = [w[:, 2:7] for w in wide]  # 5 slots amid others
    lengths = torch.tensor([4, 1, 5], device=cuda, dtype=kind)
    layer.step(x, at, *cache, lengths)
    assert lengths.tolist() == [5, 3, 5]
    for w in wide:
        used = w.flatten(2).abs().sum(-1) > 0
        assert used.nonzero().tolist() == [[0, 5], [0, 6], [1, 3], [1, 4], [2, 5], [2, 6]]
    with pytest.raises(ValueError, match='do not fit'):
        layer.step(torch.randn(3, 6, 32, device=cuda), at, *cache, lengths)


def test_example_runs(pkg, cuda, capsys):
    spec = importlib.util.spec_from_file_location('bev_tokens', ROOT / 'examples' /
                                                  'bev_tokens.py')
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.main(questions=2, answer=3)
    assert bool(torch.isfinite(r['loss'])) and 'trained on' in capsys.readouterr().out
    layer, (scene, places) = r['layer'], r['scene']
    n, answer = len(scene), r['asked'].shape[1]
    for b in range(2):
        at = torch.full((answer, 3), r['first'], device=cuda) + torch.arange(
            answer, device=cuda)[:, None]
        with torch.no_grad():
            whole = layer(torch.cat((scene, r['asked'][b])), torch.cat((places, at)),
                          torch.tensor([0, n + answer], device=cuda), causal=True)
        want = (r['asked'][b] + whole[n:]).float()
        # bf16: keys and outputs rounded at the same places, sums in another order
        assert torch.allclose(r['given'][b].float(), want, rtol=2 ** -6, atol=2 ** -6)
