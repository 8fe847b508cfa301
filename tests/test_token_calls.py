"""The token operators' Python calls where no kernel runs: what follows a call
besides gradients (tangents, traces) goes through the autograd functions, and
strides that lead nowhere are no reason to refuse."""
from __future__ import annotations

import warnings

import pytest
import torch
from torch.autograd import forward_ad


@pytest.fixture
def attention(pkg, monkeypatch):
    """The module with its launches and the check for a GPU left out."""
    from bevfusion_triton_amd import attention

    monkeypatch.setattr(attention.P, 'require_gpu', lambda *t: None)
    monkeypatch.setattr(attention, '_run', lambda call, device, what: None)
    return attention


def operands():
    g = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(s, generator=g)
    return {'q': n(6, 4, 64), 'k': n(6, 2, 64), 'cache': n(6, 9, 2, 64), 'positions': torch.arange(6),
            'frequencies': torch.ones(32), 'starts': torch.tensor([0, 6]),
            'lengths': torch.tensor([1, 2, 3, 4, 5, 6])}


CALLS = {
    'norm_rotate': lambda a, t, q: a.norm_rotate(q, t['k'], t['positions'], t['frequencies'])[0],
    'attend_packed': lambda a, t, q: a.attend_packed(q, t['k'], t['k'], t['starts']),
    'attend_cached': lambda a, t, q: a.attend_cached(q, t['cache'], t['cache'], t['lengths']),
}


@pytest.mark.parametrize('name', CALLS)
def test_tangents_are_refused(attention, name):
    """A result without a tangent would stand for a derivative of zero."""
    t = operands()
    with forward_ad.dual_level():
        q = forward_ad.make_dual(t['q'], torch.ones_like(t['q']))
        with pytest.raises(NotImplementedError, match='jvp'):
            CALLS[name](attention, t, q)
    assert CALLS[name](attention, t, t['q']).shape == t['q'].shape


@pytest.mark.parametrize('name', CALLS)
def test_a_trace_records_the_call(attention, name):
    t = operands()
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')  # (sizes as constants)
        traced = torch.jit.trace(lambda q: CALLS[name](attention, t, q), (t['q'],),
                                 check_trace=False)
    assert '^_' in str(traced.graph) and 'aten::new_empty' not in str(traced.graph)


def odd_units(*shape, dtype=torch.float32):
    """Dimensions of one with an odd stride, the others dense, from an aligned
    start."""
    strides, at = [], 1
    for n in reversed(shape):
        strides.append(at if n > 1 else 259)
        at *= n
    return torch.zeros(at, dtype=dtype).as_strided(shape, strides[::-1])


def test_strides_of_single_entries(attention):
    """The stride of a dimension of one leads nowhere: no refusal for it, and
    no copy of a cache."""
    for shape in ((1, 4, 64), (6, 1, 64), (1, 1, 64)):
        for dtype in (torch.float32, torch.bfloat16):
            x = attention._aligned(odd_units(*shape, dtype=dtype))
            assert not any(s * x.element_size() % 16 for s in x.stride()[:2]), shape
    for shape in ((1, 9, 2, 64), (3, 1, 2, 64), (3, 9, 1, 64), (1, 1, 1, 64), (1, 2, 64), (5, 1, 64)):
        x = odd_units(*shape)
        y = attention._cache('k', x, len(shape))
        assert y.data_ptr() == x.data_ptr() and y.shape == x.shape
        assert not any(s % 4 for s in y.stride()[:-1]), shape
    with pytest.raises(ValueError, match='16 bytes'):
        attention._cache('k', torch.zeros(9 * 259).as_strided((9, 2, 64), (259, 64, 1)), 3)


def test_layer_of_the_meta_device(pkg):
    """A layer made without memory has its frequencies once it is given some."""
    args = (32, 4, 2, 32, (4, 6, 6))
    want = pkg.TokenAttention(*args, base=500.0).frequencies
    layer = pkg.TokenAttention(*args, base=500.0, device='meta').to(torch.bfloat16)
    assert layer.frequencies.is_meta
    assert torch.equal(layer.to_empty(device='cpu').frequencies, want)
    layer = pkg.TokenAttention(*args, base=500.0).to('meta')
    assert torch.equal(layer.to_empty(device='cpu').double().frequencies, want)


@pytest.mark.parametrize('heads', [(0, 2), (4, 0), (0, 0)])
def test_gradients_of_no_heads(attention, heads):
    t = operands()
    q, k = (torch.zeros((6, n, 64), requires_grad=True) for n in heads)
    out = attention.norm_rotate(q, k, t['positions'], t['frequencies'])
    for x, g in zip((q, k), torch.autograd.grad(out, (q, k), [torch.ones_like(x) for x in out])):
        assert g.shape == x.shape


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
def test_one_row_of_a_wide_pitch(pkg, cuda, dtype):
    """Single rows cut from rows of an odd pitch, and a gradient of that kind:
    the same bits as contiguous ones."""
    g = torch.Generator().manual_seed(1)
    rows = [torch.randn((5, 259), generator=g).to(cuda, dtype) for _ in range(4)]
    starts = torch.tensor([0, 1], device=cuda)
    odd = [r[:, :256].unflatten(1, (4, 64))[:1] for r in rows]
    results = []
    for q, k, v, dout in (odd, [x.clone(memory_format=torch.contiguous_format) for x in odd]):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = pkg.attend_packed(*leaves, starts)
        results.append((out, *torch.autograd.grad(out, leaves, dout)))
        with torch.no_grad():
            results[-1] += (pkg.attend_cached(q, k[None], v[None], starts[1:], k, v),)
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize('name', CALLS)
def test_a_trace_runs_on_other_inputs(pkg, cuda, name):
    t = {n: x.to(cuda) for n, x in operands().items()}
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')
        traced = torch.jit.trace(lambda q: CALLS[name](pkg, t, q), (t['q'],), check_trace=False)
    other = t['q'].flip(0).contiguous()
    want = CALLS[name](pkg, t, other)
    assert not torch.equal(want, CALLS[name](pkg, t, t['q']))
    for _ in range(4):  # (the executor optimises after the first runs)
        assert torch.equal(traced(other), want)


@pytest.mark.gpu
@pytest.mark.parametrize('norm', [False, True])
def test_no_heads_and_no_keys(pkg, cuda, norm):
    """q without heads, and gradients of one output alone: those of the other
    operand are what they are without it."""
    t = {n: x.to(cuda) for n, x in operands().items()}
    w = torch.linspace(0.5, 1.5, 64, device=cuda, requires_grad=True)
    weight = {'k_weight': w} if norm else {}
    args = t['positions'], t['frequencies']
    k = t['k'].requires_grad_(True)
    leaves = [k, w] if norm else [k]
    alone = pkg.norm_rotate(t['k'][:, :0], k, *args, **weight)[1]
    beside = pkg.norm_rotate(t['q'], k, *args, **weight)[1]
    assert torch.equal(alone, beside)
    g = torch.ones_like(alone)
    for a, b in zip(torch.autograd.grad(alone, leaves, g), torch.autograd.grad(beside, leaves, g)):
        # (sums of the weights' gradient are cut at other tokens)
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
