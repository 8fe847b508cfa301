"""The token operators' Python calls where no kernel runs: what follows a call
besides gradients (tangents, traces) goes through the autograd functions."""
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
