"""What autograd asks of the block operators besides right numbers: saved
tensors that hooks take away or that change in place, a graph that is used
twice, inputs that need no gradient, gradients of any layout, and refusals."""
from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint as recompute


def leaves(cuda, rows=24, width=64):
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(s, generator=g).to(cuda, torch.bfloat16)
    return {'x': n(rows, width), 'update': n(rows, width), 'w': n(width), 'gate': n(2, width),
            'linear': n(40, width), 'bias': n(40)}


CALLS = {
    'residual_norm': lambda pkg, t, kept: pkg.residual_norm(
        t['x'], t['update'], update_weight=t['w'], scale=t['w'], gate=t['gate'], weight=t['w'],
        checkpoint=kept),
    'norm': lambda pkg, t, kept: pkg.residual_norm(t['x'], weight=t['w'], checkpoint=kept)[1:],
    'gated_activation': lambda pkg, t, kept: (pkg.gated_activation(t['x'], checkpoint=kept),),
    'checkpoint_linear': lambda pkg, t, kept: (pkg.checkpoint_linear(t['x'], t['linear'], t['bias']),),
}
every = pytest.mark.parametrize('name', CALLS)


def test_a_missing_library_is_an_error(pkg, monkeypatch, tmp_path):
    from bevfusion_triton_amd import _lib

    assert _lib.block_calls() is _lib.block_calls()
    monkeypatch.setattr(_lib, '_block_module', None)
    monkeypatch.setattr(_lib, 'BLOCK_CALLS_PATH', tmp_path / '_block_calls.so')
    with pytest.raises(_lib.LibraryNotBuilt, match='missing'):
        _lib.block_calls()
    (tmp_path / '_block_calls.so').write_bytes(b'no library')
    with pytest.raises(_lib.LibraryNotBuilt, match='cannot load'):
        _lib.block_calls()


@pytest.mark.gpu
def test_a_refusal_below_is_the_package_s_error(pkg, cuda):
    """Of what the Python call has checked before."""
    from bevfusion_triton_amd import _lib

    x = torch.zeros(4, 8, device=cuda)
    with pytest.raises(_lib.BevPoolError, match='unknown activation 7'):
        _lib.block_calls().gated_activation(x, 7, False, False)
    with pytest.raises(_lib.BevPoolError, match='neither'):
        _lib.block_calls().residual_norm(x, None, None, None, None, None, x.dtype, 0.0, False, False)


def grads(pkg, name, t, kept=None, douts=None, **more):
    t = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    outs = CALLS[name](pkg, t, kept)
    douts = [torch.ones_like(o) for o in outs] if douts is None else douts
    return torch.autograd.grad(outs, list(t.values()), douts, allow_unused=True, **more)


def same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert (x is None) == (y is None) and (x is None or torch.equal(x, y))


@pytest.mark.gpu
@every
@pytest.mark.parametrize('kept', [None, 8])
def test_saved_tensors(pkg, cuda, name, kept):
    """Kept on the host between the passes, or made again."""
    t = leaves(cuda)
    want = grads(pkg, name, t, kept)
    with torch.autograd.graph.save_on_cpu():
        u = {n: v.detach().requires_grad_(True) for n, v in t.items()}
        outs = CALLS[name](pkg, u, kept)
    same(torch.autograd.grad(outs, list(u.values()), [torch.ones_like(o) for o in outs],
                             allow_unused=True), want)
    u = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    outs = recompute(lambda *a: CALLS[name](pkg, dict(zip(u, a)), kept), *u.values(),
                     use_reentrant=False)
    same(torch.autograd.grad(outs, list(u.values()), [torch.ones_like(o) for o in outs],
                             allow_unused=True), want)


@pytest.mark.gpu
@every
def test_a_graph_used_twice(pkg, cuda, name):
    t = {n: v.requires_grad_(True) for n, v in leaves(cuda).items()}
    outs = CALLS[name](pkg, t, 8)
    douts = [torch.ones_like(o) for o in outs]
    ask = lambda **k: torch.autograd.grad(outs, list(t.values()), douts, allow_unused=True, **k)
    same(ask(retain_graph=True), ask())
    with pytest.raises(RuntimeError, match='second time'):
        ask()


@pytest.mark.gpu
@every
def test_changes_in_place(pkg, cuda, name):
    """Of what was saved: refused.  Of a result: as of any other."""
    t = {n: v.requires_grad_(True) for n, v in leaves(cuda).items()}
    x = t['x'] * 1
    outs = CALLS[name](pkg, dict(t, x=x), None)
    if name != 'checkpoint_linear':  # (that keeps a copy)
        with torch.no_grad():
            x.add_(1)
        with pytest.raises(RuntimeError, match='modified by an inplace'):
            outs[-1].sum().backward()
    want = grads(pkg, name, t, 8, [torch.full_like(o, 2.0) for o in outs])
    outs = CALLS[name](pkg, t, 8)
    got = torch.autograd.grad([o.mul_(2) for o in outs], list(t.values()),
                              [torch.ones_like(o) for o in outs], allow_unused=True)
    same(got, want)


@pytest.mark.gpu
@every
def test_inputs_without_a_gradient(pkg, cuda, name):
    t = leaves(cuda)
    want = dict(zip(t, grads(pkg, name, t, 8)))
    for n in t:
        if want[n] is None:
            continue
        one = dict(t, **{n: t[n].detach().requires_grad_(True)})
        outs = CALLS[name](pkg, one, 8)
        got, = torch.autograd.grad(outs, one[n], [torch.ones_like(o) for o in outs])
        assert torch.equal(got, want[n]), n


@pytest.mark.gpu
@every
def test_gradients_of_any_layout(pkg, cuda, name):
    """Broadcast, transposed and strided ones, ones of a leaf that collects."""
    t = leaves(cuda)
    outs = CALLS[name](pkg, t, 8)
    for lay in (lambda d: d[:1, :1].expand(d.shape), lambda d: d.t().contiguous().t(),
                lambda d: torch.stack((d, d), 2)[..., 0]):
        douts = [lay(torch.randn_like(o)) for o in outs]
        same(grads(pkg, name, t, 8, douts), grads(pkg, name, t, 8, [d.contiguous() for d in douts]))
    t = {n: v.requires_grad_(True) for n, v in t.items()}
    for _ in range(2):
        sum(o.sum() for o in CALLS[name](pkg, t, 8)).backward()
    for v, g in zip(t.values(), grads(pkg, name, t, 8)):
        assert (v.grad is None) == (g is None) and (g is None or torch.equal(v.grad, 2 * g))


@pytest.mark.gpu
@every
def test_refusals(pkg, cuda, name):
    """Of second derivatives, also where the gradient itself needs none, and of
    transformed functions."""
    t = {n: v.requires_grad_(True) for n, v in leaves(cuda).items()}
    outs = CALLS[name](pkg, t, None)
    g = torch.autograd.grad(outs, t['x'], [torch.ones_like(o) for o in outs], create_graph=True)[0]
    with pytest.raises(RuntimeError, match='second derivative'):
        (g.float().sum() + t['x'].float().sum()).backward()
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: CALLS[name](pkg, dict(t, x=x), None)[0].float().sum())(t['x'].detach())
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: CALLS[name](pkg, dict(t, x=x), None)[-1])(t['x'].detach()[None])


@pytest.mark.gpu
@every
def test_a_trace_has_gradients(pkg, cuda, name):
    t = leaves(cuda)
    import warnings

    with warnings.catch_warnings():
        warnings.simplefilter('ignore')
        traced = torch.jit.trace(lambda x: CALLS[name](pkg, dict(t, x=x), 8)[-1], (t['x'],),
                                 check_trace=False)
    x = t['x'].detach().requires_grad_(True)
    out = traced(x)
    got, = torch.autograd.grad(out, x, torch.ones_like(out))
    y = t['x'].detach().requires_grad_(True)
    out = CALLS[name](pkg, dict(t, x=y), 8)[-1]
    want, = torch.autograd.grad(out, y, torch.ones_like(out))
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_two_threads(pkg, cuda):
    """Steps of two threads at once, each on a stream of its own."""
    from concurrent.futures import ThreadPoolExecutor

    t = leaves(cuda, 3000, 512)
    want = {n: grads(pkg, n, t, 8) for n in CALLS}
    codes = pkg.quantize_weight(t['linear'])
    product = pkg.linear_int8(t['x'], *codes)
    torch.cuda.synchronize()

    def work(_):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = {n: grads(pkg, n, t, 8) for n in CALLS}
                y = pkg.linear_int8(t['x'], *codes)
            torch.cuda.current_stream().synchronize()
        return got, y

    with ThreadPoolExecutor(2) as pool:
        for got, y in pool.map(work, range(2)):
            assert torch.equal(y, product)
            for n in CALLS:
                same(got[n], want[n])


@pytest.mark.gpu
@every
@pytest.mark.parametrize('kept', [None, 8])
def test_saved_tensors_in_another_layout(pkg, cuda, name, kept):
    """A hook may give a saved tensor back as it likes it laid out."""
    def lay(t):
        if t.dim() == 2:
            return t.t().contiguous().t()
        return torch.stack((t, torch.zeros_like(t)), 1)[:, 0]

    t = leaves(cuda)
    want = grads(pkg, name, t, kept)
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s, lay):
        got = grads(pkg, name, t, kept)
    same(got, want)


@pytest.mark.gpu
@every
@pytest.mark.parametrize('kept', [None, 8])
def test_what_does_not_fit_is_refused(pkg, cuda, name, kept):
    """Saved tensors of another size, type or place, and gradients that a caller
    of a node gives: before any kernel reads them."""
    t = leaves(cuda)
    for change in (lambda s: s[..., :-1], lambda s: s[:-1], lambda s: s.double(), lambda s: s.cpu()):
        u = {n: v.detach().requires_grad_(True) for n, v in t.items()}
        with torch.autograd.graph.saved_tensors_hooks(lambda s: s, change):
            outs = CALLS[name](pkg, u, kept)
            with pytest.raises(RuntimeError):
                torch.autograd.grad(outs, list(u.values()), [torch.ones_like(o) for o in outs],
                                    allow_unused=True)
    for n in t:
        t[n].requires_grad_(True)
    out = CALLS[name](pkg, t, kept)[-1]
    node, nothing = out.grad_fn, [None] * (name in ('residual_norm', 'norm'))
    for d in (torch.ones_like(out)[:-1], torch.ones_like(out)[:, :-1], torch.ones_like(out).cpu(),
              torch.ones_like(out)[0]):
        with pytest.raises(RuntimeError):
            node(*nothing, d)
    torch.cuda.synchronize()
    douts = [torch.zeros_like(o) for o in CALLS[name](pkg, t, kept)[:-1]] + [torch.ones_like(out)]
    got = node(*nothing, douts[-1])
    got = got if isinstance(got, torch.Tensor) else got[0]  # (a node of one input)
    assert torch.equal(got, grads(pkg, name, t, kept, douts)[0])


@pytest.mark.gpu
def test_a_refusal_in_a_backward_pass_is_the_package_s_error(pkg, cuda):
    """As in the forward, through the autograd engine and from the node."""
    from bevfusion_triton_amd import _lib

    t = {n: v.requires_grad_(True) for n, v in leaves(cuda).items()}
    more = lambda s: s[:1].repeat(5, 1) if s.shape == t['gate'].shape else s
    with torch.autograd.graph.saved_tensors_hooks(lambda s: s, more):
        out = CALLS['residual_norm'](pkg, t, None)[0]
        with pytest.raises(_lib.BevPoolError, match='do not divide'):
            out.grad_fn(torch.ones_like(out), None)
        with pytest.raises(_lib.BevPoolError, match='do not divide'):
            out.sum().backward()
