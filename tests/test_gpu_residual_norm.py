"""residual_norm against its definition in 64 bits: types, widths that end
inside a chunk, a lane group and a block, gates of every kind, what may be left
out, checkpoints, strides, and gradients (of the formula and of differences)."""
from __future__ import annotations

import pytest
import torch

from oracle import block as ref

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16),
         (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16),
         (torch.float32, torch.bfloat16)]
NAMES = ('x', 'update', 'update_weight', 'scale', 'gate', 'weight')
EPS = 1e-6


def make(rows, width, x_dtype, dtype, seed, gate=None, parts=NAMES):
    """gate: None, 'element' or a number of rows."""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)
    case = {'x': (2 * n(rows, width)).to(x_dtype), 'update': (0.7 * n(rows, width)).to(dtype),
            'update_weight': (1 + 0.3 * n(width)).to(dtype), 'scale': (0.5 + 0.2 * n(width)).to(dtype),
            'weight': (1 + 0.3 * n(width)).to(dtype)}
    if gate is not None:
        case['gate'] = n(rows if gate == 'element' else gate, width).to(dtype)
    grads = {'sum': n(rows, width).to(x_dtype), 'normed': n(rows, width).to(dtype)}
    return {k: v for k, v in case.items() if k in parts}, grads


def close(got, want, bound, what):
    u, tiny = ref.U[got.dtype], ref.TINY[got.dtype]
    assert got.shape == want.shape, what
    off = (got.detach().cpu().double() - want).abs() - bound - u * (want.abs() + bound) - tiny
    assert bool((off <= 0).all()), f'{what}: over its bound by {off.max().item():.3e}'


def run(pkg, leaves, grads, **more):
    """Results and gradients of one call."""
    args = {k: v for k, v in leaves.items() if k != 'x'}
    total, normed = pkg.residual_norm(leaves['x'], **args, eps=EPS, **more)
    out = {'sum': total, 'normed': normed}
    outs = [t for n, t in out.items() if t is not None and n in grads and t is not leaves['x']]
    douts = [grads[n] for n, t in out.items() if t is not None and n in grads and t is not leaves['x']]
    got = torch.autograd.grad(outs, list(leaves.values()), douts)
    out.update({'d' + n: t for n, t in zip(leaves, got)})
    return out


def check(pkg, cuda, case, grads, checkpoint=None):
    dev = {n: t.to(cuda).requires_grad_(True) for n, t in case.items()}
    got = run(pkg, dev, {n: t.to(cuda) for n, t in grads.items()}, checkpoint=checkpoint)
    torch.cuda.synchronize()
    rows, width = case['x'].shape
    groups = case['gate'].shape[0] if 'gate' in case else rows

    def reference(x, update):
        w = {n: t.double() for n, t in case.items()}
        w['x'] = x
        if 'update' in case:
            w['update'] = update
        w = {n: t.clone().requires_grad_(True) for n, t in w.items()}
        wide = {n: w.get(n) for n in NAMES}
        if 'gate' in w and rows:
            wide['gate'] = w['gate'].repeat_interleave(rows // groups, 0)
        return w, wide, ref.residual_norm(*(wide[n] for n in NAMES), EPS)

    u = case['update'].double() if 'update' in case else None
    w, wide, (total, normed) = reference(case['x'].double(), u)
    flat = [None if wide[n] is None else wide[n].detach() for n in NAMES]
    bounds = ref.residual_bounds(*flat, EPS, case['x'].dtype, case.get('update', case['x']).dtype)
    if 'update' in case:
        assert got['sum'].dtype == case['x'].dtype and got['sum'].is_contiguous()
        close(got['sum'], total.detach(), bounds['sum'], 'sum')
    else:
        assert got['sum'] is dev['x']
    if 'weight' in case:
        close(got['normed'], normed.detach(), bounds['normed'], 'normed')
    else:
        assert got['normed'] is None
    if checkpoint:
        w, wide, (total, normed) = reference(
            ref.kept(case['x']), None if u is None else ref.kept(case['update']))
        flat = [None if wide[n] is None else wide[n].detach() for n in NAMES]
    has = {'sum': 'update' in case and 'sum' in grads, 'normed': 'weight' in case and 'normed' in grads}
    outs = [t for n, t in (('sum', total), ('normed', normed)) if has[n]]
    douts = [grads[n].double() for n in has if has[n]]
    want = torch.autograd.grad(outs, list(w.values()), douts, allow_unused=True)
    bounds = ref.residual_bounds(
        *flat, EPS, case['x'].dtype, case.get('update', case['x']).dtype,
        grads['sum'].double() if has['sum'] else None,
        grads['normed'].double() if has['normed'] else None, groups if groups < rows else None)
    for (n, leaf), g in zip(w.items(), want):
        g = torch.zeros_like(leaf) if g is None else g
        close(got['d' + n], g, bounds.get('d' + n, torch.zeros(()).double()), 'd' + n)
    return got


@pytest.mark.parametrize('types', TYPES, ids=str)
@pytest.mark.parametrize('width', [1, 7, 80, 129, 257, 512, 1024, 1283, 2048, 2049, 4097, 8192])
def test_widths(pkg, cuda, width, types):
    check(pkg, cuda, *make(11, width, *types, seed=width, gate='element'))


@pytest.mark.parametrize('gate', [None, 'element', 1, 2, 6, 33])
@pytest.mark.parametrize('width', [96, 1280, 2056])
def test_gates(pkg, cuda, width, gate):
    """33 rows of gate for 66 rows, and one for all."""
    check(pkg, cuda, *make(66, width, torch.bfloat16, torch.bfloat16, seed=3, gate=gate))


@pytest.mark.parametrize('rows,gate', [(1, 1), (2, 1), (4099, None), (4098, 3), (4096, 2048),
                                       (2100, 2100)])
def test_rows(pkg, cuda, rows, gate):
    """More rows than blocks at once, parts of a gate's rows that end unevenly,
    more rows of gate than blocks, one for each row."""
    check(pkg, cuda, *make(rows, 40, torch.float32, torch.float32, seed=rows, gate=gate))


@pytest.mark.parametrize('rows,width,gate', [
    (1200, 200, 40), (4000, 1030, 40), (2600, 600, 20), (3200, 1283, 800), (8000, 40, 1000),
    (6000, 2048, 3)])
def test_shared_gates(pkg, cuda, rows, width, gate):
    """Parts of a gate's rows that a slice of the sums takes alone, or all do."""
    check(pkg, cuda, *make(rows, width, torch.float32, torch.float16, seed=gate, gate=gate))


@pytest.mark.parametrize('parts', [
    ('x', 'weight'), ('x', 'update'), ('x', 'update', 'weight'), ('x', 'update', 'update_weight'),
    ('x', 'update', 'scale'), ('x', 'update', 'gate', 'weight'),
    ('x', 'update', 'scale', 'gate'), ('x', 'update', 'update_weight', 'weight')], ids='-'.join)
@pytest.mark.parametrize('checkpoint', [None, 8])
def test_parts(pkg, cuda, parts, checkpoint):
    for gate in ('element', 3):
        for types in (TYPES[0], TYPES[4]):
            check(pkg, cuda, *make(21, 200, *types, seed=7, gate=gate, parts=parts), checkpoint)


@pytest.mark.parametrize('only', ['sum', 'normed'])
def test_gradient_of_one_output(pkg, cuda, only):
    case, grads = make(13, 100, torch.float32, torch.bfloat16, seed=5, gate='element')
    check(pkg, cuda, case, {only: grads[only]})


@pytest.mark.parametrize('only', ['sum', 'normed'])
@pytest.mark.parametrize('gate', [None, 5])
@pytest.mark.parametrize('width', [5, 1283])
def test_gradient_of_one_output_from_checkpoints(pkg, cuda, width, gate, only):
    """Rows, of gradients or of a gate, that are not there."""
    case, grads = make(10, width, torch.float32, torch.float16, seed=width, gate=gate)
    check(pkg, cuda, case, {only: grads[only]}, 8)


@pytest.mark.parametrize('types', TYPES, ids=str)
@pytest.mark.parametrize('width', [1, 31, 80, 1283, 2056, 5000])
def test_checkpoints(pkg, cuda, width, types):
    check(pkg, cuda, *make(19, width, *types, seed=width, gate='element'), 8)


def test_differences(pkg, cuda):
    """The gradient along a direction is the difference of the definition, in
    64 bits, to both sides."""
    case, grads = make(9, 150, torch.float32, torch.float32, seed=21, gate=3)
    dev = {n: t.to(cuda).requires_grad_(True) for n, t in case.items()}
    got = run(pkg, dev, {n: t.to(cuda) for n, t in grads.items()})
    g = torch.Generator().manual_seed(22)
    step = 2.0 ** -14

    def value(at):
        w = dict(at, gate=at['gate'].repeat_interleave(3, 0))
        outs = ref.residual_norm(*(w[n] for n in NAMES), EPS)
        return sum((o * grads[n].double()).sum() for n, o in zip(('sum', 'normed'), outs))

    for n, t in case.items():
        along = torch.randn(t.shape, generator=g, dtype=torch.float64)
        there, back = (value({**{k: v.double() for k, v in case.items()},
                              n: t.double() + i * step * along}) for i in (1, -1))
        want = (there - back) / (2 * step)
        d = got['d' + n].cpu().double()
        # fp32 gradients, each good to 1e-5 of their magnitudes here; differences to step^2 of
        # third derivatives (of values and weights around one)
        size = (d * along).abs().sum()
        assert abs((d * along).sum() - want) <= 1e-5 * size + 200 * step ** 2 * size, n


def test_strides(pkg, cuda):
    """Parts of wider rows, transposed and expanded operands and gradients, and
    leading dimensions: the bits of contiguous ones."""
    case, grads = make(24, 72, torch.bfloat16, torch.bfloat16, seed=9, gate='element')
    dev = {n: t.to(cuda) for n, t in case.items()}
    wide = torch.zeros((24, 3 * 72 + 5), device=cuda, dtype=torch.bfloat16)
    odd = dict(dev)
    odd['x'] = wide[:, 1:73].copy_(dev['x'])
    odd['update'] = dev['update'].t().contiguous().t()
    odd['gate'] = wide[:, 75:147].copy_(dev['gate'])
    odd['scale'] = torch.stack((dev['scale'], dev['scale']), 1)[:, 0]
    dgrads = {n: t.to(cuda) for n, t in grads.items()}
    ograds = {'sum': dgrads['sum'].t().contiguous().t(), 'normed': wide[:, 148:220].copy_(dgrads['normed'])}
    a = run(pkg, {n: t.detach().requires_grad_(True) for n, t in dev.items()}, dgrads)
    b = run(pkg, {n: t.detach().requires_grad_(True) for n, t in odd.items()}, ograds)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    shaped = {n: t.view(2, 3, 4, 72) if t.dim() == 2 else t for n, t in dev.items()}
    c = run(pkg, {n: t.detach().requires_grad_(True) for n, t in shaped.items()},
            {n: t.view(2, 3, 4, 72) for n, t in dgrads.items()})
    for n in a:
        assert torch.equal(a[n].flatten(), c[n].flatten()), n
    # one value for a whole row, and one row for all: gradients of broadcast inputs
    for gate in (torch.randn(24, 1), torch.randn(1, 72)):
        gate = gate.to(cuda, torch.bfloat16).requires_grad_(True)
        total, _ = pkg.residual_norm(dev['x'], dev['update'], gate=gate.expand(24, 72))
        d, = torch.autograd.grad(total, gate, dgrads['sum'])
        size = dev['update'].double() * dgrads['sum'].double()
        want = size.sum(1, keepdim=True) if gate.shape[1] == 1 else size.sum(0, keepdim=True)
        mag = size.abs().sum(1, keepdim=True) if gate.shape[1] == 1 else size.abs().sum(0, keepdim=True)
        # each part rounded to bf16 by the operator, then the sum
        close(d, want.cpu(), (2.0 ** -8 * mag).cpu() + 72 * ref.F * mag.cpu(), 'expanded gate')
    one = pkg.residual_norm(dev['x'], dev['update'], gate=dev['scale'])[0]
    assert torch.equal(one, pkg.residual_norm(dev['x'], dev['update'],
                                              gate=dev['scale'].expand(24, 72))[0])


@pytest.mark.parametrize('checkpoint', [None, 8])
def test_no_rows(pkg, cuda, checkpoint):
    for gate in (None, 'element', 3):
        case, grads = make(0, 24, torch.float32, torch.bfloat16, seed=1, gate=gate)
        leaves = {n: t.to(cuda).requires_grad_(True) for n, t in case.items()}
        got = run(pkg, leaves, {n: t.to(cuda) for n, t in grads.items()}, checkpoint=checkpoint)
        for n, t in leaves.items():
            assert got['d' + n].shape == t.shape and not got['d' + n].any()


def test_values_that_are_not_finite(pkg, cuda):
    """They reach their own row and the sums over rows, and no other row."""
    case, grads = make(40, 300, torch.float32, torch.bfloat16, seed=2, gate='element')
    leaves = {n: t.to(cuda).requires_grad_(True) for n, t in case.items()}
    dgrads = {n: t.to(cuda) for n, t in grads.items()}
    for checkpoint in (None, 8):
        clean = run(pkg, leaves, dgrads, checkpoint=checkpoint)
        for name, value in (('x', float('inf')), ('update', float('nan')), ('gate', float('-inf'))):
            bad = {n: t.detach().clone() for n, t in leaves.items()}
            bad[name][7, 33] = value
            got = run(pkg, {n: t.requires_grad_(True) for n, t in bad.items()}, dgrads,
                      checkpoint=checkpoint)
            rest = [i for i in range(40) if i != 7]
            for n in ('sum', 'normed', 'dx', 'dupdate', 'dgate'):
                assert torch.equal(got[n][rest], clean[n][rest]), (name, n)
            assert not got['normed'][7].isfinite().all()


def test_zero_rows_and_no_eps(pkg, cuda):
    """Rows of zeros: the norm of nothing is nothing, with finite gradients."""
    x = torch.zeros((3, 64), device=cuda, requires_grad=True)
    w = torch.ones(64, device=cuda, requires_grad=True)
    for checkpoint in (None, 8):
        total, normed = pkg.residual_norm(x, x.detach().requires_grad_(True), update_weight=w,
                                          weight=w, checkpoint=checkpoint)
        assert not total.any() and not normed.any()
        dx, dw = torch.autograd.grad((total, normed), (x, w), (torch.ones_like(x),) * 2)
        assert torch.equal(dx, torch.full_like(dx, 1 + 1000.0)) or torch.allclose(
            dx, torch.full_like(dx, 1001.0), rtol=1e-6)
        assert not dw.any()


def test_largest_halves(pkg, cuda):
    """fp16's largest numbers come back from a checkpoint as its largest, not as
    the power of two above it."""
    half = torch.float16
    g = torch.Generator().manual_seed(6)
    case, grads = make(12, 64, torch.float32, half, seed=6, parts=('x', 'update', 'weight'))
    at = torch.randint(0, 64, (12,), generator=g)
    case['update'][torch.arange(12), at] = torch.linspace(64900, 65504, 12).to(half)
    check(pkg, cuda, case, grads, 8)
    case, grads = make(12, 64, half, half, seed=7, parts=('x', 'weight'))
    case['x'][torch.arange(12), at] = torch.linspace(65504, 64900, 12).to(half)
    check(pkg, cuda, case, {'normed': 64 * grads['normed']}, 8)


@pytest.mark.parametrize('rows,width,types,gate', [
    (4002, 1283, TYPES[4], 6), (4002, 1280, TYPES[2], 6), (3000, 2056, TYPES[3], 3),
    (2000, 5000, TYPES[0], None), (1500, 8191, TYPES[4], 'element'), (6000, 640, TYPES[1], 2)])
@pytest.mark.parametrize('checkpoint', [None, 8])
def test_many_rows(pkg, cuda, rows, width, types, gate, checkpoint):
    """Rows of several waves, and many of them for each block: the next row's
    loads, the places of the sums and what is summed over rows."""
    check(pkg, cuda, *make(rows, width, *types, seed=rows, gate=gate), checkpoint)


def test_no_eps(pkg, cuda):
    """eps of zero: the formula, and for a row of zeros its quotient of zeros in
    that row and in the sums over rows, and nowhere else."""
    case, _ = make(9, 72, torch.float32, torch.float32, seed=8, parts=('x', 'weight'))
    dev = {n: t.to(cuda).requires_grad_(True) for n, t in case.items()}
    _, normed = pkg.residual_norm(dev['x'], weight=dev['weight'], eps=0.0)
    x, w = (case[n].double() for n in ('x', 'weight'))
    _, want = ref.residual_norm(x, None, None, None, None, w, 0.0)
    bounds = ref.residual_bounds(x, None, None, None, None, w, 0.0, torch.float32, torch.float32)
    close(normed, want, bounds['normed'], 'normed')
    zeros = case['x'].clone()
    zeros[4] = 0
    leaf = zeros.to(cuda).requires_grad_(True)
    for checkpoint in (None, 8):
        _, y = pkg.residual_norm(leaf, weight=dev['weight'], eps=0.0, checkpoint=checkpoint)
        dx, dw = torch.autograd.grad(y, (leaf, dev['weight']), torch.ones_like(y))
        rest = [i for i in range(9) if i != 4]
        assert y[4].isnan().all() and torch.equal(y[rest], normed[rest])
        assert dx[4].isnan().all() and dx[rest].isfinite().all() and dw.isnan().all()
