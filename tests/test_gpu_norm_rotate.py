"""norm_rotate against its definition in 64 bits: types, layouts, axes, sizes
that fit no vector, strides, long positions, gradients (of the formula and of
differences) and refusals."""
from __future__ import annotations

import itertools

import pytest
import torch

from oracle import tokens as ref

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(tokens, q_heads, k_heads, dim, pairs, dtype, norm, seed, far=False):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g).to(dtype)
    case = {'q': n(tokens, q_heads, dim), 'k': n(tokens, k_heads, dim),
            'positions': torch.randint(0, 10 ** 6 if far else 400, (tokens, max(1, len(pairs))),
                                       generator=g),
            'frequencies': torch.cat([10000.0 ** (-torch.arange(m) / max(m, 1)) for m in pairs]
                                     or [torch.zeros(0)]).float(),
            'dq': n(tokens, q_heads, dim), 'dk': n(tokens, k_heads, dim)}
    if norm:
        case['q_weight'], case['k_weight'] = (1 + 0.3 * n(dim)).to(dtype), n(dim)
    return case


def close(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    off = (got - want).abs() - bound
    assert bool((off <= 0).all()), f'{what}: over its bound by {off.max().item():.3e}'


def check(pkg, cuda, case, pairs, interleaved, eps=1e-6, positions=None):
    dtype = case['q'].dtype
    u, F = ref.U[dtype], ref.F
    dim = case['q'].shape[-1]
    names = [n for n in ('q', 'k', 'q_weight', 'k_weight') if n in case]
    dev = {n: case[n].to(cuda).requires_grad_(True) for n in names}
    pos = (case['positions'] if positions is None else positions).to(cuda)
    out = pkg.norm_rotate(dev['q'], dev['k'], pos, case['frequencies'].to(cuda), pairs,
                          q_weight=dev.get('q_weight'), k_weight=dev.get('k_weight'), eps=eps,
                          interleaved=interleaved)
    grads = torch.autograd.grad(out, [dev[n] for n in names],
                                (case['dq'].to(cuda), case['dk'].to(cuda)))
    torch.cuda.synchronize()
    grads = dict(zip(names, grads))
    for i, n in enumerate(('q', 'k')):
        x = case[n].double().requires_grad_(True)
        w = case.get(n + '_weight')
        w = w.double().requires_grad_(True) if w is not None else None
        y, size = ref.norm_rotate(x, case['positions'], case['frequencies'], pairs, w, eps,
                                  interleaved)
        assert out[i].is_contiguous() and out[i].dtype == dtype
        # norm: a sum of dim squares, root and products; rotation: 2 products, 1 sum, functions
        # good to 2 units
        close(out[i], y.detach(), u * y.detach().abs() + (dim / 2 + 16) * F * size
              + ref.TINY[dtype], n)
        g = case['d' + n].double()
        want = torch.autograd.grad(y, [x] + ([w] if w is not None else []), g)
        # the gradient's magnitudes: |R^T g| <= the pair's |g|, times w r, and the mean's part
        index, partner, _ = ref.pair_of(dim, pairs, interleaved)
        ga = g.abs() + g.abs()[..., partner]
        if w is None:
            size = ga
        else:
            xd, wd = x.detach(), w.detach().abs()
            r = 1 / torch.sqrt((xd * xd).mean(-1, keepdim=True) + eps)
            size = r * ga * wd + xd.abs() * r ** 3 * (ga * wd * xd.abs()).mean(-1, keepdim=True)
            parts = (ga * xd.abs() * r).sum((0, 1))
            rows = xd.shape[0] * xd.shape[1]
            close(grads[n + '_weight'], want[1], u * want[1].abs() + (rows + dim + 24) * F * parts
                  + ref.TINY[dtype], f'd{n}_weight')
        close(grads[n], want[0], u * want[0].abs() + (dim + 32) * F * size + ref.TINY[dtype],
              f'd{n}')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('norm', [True, False])
@pytest.mark.parametrize('tokens, q_heads, k_heads, dim, pairs, interleaved', [
    (1, 1, 1, 2, (1,), False),
    (1, 4, 2, 128, (16, 24, 24), False),
    (3, 2, 1, 80, (8, 16, 16), False),
    (7, 3, 3, 80, (8, 16, 16), True),
    (129, 5, 1, 72, (36,), False),     # units of 4 elements
    (65, 7, 1, 72, (27,), True),       # a part of the head; pairs end inside a unit
    (65, 7, 1, 72, (27,), False),      # single elements
    (33, 2, 2, 256, (127,), False),    # single elements, two units a lane
    (33, 2, 2, 256, (30, 1, 33, 64), False),
    (40, 2, 2, 34, (5, 0, 6), True),
    (50, 3, 1, 64, (), False),         # no pair at all
    (700, 8, 2, 64, (10, 11, 11), False),
])
def test_sizes(pkg, cuda, dtype, norm, tokens, q_heads, k_heads, dim, pairs, interleaved):
    case = make(tokens, q_heads, k_heads, dim, pairs, dtype, norm, 1)
    check(pkg, cuda, case, pairs, interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize('kind', [torch.int32, torch.int64, torch.float32])
def test_long_positions(pkg, cuda, kind):
    """Angles of 10^6 radians are as good as those of 1."""
    pairs = (16, 16)
    case = make(300, 2, 1, 64, pairs, torch.float32, True, 2, far=True)
    check(pkg, cuda, case, pairs, False, positions=case['positions'].to(kind))


@pytest.mark.gpu
def test_one_axis_and_strided_positions(pkg, cuda):
    case = make(37, 2, 1, 64, (32,), torch.bfloat16, True, 3)
    check(pkg, cuda, case, (32,), False, positions=case['positions'][:, 0])
    wide = torch.zeros((37, 5), dtype=torch.int64)
    wide[:, 0] = case['positions'][:, 0]
    check(pkg, cuda, case, (32,), False, positions=wide[:, :2])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_parts_of_one_projection(pkg, cuda, dtype):
    """Queries and keys as slices of one matrix at an odd offset, a gradient
    with its own strides: the same bits as contiguous copies."""
    pairs, T, hq, hk, dim = (8, 12, 12), 53, 4, 2, 64
    case = make(T, hq, hk, dim, pairs, dtype, True, 4)
    rows = torch.zeros((T, (hq + 2 * hk) * dim + 7), dtype=dtype)
    rows[:, 3:3 + hq * dim] = case['q'].flatten(1)
    rows[:, 3 + hq * dim:3 + (hq + hk) * dim] = case['k'].flatten(1)
    rows = rows.to(cuda)
    q = rows[:, 3:3 + hq * dim].view(T, hq, dim)
    k = rows[:, 3 + hq * dim:3 + (hq + hk) * dim].unflatten(1, (hk, dim))
    pos, freq = case['positions'].to(cuda), case['frequencies'].to(cuda)
    w = [case['q_weight'].to(cuda), case['k_weight'].to(cuda)]
    dq = case['dq'].to(cuda).transpose(0, 1).contiguous().transpose(0, 1)
    dk = case['dk'].to(cuda)[..., None].expand(-1, -1, -1, 2).contiguous()[..., 0]
    got = []
    for a, b, ga, gb in ((q, k, dq, dk), (case['q'].to(cuda), case['k'].to(cuda),
                                          case['dq'].to(cuda), case['dk'].to(cuda))):
        leaves = [t.detach().requires_grad_(True) for t in (a, b, *w)]
        out = pkg.norm_rotate(leaves[0], leaves[1], pos, freq, pairs, q_weight=leaves[2],
                              k_weight=leaves[3])
        got.append([*out, *torch.autograd.grad(out, leaves, (ga, gb))])
    for x, y in zip(*got):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_queries_alone_and_nothing(pkg, cuda):
    case = make(9, 3, 1, 64, (32,), torch.float32, True, 5)
    both = pkg.norm_rotate(case['q'].to(cuda), case['k'].to(cuda), case['positions'].to(cuda),
                           case['frequencies'].to(cuda), q_weight=case['q_weight'].to(cuda))
    q = case['q'].to(cuda).requires_grad_(True)
    w = case['q_weight'].to(cuda).requires_grad_(True)
    one, none = pkg.norm_rotate(q, None, case['positions'].to(cuda),
                                case['frequencies'].to(cuda), q_weight=w)
    assert none is None and torch.equal(one, both[0])
    one.sum().backward()
    assert q.grad.shape == q.shape and w.grad.shape == w.shape
    # no tokens: empty results, a weight's gradient of zeros
    q = torch.zeros((0, 3, 64), device=cuda, requires_grad=True)
    w = case['q_weight'].to(cuda).requires_grad_(True)
    out, _ = pkg.norm_rotate(q, None, torch.zeros((0,), dtype=torch.int32, device=cuda),
                             case['frequencies'].to(cuda), q_weight=w)
    out.sum().backward()
    assert out.shape == (0, 3, 64) and torch.equal(w.grad, torch.zeros_like(w))


@pytest.mark.gpu
def test_one_output_used(pkg, cuda):
    """A gradient that reaches queries or keys alone."""
    case = make(20, 2, 2, 64, (32,), torch.float32, True, 6)
    q, k = (case[n].to(cuda).requires_grad_(True) for n in ('q', 'k'))
    w = case['k_weight'].to(cuda).requires_grad_(True)
    out = pkg.norm_rotate(q, k, case['positions'].to(cuda), case['frequencies'].to(cuda),
                          k_weight=w)
    out[0].square().sum().backward()
    assert float(q.grad.abs().max()) > 0
    assert torch.equal(k.grad, torch.zeros_like(k)) and torch.equal(w.grad, torch.zeros_like(w))


@pytest.mark.gpu
def test_zero_rows_and_nonfinite(pkg, cuda):
    """A row of zeros stays zero with finite gradients; a row with a NaN
    keeps to itself."""
    case = make(6, 2, 1, 64, (32,), torch.bfloat16, True, 7)
    case['q'][1] = 0
    case['q'][3, 1, 5] = float('nan')
    out, _ = pkg.norm_rotate(case['q'].to(cuda), None, case['positions'].to(cuda),
                             case['frequencies'].to(cuda), q_weight=case['q_weight'].to(cuda))
    out = out.cpu()
    assert torch.equal(out[1], torch.zeros_like(out[1]))
    bad = torch.isnan(out).flatten(2).any(-1)
    assert bad.nonzero().tolist() == [[3, 1]]


@pytest.mark.gpu
def test_same_bits_each_time_and_on_another_stream(pkg, cuda):
    case = make(5000, 4, 2, 80, (8, 16, 16), torch.bfloat16, True, 8)
    t = {n: x.to(cuda) for n, x in case.items()}
    runs = []
    side = torch.cuda.Stream()
    for i in range(3):
        leaves = [t[n].detach().requires_grad_(True) for n in ('q', 'k', 'q_weight', 'k_weight')]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side if i == 2 else torch.cuda.current_stream()):
            out = pkg.norm_rotate(leaves[0], leaves[1], t['positions'], t['frequencies'],
                                  (8, 16, 16), q_weight=leaves[2], k_weight=leaves[3])
            runs.append([*out, *torch.autograd.grad(out, leaves, (t['dq'], t['dk']))])
        torch.cuda.synchronize()
    for other in runs[1:]:
        for x, y in zip(runs[0], other):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_against_differences(pkg, cuda):
    """The gradients against central differences of the definition."""
    pairs = (6, 10)
    case = make(5, 2, 1, 40, pairs, torch.float32, True, 9)
    dev = [case[n].to(cuda).requires_grad_(True) for n in ('q', 'q_weight')]
    out, _ = pkg.norm_rotate(dev[0], None, case['positions'].to(cuda),
                             case['frequencies'].to(cuda), pairs, q_weight=dev[1])
    grads = torch.autograd.grad(out, dev, case['dq'].to(cuda))

    def loss(q, w):
        y, _ = ref.norm_rotate(q, case['positions'], case['frequencies'], pairs, w)
        return (y * case['dq'].double()).sum()

    gen = torch.Generator().manual_seed(10)
    x = [case['q'].double(), case['q_weight'].double()]
    for i, g in enumerate(grads):
        for _ in range(4):
            d = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
            h = 1e-5
            up, down = ([t + (s * h * d if j == i else 0) for j, t in enumerate(x)]
                        for s in (1, -1))
            want = (loss(*up) - loss(*down)) / (2 * h)
            got = (g.cpu().double() * d).sum()
            # (fp32 gradients of about 1: 2^-24 times some 50 roundings, over all elements)
            assert abs(got - want) <= 64 * ref.F * (d.abs() * (g.cpu().double().abs() + 4)).sum()


def test_refusals(pkg):
    x = torch.zeros((4, 2, 64))
    pos, freq = torch.zeros(4, dtype=torch.int32), torch.zeros(32)
    with pytest.raises(ValueError, match='3 dimensions'):
        pkg.norm_rotate(x[0], None, pos, freq)
    with pytest.raises(TypeError, match='q must have dtype'):
        pkg.norm_rotate(x.double(), None, pos, freq)
    with pytest.raises(TypeError, match='dtype of q'):
        pkg.norm_rotate(x, x.half(), pos, freq)
    with pytest.raises(ValueError, match='agree on tokens and dim'):
        pkg.norm_rotate(x, x[:3], pos, freq)
    with pytest.raises(ValueError, match='even'):
        pkg.norm_rotate(x[..., :63], None, pos, freq[:8])
    with pytest.raises(ValueError, match='positions'):
        pkg.norm_rotate(x, None, pos[:3], freq)
    with pytest.raises(TypeError, match='positions'):
        pkg.norm_rotate(x, None, pos.double(), freq)
    with pytest.raises(ValueError, match='frequencies'):
        pkg.norm_rotate(x, None, pos, freq.double())
    with pytest.raises(ValueError, match='sum to the number'):
        pkg.norm_rotate(x, None, pos, freq, (8, 8))
    with pytest.raises(ValueError, match='sum to the number'):
        pkg.norm_rotate(x, None, pos, torch.zeros(33))
    with pytest.raises(ValueError, match='column for each axis'):
        pkg.norm_rotate(x, None, pos, freq, (16, 16))
    with pytest.raises(ValueError, match='at most 4'):
        pkg.norm_rotate(x, None, pos, freq, (8, 8, 8, 4, 4))
    with pytest.raises(ValueError, match='q_weight must have shape'):
        pkg.norm_rotate(x, None, pos, freq, q_weight=torch.zeros(32))
    with pytest.raises(ValueError, match='k_weight without k'):
        pkg.norm_rotate(x, None, pos, freq, k_weight=torch.zeros(64))
    with pytest.raises(ValueError, match='eps'):
        pkg.norm_rotate(x, None, pos, freq, eps=-1.0)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        pkg.norm_rotate(x, None, pos, freq)


def test_frequencies(pkg):
    f = pkg.axis_frequencies((2, 4))
    assert f.dtype == torch.float32 and f.shape == (6,)
    assert f.tolist() == pytest.approx([1.0, 0.01, 1.0, 0.1, 0.01, 0.001], rel=1e-6)
    s = pkg.axis_frequencies((2, 2), base=16.0, shared=True)
    assert s.tolist() == pytest.approx([1.0, 0.5, 0.25, 0.125], rel=1e-6)
    with pytest.raises(ValueError):
        pkg.axis_frequencies((2, -1))
    assert pkg.axis_frequencies((0, 3)).shape == (3,)
    for pairs, inter in itertools.product([(1,), (3, 2), ()], [False, True]):
        index, partner, first = ref.pair_of(12, pairs, inter)
        assert sorted(i for i in index if i >= 0) == sorted(2 * list(range(sum(pairs))))
        assert all(partner[partner[d]] == d for d in range(12))


@pytest.mark.gpu
def test_no_second_derivative(pkg, cuda):
    """A second derivative is refused, not silently left out."""
    q = torch.randn((6, 2, 32), device=cuda, requires_grad=True)
    pos = torch.arange(6, device=cuda, dtype=torch.int32)[:, None]
    out, _ = pkg.norm_rotate(q, None, pos, pkg.axis_frequencies((16,), device=cuda),
                             q_weight=torch.ones(32, device=cuda))
    grad, = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        grad.sum().backward()
