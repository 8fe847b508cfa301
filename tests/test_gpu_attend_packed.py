"""attend_packed against its definition in 64 bits: forward, log-sum-exp and
gradients over types, head layouts, lengths from none to long, causal and not,
rows that see nothing, strides, non-finite values in rows of others, and
refusals."""
from __future__ import annotations

import pytest
import torch

from oracle import tokens as ref

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(q_lengths, k_lengths, q_heads, k_heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g).to(dtype)
    tq, tk = sum(q_lengths), sum(k_lengths)
    return {'q': n(tq, q_heads, dim), 'k': n(tk, k_heads, dim), 'v': n(tk, k_heads, dim),
            'dout': n(tq, q_heads, dim),
            'q_starts': torch.tensor([0, *q_lengths]).cumsum(0),
            'k_starts': torch.tensor([0, *k_lengths]).cumsum(0)}


def run(pkg, cuda, case, causal, scale=None):
    q, k, v = (case[n].to(cuda).detach().requires_grad_(True) for n in 'qkv')
    out, lse = pkg.attend_packed(q, k, v, case['q_starts'].to(cuda), case['k_starts'].to(cuda),
                                 causal=causal, scale=scale, return_lse=True)
    grads = torch.autograd.grad(out, (q, k, v), case['dout'].to(cuda))
    torch.cuda.synchronize()
    return dict(zip(('out', 'lse', 'dq', 'dk', 'dv'), (out.detach(), lse, *grads)))


def compare(got, want):
    for name, (value, bound) in want.items():
        x = got[name].detach().cpu().double()
        assert x.shape == value.shape, name
        same = x == value  # (-inf among them)
        off = torch.where(same, torch.zeros(()).double(), (x - value).abs() - bound)
        assert bool((off <= 0).all()), \
            f'{name}: over its bound by {off.max().item():.3e} (nan: {bool(off.isnan().any())})'


def check(pkg, cuda, case, causal, scale=None):
    got = run(pkg, cuda, case, causal, scale)
    dtype = case['q'].dtype
    assert got['out'].dtype == dtype and got['lse'].dtype == torch.float32
    compare(got, ref.attend_packed(case['q'], case['k'], case['v'], case['q_starts'],
                                   case['k_starts'], causal,
                                   case['q'].shape[-1] ** -0.5 if scale is None else scale,
                                   case['dout'], dtype))


LENGTHS = [  # queries, keys of each sequence
    ([1], [1]),
    ([1, 1, 1], [1, 40, 300]),             # single tokens
    ([5, 128, 33, 1], [5, 128, 33, 1]),
    ([129, 64, 31], [200, 65, 90]),        # keys before the first query
    ([100, 7], [30, 7]),                   # rows that see nothing when causal
    ([0, 40, 0, 9, 0], [20, 0, 0, 300, 0]),  # no queries, no keys, neither
    ([257], [513]),
]


@pytest.mark.gpu
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('q_heads, k_heads, dim', [(2, 2, 64), (4, 1, 128), (6, 2, 80), (3, 1, 32),
                                                   (5, 5, 96)])
@pytest.mark.parametrize('lengths', LENGTHS, ids=str)
def test_lengths(pkg, cuda, lengths, q_heads, k_heads, dim, dtype, causal):
    check(pkg, cuda, make(*lengths, q_heads, k_heads, dim, dtype), causal)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [8, 16, 24, 40, 48, 56, 72, 88, 104, 112, 120])
def test_head_sizes(pkg, cuda, dim, dtype):
    """Every multiple of 8: heads that end inside a fragment or a tile."""
    check(pkg, cuda, make([70, 3], [70, 50], 4, 2, dim, dtype, seed=dim), True)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_wide_groups(pkg, cuda, dtype):
    """More heads in a group than a wave has rows."""
    check(pkg, cuda, make([9, 1, 20], [9, 70, 21], 40, 1, 32, dtype), True)
    check(pkg, cuda, make([9, 1, 20], [9, 70, 21], 21, 3, 32, dtype), False)


@pytest.mark.gpu
def test_many_sequences(pkg, cuda):
    """More sequences than one round of the search looks at, most short."""
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 4, (5000,), generator=g).tolist()
    lengths[777], lengths[4321] = 150, 90
    check(pkg, cuda, make(lengths, lengths, 2, 1, 32, torch.bfloat16), True)


@pytest.mark.gpu
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [32, 64, 80, 96, 128])
def test_full_card(pkg, cuda, dim, dtype, causal):
    """Enough blocks for the form that takes 128 rows a block (the smaller
    cases take 64)."""
    g = torch.Generator().manual_seed(dim)
    lengths = torch.randint(0, 3, (600,), generator=g).tolist()
    lengths[5], lengths[300], lengths[599] = 150, 260, 70
    keys = list(lengths)
    keys[300], keys[599] = 200, 130
    check(pkg, cuda, make(lengths, keys, 2, 1, dim, dtype), causal)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [32, 80, 128])
def test_long_walks(pkg, cuda, dim, dtype):
    """Few keys that very many rows see: the walk over them is cut."""
    check(pkg, cuda, make([1100, 900], [70, 140], 8, 1, dim, dtype), False)
    check(pkg, cuda, make([700], [700], 6, 1, dim, dtype), True)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [64, 80, 128])
def test_long_walks_of_a_full_card(pkg, cuda, dim, dtype):
    """Many short sequences fill the card with blocks of 128 keys, and the walks
    of a long one among them are cut in two; the same bits each time."""
    lengths = [3] * 25 + [1100] + [3] * 35
    case = make(lengths, lengths, 16, 8, dim, dtype)
    check(pkg, cuda, case, True)
    first, again = run(pkg, cuda, case, True), run(pkg, cuda, case, True)
    for n in first:
        assert torch.equal(first[n], again[n]), n


def check_far(pkg, cuda, case, causal, scale=None):
    """fp16 gradients of a dout far from 1, against the bound of the same dout
    brought to between 1 and 2: gradients are linear in it, and all that their
    own size costs is the last rounding."""
    dtype = case['q'].dtype
    got = run(pkg, cuda, case, causal, scale)
    by = 2.0 ** case['dout'].abs().max().double().log2().floor().item()
    want = ref.attend_packed(case['q'], case['k'], case['v'], case['q_starts'], case['k_starts'],
                             causal, case['q'].shape[-1] ** -0.5 if scale is None else scale,
                             case['dout'].double() / by, dtype)
    tiny = ref.TINY[dtype]
    for n in ('dq', 'dk', 'dv'):
        value, bound = want[n]
        want[n] = value * by, (bound - tiny) * by + tiny
    compare(got, want)
    return want


@pytest.mark.gpu
@pytest.mark.parametrize('small', ['q', 'k'])
@pytest.mark.parametrize('dim', [32, 80, 128])
def test_small_gradients_fp16(pkg, cuda, dim, small):
    """A dout of 1e-5 over hundreds of keys: score gradients far below what the
    type can hold."""
    for lengths, heads in ((([300, 9], [700, 30]), (4, 2)),
                           (([3] * 25 + [1100] + [3] * 35,) * 2, (16, 8))):
        case = make(*lengths, *heads, dim, torch.float16)
        case[small] = (case[small].float() * 0.02).half()
        case['dout'] = (case['dout'].float() * 1e-5).half()
        check_far(pkg, cuda, case, heads[0] == 16, scale=64.0 * dim ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize('dim', [32, 64, 80, 128])
def test_large_gradients_fp16(pkg, cuda, dim):
    """Gradients that fp16 can hold where those of the scores pass its range."""
    case = make([40, 3, 90], [40, 3, 90], 4, 2, dim, torch.float16)
    case['v'] = case['v'] * 4
    case['k'] = case['k'] * 0.5
    case['dout'] = case['dout'] * (5000 if dim < 64 else 4000)
    want = check_far(pkg, cuda, case, True)
    assert all(want[n][0].abs().max() < 60000 for n in ('dq', 'dk', 'dv'))
    a, most = 0, 0.0  # the scores' own
    for n in (40, 3, 90):
        for h in range(4):
            rows = slice(a, a + n)
            p = ref.attend_rows(case['q'][rows, h].double(), case['k'][rows, h // 2].double(),
                                case['v'][rows, h // 2].double(), list(range(1, n + 1)),
                                dim ** -0.5)[0]
            dp = case['dout'][rows, h].double() @ case['v'][rows, h // 2].double().T
            most = max(most, (p * (dp - (p * dp).sum(-1, keepdim=True))).abs().max().item())
        a += n
    assert most > 66000


@pytest.mark.gpu
def test_rows_of_far_gradients_fp16(pkg, cuda):
    """Rows whose dout lies 2^20 apart: each row's dq is as good as alone, and
    zeros, infinities and NaN in dout keep to their row's dq."""
    case = make([200], [200], 4, 2, 64, torch.float16)
    case['dout'][::2] = (case['dout'][::2].float() * 2.0 ** -20).half()
    case['dout'][5] = 0
    alone = dict(case, dout=case['dout'].clone())
    alone['dout'][1::2] = 0
    got, even = run(pkg, cuda, case, False), run(pkg, cuda, alone, False)
    assert torch.equal(got['dq'][::2], even['dq'][::2])
    assert not bool(got['dq'][5].any())
    case['dout'][7, 0, 3], case['dout'][8, 1, 2] = float('inf'), float('nan')
    far = run(pkg, cuda, case, False)
    keep = [i for i in range(200) if i not in (7, 8)]
    assert torch.equal(far['dq'][keep], got['dq'][keep])
    assert bool(far['dq'][8, 1].isnan().all()) and not bool(far['dq'][7, 0].isfinite().any())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_parts_of_one_projection(pkg, cuda, dtype):
    """Operands as slices of one matrix, aligned and not, and a gradient with
    strides: the same bits as contiguous copies."""
    T, hq, hk, dim = 75, 4, 2, 64
    case = make([40, 35], [40, 35], hq, hk, dim, dtype)
    base = run(pkg, cuda, case, True)
    for skip in (0, 8, 3):
        rows = torch.zeros((T, (hq + 2 * hk) * dim + 16), dtype=dtype, device=cuda)
        parts, at = [], skip
        for n, h in (('q', hq), ('k', hk), ('v', hk)):
            part = rows[:, at:at + h * dim].unflatten(1, (h, dim))
            part.copy_(case[n])
            parts.append(part)
            at += h * dim
        leaves = [p.detach().requires_grad_(True) for p in parts]
        out, lse = pkg.attend_packed(*leaves, case['q_starts'].to(cuda), causal=True,
                                     return_lse=True)
        dout = case['dout'].to(cuda).transpose(0, 2).contiguous().transpose(0, 2)
        grads = torch.autograd.grad(out, leaves, dout)
        for n, t in zip(('out', 'lse', 'dq', 'dk', 'dv'), (out, lse, *grads)):
            assert torch.equal(t, base[n]), (skip, n)


@pytest.mark.gpu
def test_broadcast_operands(pkg, cuda):
    """One head expanded to several (stride 0): its gradient is their sum."""
    T, dim = 50, 64
    case = make([50], [50], 4, 1, dim, torch.float32)
    k, v = (case[n].to(cuda).requires_grad_(True) for n in 'kv')
    q = case['q'].to(cuda).requires_grad_(True)
    s = case['q_starts'].to(cuda)
    out = pkg.attend_packed(q, k.expand(T, 4, dim), v.expand(T, 4, dim), s)
    grads = torch.autograd.grad(out, (q, k, v), case['dout'].to(cuda))
    want = ref.attend_packed(case['q'], case['k'], case['v'], case['q_starts'], case['k_starts'],
                             False, dim ** -0.5, case['dout'], torch.float32)
    compare(dict(zip(('out', 'dq', 'dk', 'dv'), (out, *grads))),
            {n: want[n] for n in ('out', 'dq', 'dk', 'dv')})


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_large_and_shifted_scores(pkg, cuda, dtype):
    """Scores of +-hundreds, rising along the keys so that the maximum moves
    in every tile, and rows far below zero."""
    case = make([90], [300], 2, 1, 64, dtype)
    case['k'] = (case['k'].float() * torch.linspace(0.1, 6, 300)[:, None, None]).to(dtype)
    case['q'][::3] *= 8
    case['k'][:, :, 0] = 0
    check(pkg, cuda, case, True)
    check(pkg, cuda, case, False, scale=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_rows_of_no_sequence(pkg, cuda, dtype):
    """Tokens after the last sequence: zeros and no gradient, whatever they
    hold."""
    case = make([30, 20], [30, 20], 2, 2, 64, dtype)
    case['q_starts'], case['k_starts'] = torch.tensor([0, 30]), torch.tensor([0, 30])
    for n in ('q', 'k', 'v'):
        case[n][30:] = float('nan')
    got = run(pkg, cuda, case, True)
    for n in ('out', 'dq', 'dk', 'dv'):
        assert torch.equal(got[n][30:], torch.zeros_like(got[n][30:])), n
    assert bool((got['lse'][30:] == float('-inf')).all())
    want = ref.attend_packed(*(case[n][:30] for n in 'qkv'), case['q_starts'], case['k_starts'],
                             True, 64 ** -0.5, case['dout'][:30], dtype)
    compare({n: t[:30] for n, t in got.items()}, want)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_nonfinite_stays_in_its_sequence(pkg, cuda, dtype):
    case = make([40, 50, 33], [40, 50, 33], 4, 2, 64, dtype)
    clean = run(pkg, cuda, case, True)
    case['k'][55, 0, 3], case['v'][60, 1, 5] = float('nan'), float('inf')
    case['q'][70, 1, 1], case['dout'][44, 2, 2] = float('-inf'), float('nan')
    got = run(pkg, cuda, case, True)
    for n in got:
        for part in (slice(0, 40), slice(90, 123)):
            assert torch.equal(got[n][part], clean[n][part]), n
    assert bool(got['out'][40:90].isnan().any())


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_same_bits_each_time_and_on_another_stream(pkg, cuda, dtype):
    case = make([700, 300], [700, 300], 4, 2, 64, dtype)
    first = run(pkg, cuda, case, True)
    again = run(pkg, cuda, case, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(pkg, cuda, case, True)
    for n in first:
        assert torch.equal(first[n], again[n]) and torch.equal(first[n], other[n]), n


@pytest.mark.gpu
def test_replayed_graph(pkg, cuda):
    """Forward and backward in a captured graph, new inputs for each replay."""
    case = make([130, 60], [130, 60], 4, 2, 64, torch.bfloat16)
    q, k, v = (case[n].to(cuda).requires_grad_(True) for n in 'qkv')
    dout, s = case['dout'].to(cuda), case['q_starts'].to(cuda, torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(pkg.attend_packed(q, k, v, s, causal=True), (q, k, v), dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.attend_packed(q, k, v, s, causal=True)
        grads = torch.autograd.grad(out, (q, k, v), dout)
    for seed in range(4):
        new = make([130, 60], [130, 60], 4, 2, 64, torch.bfloat16, seed)
        with torch.no_grad():
            for t, n in ((q, 'q'), (k, 'k'), (v, 'v'), (dout, 'dout')):
                t.copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        want = run(pkg, cuda, new, True)
        for n, t in zip(('out', 'dq', 'dk', 'dv'), (out, *grads)):
            assert torch.equal(t, want[n]), (seed, n)


@pytest.mark.gpu
@pytest.mark.parametrize('causal', [False, True])
def test_against_differences(pkg, cuda, causal):
    """Gradients against central differences of the definition."""
    case = make([9, 6], [9, 11], 2, 1, 16, torch.float32, 3)
    got = run(pkg, cuda, case, causal)
    args = (case['q_starts'], case['k_starts'], causal, 0.25)
    bounds = ref.attend_packed(case['q'], case['k'], case['v'], *args, case['dout'],
                               torch.float32)
    gen = torch.Generator().manual_seed(4)

    def loss(x):
        out = ref.attend_packed(x['q'], x['k'], x['v'], *args)['out'][0]
        return (out * case['dout'].double()).sum()

    for n in 'qkv':
        for _ in range(3):
            d = torch.randn(case[n].shape, generator=gen, dtype=torch.float64)
            h = 1e-5
            want = (loss({**case, n: case[n].double() + h * d})
                    - loss({**case, n: case[n].double() - h * d})) / (2 * h)
            found = (got['d' + n].cpu().double() * d).sum()
            # (the kernel's bound, and h^2 of the difference's own)
            assert abs(found - want) <= (bounds['d' + n][1] * d.abs()).sum() + 1e-7


def test_refusals(pkg):
    q, k = torch.zeros((6, 4, 64)), torch.zeros((6, 2, 64))
    s = torch.tensor([0, 6])
    with pytest.raises(ValueError, match='3 dimensions'):
        pkg.attend_packed(q[0], k, k, s)
    with pytest.raises(TypeError, match='q must have dtype'):
        pkg.attend_packed(q.double(), k, k, s)
    with pytest.raises(TypeError, match='dtype of q'):
        pkg.attend_packed(q, k.half(), k.half(), s)
    with pytest.raises(ValueError, match='same shape'):
        pkg.attend_packed(q, k, k[:5], s)
    with pytest.raises(ValueError, match='same dim'):
        pkg.attend_packed(q, k[..., :32], k[..., :32], s)
    with pytest.raises(ValueError, match='multiple of 8'):
        pkg.attend_packed(q[..., :60], k[..., :60], k[..., :60], s)
    with pytest.raises(ValueError, match='multiple of 8'):
        pkg.attend_packed(*(torch.zeros((6, 2, 136)),) * 3, s)
    with pytest.raises(ValueError, match='multiple of that of key heads'):
        pkg.attend_packed(q[:, :3], k, k, s)
    with pytest.raises(ValueError, match='scale'):
        pkg.attend_packed(q, k, k, s, scale=0.0)
    with pytest.raises(ValueError, match='scale'):
        pkg.attend_packed(q, k, k, s, scale=float('inf'))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        pkg.attend_packed(q, k, k, s)


@pytest.mark.gpu
def test_refusals_of_starts(pkg, cuda):
    q, k = torch.zeros((6, 4, 64), device=cuda), torch.zeros((7, 2, 64), device=cuda)
    s = torch.tensor([0, 6], device=cuda)
    with pytest.raises(ValueError, match='without k_starts'):
        pkg.attend_packed(q, k, k, s)
    with pytest.raises(ValueError, match=r'q_starts must have shape'):
        pkg.attend_packed(q, k, k, s[:0], s)
    with pytest.raises(TypeError, match='q_starts must have dtype'):
        pkg.attend_packed(q, k, k, s.float(), s)
    with pytest.raises(ValueError, match='same length'):
        pkg.attend_packed(q, k, k, s, torch.tensor([0, 3, 7], device=cuda))
    with pytest.raises(ValueError, match='device of q'):
        pkg.attend_packed(q, k, k, s.cpu(), s)
    # nothing at all
    none = pkg.attend_packed(q[:0], k[:0], k[:0], s[:1] * 0)
    assert none.shape == (0, 4, 64)


@pytest.mark.gpu
def test_starts_out_of_range_stay_inside(pkg, cuda):
    """Starts past the rows there are read and write nothing outside them
    (values that a caller got wrong: clamped, so no fault)."""
    case = make([40, 24], [40, 24], 2, 1, 32, torch.bfloat16)
    case['q_starts'] = torch.tensor([0, 40, 90])
    case['k_starts'] = torch.tensor([0, 40, 1000])
    got = run(pkg, cuda, case, True)
    case['q_starts'] = case['k_starts'] = torch.tensor([0, 40, 64])
    want = run(pkg, cuda, case, True)
    for n in got:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.gpu
def test_no_second_derivative(pkg, cuda):
    """A second derivative is refused, not silently left out."""
    q = torch.randn((6, 2, 32), device=cuda, requires_grad=True)
    starts = torch.tensor([0, 6], device=cuda)
    out = pkg.attend_packed(q, q, q, starts)
    grad, = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        grad.sum().backward()
