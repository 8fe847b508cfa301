"""attend_cached against its definition in 64 bits: single and several new
tokens, caches of every length with and without a shared prefix, types, head
layouts, strides, slots past the lengths that hold anything, and refusals."""
from __future__ import annotations

import pytest
import torch

from oracle import tokens as ref

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(lengths, new, capacity, prefix, q_heads, k_heads, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g).to(dtype)
    B = len(lengths)
    return {'q': n(B, new, q_heads, dim), 'k': n(B, capacity, k_heads, dim),
            'v': n(B, capacity, k_heads, dim), 'lengths': torch.tensor(lengths),
            'prefix_k': n(prefix, k_heads, dim) if prefix else None,
            'prefix_v': n(prefix, k_heads, dim) if prefix else None}


def run(pkg, cuda, case, **kw):
    t = {n: x.to(cuda) if x is not None else None for n, x in case.items()}
    out = pkg.attend_cached(t['q'], t['k'], t['v'], t['lengths'], t['prefix_k'], t['prefix_v'],
                            **kw)
    torch.cuda.synchronize()
    return out


def check(pkg, cuda, case, scale=None):
    got = run(pkg, cuda, case, scale=scale)
    dtype, dim = case['q'].dtype, case['q'].shape[-1]
    value, bound = ref.attend_cached(case['q'], case['k'], case['v'], case['lengths'],
                                     case['prefix_k'], case['prefix_v'],
                                     dim ** -0.5 if scale is None else scale, dtype)
    assert got.shape == value.shape and got.dtype == dtype and got.is_contiguous()
    x = got.cpu().double()
    off = torch.where(x == value, torch.zeros(()).double(), (x - value).abs() - bound)
    assert bool((off <= 0).all()), f'over its bound by {off.max().item():.3e}'


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('q_heads, k_heads, dim', [(8, 2, 128), (3, 3, 64), (7, 1, 80), (4, 4, 32),
                                                   (2, 1, 96)])
@pytest.mark.parametrize('lengths, new, capacity, prefix', [
    ([1], 1, 1, 0),
    ([100], 1, 100, 0),                     # one part: no join
    ([0, 5, 200, 1000], 1, 1000, 0),        # an empty cache among others
    ([3, 4, 129, 700], 4, 700, 0),          # rows of a short cache that see nothing
    ([5, 1, 128], 1, 128, 300),
    ([5, 0, 64, 17, 40], 3, 64, 1111),      # rows that see the prefix alone
    ([0, 0], 1, 0, 33),                     # no cache at all
    ([1] * 70, 1, 2, 500),                  # many rows: the prefix by rows
], ids=str)
def test_lengths(pkg, cuda, lengths, new, capacity, prefix, q_heads, k_heads, dim, dtype):
    check(pkg, cuda, make(lengths, new, capacity, prefix, q_heads, k_heads, dim, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [8, 24, 40, 56, 72, 88, 112, 120])
def test_head_sizes(pkg, cuda, dim, dtype):
    check(pkg, cuda, make([50, 333], 2, 400, 0, 4, 2, dim, dtype))
    check(pkg, cuda, make([2] * 20, 2, 3, 300, 4, 2, dim, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_more_rows_than_a_tile(pkg, cuda, dtype):
    """Tokens times heads of a group above 32: several row tiles."""
    check(pkg, cuda, make([9, 200, 50], 9, 256, 0, 8, 2, 64, dtype))
    check(pkg, cuda, make([9, 40], 9, 64, 400, 10, 1, 64, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_long_cache(pkg, cuda, dtype):
    """Many parts, lengths at and around their ends."""
    check(pkg, cuda, make([4096, 128, 127, 129, 1, 2049], 1, 4097, 0, 2, 1, 64, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('prefix', [0, 200])
def test_unused_slots_hold_anything(pkg, cuda, dtype, prefix):
    """NaN and infinities past a request's length change no bit."""
    case = make([0, 1, 31, 64, 100, 300], 1, 300, prefix, 4, 2, 64, dtype)
    clean = run(pkg, cuda, case)
    for b, n in enumerate(case['lengths'].tolist()):
        case['k'][b, n:] = float('nan')
        case['v'][b, n::2] = float('inf')
        case['v'][b, n + 1::2] = float('nan')
    assert torch.equal(run(pkg, cuda, case), clean)
    assert bool(clean.isfinite().all())


@pytest.mark.gpu
def test_lengths_out_of_range(pkg, cuda):
    """Lengths below zero and above the capacity: as if within it."""
    case = make([-5, 70, 10 ** 6], 1, 64, 0, 4, 2, 64, torch.bfloat16)
    got = run(pkg, cuda, case)
    case['lengths'] = torch.tensor([0, 64, 64])
    assert torch.equal(got, run(pkg, cuda, case))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_strides(pkg, cuda, dtype):
    """Caches as (heads, slots) with keys and values interleaved, queries as a
    slice of a projection: the same bits as contiguous ones."""
    case = make([40, 7, 90], 2, 100, 50, 4, 2, 64, dtype)
    base = run(pkg, cuda, case)
    t = {n: x.to(cuda) for n, x in case.items()}
    both = torch.stack((t['k'], t['v']), 3).permute(0, 2, 1, 3, 4).contiguous()  # (B, Hk, cap, 2, D)
    k, v = both[..., 0, :].transpose(1, 2), both[..., 1, :].transpose(1, 2)
    pk = torch.stack((t['prefix_k'], t['prefix_v']), 1)
    for skip in (0, 3):
        wide = torch.zeros((3, 2, 4 * 64 + 40), dtype=dtype, device=cuda)
        q = wide[..., skip:skip + 256].unflatten(2, (4, 64))
        q.copy_(t['q'])
        out = pkg.attend_cached(q, k, v, t['lengths'].int(), pk[:, 0], pk[:, 1])
        assert torch.equal(out, base)


@pytest.mark.gpu
def test_single_tokens_and_agreement_with_packed(pkg, cuda):
    """(requests, heads, dim) queries; single tokens over caches are the last
    rows of causal prompts."""
    case = make([40, 1, 77], 1, 80, 0, 4, 2, 64, torch.float32)
    t = {n: x.to(cuda) if x is not None else None for n, x in case.items()}
    one = pkg.attend_cached(t['q'][:, 0], t['k'], t['v'], t['lengths'])
    assert one.shape == (3, 4, 64) and torch.equal(one, run(pkg, cuda, case)[:, 0])
    ks = torch.cat([t['k'][b, :n] for b, n in enumerate(case['lengths'].tolist())])
    vs = torch.cat([t['v'][b, :n] for b, n in enumerate(case['lengths'].tolist())])
    packed = pkg.attend_packed(t['q'][:, 0].contiguous(), ks, vs, torch.arange(4, device=cuda),
                               torch.tensor([0, 40, 41, 118], device=cuda), causal=True)
    assert float((packed - one).abs().max()) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_rising_scores(pkg, cuda, dtype):
    """The maximum moves from part to part by hundreds."""
    case = make([600, 900], 1, 900, 700, 2, 1, 64, dtype)
    for n in ('k', 'prefix_k'):
        x = case[n].float()
        rise = torch.linspace(0.1, 6, x.shape[-3])[:, None, None]
        case[n] = (x * rise).to(dtype)
    check(pkg, cuda, case, scale=1.0)


@pytest.mark.gpu
def test_same_bits_each_time_and_on_another_stream(pkg, cuda):
    case = make([700, 30, 1500], 2, 1500, 900, 8, 2, 128, torch.bfloat16)
    first = run(pkg, cuda, case)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(pkg, cuda, case)
    assert torch.equal(first, other) and torch.equal(first, run(pkg, cuda, case))


@pytest.mark.gpu
def test_offsets_past_32_bits(pkg, cuda):
    """A cache whose last request lies more than 4 GiB from its first."""
    case = make([300, 300, 300], 1, 300, 0, 2, 1, 64, torch.bfloat16)
    base = run(pkg, cuda, case)
    apart = (5 << 30) // 2 // 2  # elements between requests: 2.5 GiB
    big = torch.empty(2 * apart + 300 * 2 * 64, dtype=torch.bfloat16, device=cuda)
    k = big.as_strided((3, 300, 1, 64), (apart, 128, 64, 1))
    v = big.as_strided((3, 300, 1, 64), (apart, 128, 64, 1), 64)
    k.copy_(case['k'])
    v.copy_(case['v'])
    got = pkg.attend_cached(case['q'].to(cuda), k, v, case['lengths'].to(cuda))
    assert torch.equal(got, base)


@pytest.mark.gpu
def test_replayed_graph(pkg, cuda):
    """A captured step whose lengths grow between the replays."""
    case = make([10, 200], 1, 400, 300, 4, 2, 64, torch.bfloat16)
    t = {n: x.to(cuda) for n, x in case.items()}
    lengths = t['lengths'].int()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call = lambda: pkg.attend_cached(t['q'], t['k'], t['v'], lengths, t['prefix_k'],
                                     t['prefix_v'])
    with torch.cuda.stream(side):
        call(), call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        lengths.add_(45)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call()), i


@pytest.mark.gpu
def test_nothing(pkg, cuda):
    q, k = torch.zeros((0, 1, 4, 64), device=cuda), torch.zeros((0, 9, 2, 64), device=cuda)
    assert pkg.attend_cached(q, k, k, torch.zeros(0, dtype=torch.int32,
                                                  device=cuda)).shape == (0, 1, 4, 64)
    q, k = torch.ones((2, 1, 4, 64), device=cuda), torch.zeros((2, 0, 2, 64), device=cuda)
    out = pkg.attend_cached(q, k, k, torch.zeros(2, dtype=torch.int32, device=cuda))
    assert torch.equal(out, torch.zeros_like(out))


def test_refusals(pkg):
    q, k = torch.zeros((2, 1, 4, 64)), torch.zeros((2, 9, 2, 64))
    n = torch.tensor([3, 4])
    p = torch.zeros((5, 2, 64))
    with pytest.raises(ValueError, match='q must have 4 dimensions'):
        pkg.attend_cached(q[0, 0], k, k, n)
    with pytest.raises(ValueError, match='k must have 4 dimensions'):
        pkg.attend_cached(q, k[0], k[0], n)
    with pytest.raises(TypeError, match='k must have dtype'):
        pkg.attend_cached(q, k.double(), k.double(), n)
    with pytest.raises(TypeError, match='dtype of q'):
        pkg.attend_cached(q, k.half(), k.half(), n)
    with pytest.raises(ValueError, match='same shape'):
        pkg.attend_cached(q, k, k[:, :8], n)
    with pytest.raises(ValueError, match='same number of requests'):
        pkg.attend_cached(q[:1], k, k, n)
    with pytest.raises(ValueError, match='multiple of that of key heads'):
        pkg.attend_cached(q[:, :, :3], k, k, n)
    with pytest.raises(ValueError, match='at least one token'):
        pkg.attend_cached(q[:, :0], k, k, n)
    with pytest.raises(ValueError, match='go together'):
        pkg.attend_cached(q, k, k, n, p)
    with pytest.raises(ValueError, match='prefix_v must have shape'):
        pkg.attend_cached(q, k, k, n, p, p[:4])
    with pytest.raises(ValueError, match='prefix_k must have shape'):
        pkg.attend_cached(q, k, k, n, p[:, :1], p[:, :1])
    with pytest.raises(ValueError, match='16 bytes'):
        pkg.attend_cached(q, torch.zeros((2, 9, 2, 65))[..., 1:], k, n)
    with pytest.raises(ValueError, match=r'lengths must have shape \[requests\]'):
        pkg.attend_cached(q, k, k, n[:1])
    with pytest.raises(TypeError, match='lengths must have dtype'):
        pkg.attend_cached(q, k, k, n.float())
    with pytest.raises(ValueError, match='scale'):
        pkg.attend_cached(q, k, k, n, scale=-1.0)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        pkg.attend_cached(q, k, k, n)


@pytest.mark.gpu
def test_no_gradient(pkg, cuda):
    case = make([3], 1, 4, 0, 2, 1, 64, torch.float32)
    q = case['q'].to(cuda).requires_grad_(True)
    k, v, n = (case[x].to(cuda) for x in ('k', 'v', 'lengths'))
    with pytest.raises(RuntimeError, match='no gradient'):
        pkg.attend_cached(q, k, v, n)
    with torch.no_grad():
        assert pkg.attend_cached(q, k, v, n).shape == q.shape
