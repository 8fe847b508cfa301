"""gated_activation, 8-bit checkpoints and checkpoint_linear against their
definitions in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import block as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
KINDS = ['silu', 'gelu', 'sigmoid']


def close(got, want, bound, what):
    u, tiny = ref.U[got.dtype], ref.TINY[got.dtype]
    assert got.shape == want.shape, what
    off = (got.detach().cpu().double() - want).abs() - bound - u * (want.abs() + bound) - tiny
    assert bool((off <= 0).all()), f'{what}: over its bound by {off.max().item():.3e}'


def check(pkg, cuda, x, dout, kind, checkpoint):
    leaf = x.to(cuda).requires_grad_(True)
    out = pkg.gated_activation(leaf, kind, checkpoint=checkpoint)
    grad, = torch.autograd.grad(out, leaf, dout.to(cuda))
    assert out.dtype == grad.dtype == x.dtype and out.is_contiguous()
    close(out, ref.gated(x.double(), kind), ref.gated_bounds(x.double(), kind)['out'], 'out')
    at = x.double()
    if checkpoint:
        at = ref.kept(x.unflatten(-1, (2, -1))).flatten(-2)
    at.requires_grad_(True)
    want, = torch.autograd.grad(ref.gated(at, kind), at, dout.double())
    close(grad, want, ref.gated_bounds(at.detach(), kind, dout.double())['dx'], 'dx')


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('kind', KINDS)
@pytest.mark.parametrize('checkpoint', [None, 8])
def test_sizes(pkg, cuda, dtype, kind, checkpoint):
    """One row and value, widths on both sides of chunks, blocks of values and
    blocks of threads, and rows that a block of threads shares."""
    for rows, width in ((1, 1), (3, 7), (5, 31), (4, 33), (70, 40), (3, 2047), (2, 2056), (1, 5001)):
        g = torch.Generator().manual_seed(rows * width)
        x = (2 * torch.randn((rows, 2 * width), generator=g)).to(dtype)
        check(pkg, cuda, x, torch.randn((rows, width), generator=g).to(dtype), kind, checkpoint)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('kind', KINDS)
def test_far_values(pkg, cuda, dtype, kind):
    """Tails on both sides, where exponentials underflow, and zeros."""
    a = torch.cat((torch.linspace(-40, 40, 2001), torch.tensor([-200.0, -104.0, -88.0, 88.0, 200.0,
                                                               0.0, -0.0]))).to(dtype)
    x = torch.stack((a, torch.full_like(a, 1.5)), 0).flatten()[None]
    check(pkg, cuda, x, torch.full((1, a.numel()), 0.75).to(dtype), kind, None)


@pytest.mark.parametrize('kind', KINDS)
def test_differences(pkg, cuda, kind):
    g = torch.Generator().manual_seed(3)
    x, dout = torch.randn((6, 90), generator=g), torch.randn((6, 45), generator=g)
    along, step = torch.randn((6, 90), generator=g).double(), 2.0 ** -14
    leaf = x.to(cuda).requires_grad_(True)
    d, = torch.autograd.grad(pkg.gated_activation(leaf, kind), leaf, dout.to(cuda))
    there, back = ((ref.gated(x.double() + i * step * along, kind) * dout.double()).sum()
                   for i in (1, -1))
    d = d.cpu().double()
    size = (d * along).abs().sum()
    assert abs((d * along).sum() - (there - back) / (2 * step)) <= (1e-5 + 200 * step ** 2) * size


def test_strides(pkg, cuda):
    g = torch.Generator().manual_seed(4)
    x = torch.randn((12, 60), generator=g).to(cuda, torch.bfloat16)
    dout = torch.randn((12, 30), generator=g).to(cuda, torch.bfloat16)
    wide = torch.zeros((12, 131), device=cuda, dtype=torch.bfloat16)
    results = []
    for checkpoint in (None, 8):
        for y, d in ((x, dout), (wide[:, 3:63].copy_(x), wide[:, 70:100].copy_(dout)),
                     (x.t().contiguous().t(), dout.t().contiguous().t()),
                     (x.view(3, 4, 60), dout.view(3, 4, 30))):
            leaf = y.detach().requires_grad_(True)
            out = pkg.gated_activation(leaf, 'silu', checkpoint=checkpoint)
            grad, = torch.autograd.grad(out, leaf, d)
            results.append((out.flatten(), grad.flatten()))
        for out, grad in results[1:]:
            assert torch.equal(out, results[0][0]) and torch.equal(grad, results[0][1])
        results = []
    leaf = x.clone().requires_grad_(True)
    a, = torch.autograd.grad(pkg.gated_activation(leaf).sum(), leaf)  # (a gradient of strides 0)
    b, = torch.autograd.grad(pkg.gated_activation(leaf), leaf, torch.ones_like(dout))
    assert torch.equal(a, b)
    for rows in (0,):
        leaf = torch.zeros((rows, 60), device=cuda, requires_grad=True)
        for checkpoint in (None, 8):
            out = pkg.gated_activation(leaf, checkpoint=checkpoint)
            assert out.shape == (0, 30)
            assert torch.autograd.grad(out, leaf, out)[0].shape == (0, 60)


# ---- 8-bit checkpoints -----------------------------------------------------

def edge_values(dtype):
    """Ties, ends of the scale's steps, zeros, subnormals, the largest values,
    and ones that are not finite."""
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = [torch.arange(-127, 128) / 127 * 127.0, torch.arange(-127, 128) + 0.5,
            torch.arange(0, 255) * 0.25, torch.zeros(255),
            torch.linspace(126, 128, 255), torch.full((255,), 127.5), torch.linspace(-big, big, 255),
            torch.linspace(-small, small, 255), torch.linspace(-small, small, 255) / 64,
            torch.linspace(0, 300, 255)]
    x = torch.stack([r.double() for r in rows]).to(dtype)
    bad = torch.linspace(-3, 3, 255).to(dtype)
    bad[[0, 40, 41, 254]] = torch.tensor([math.inf, math.nan, -math.inf, math.nan]).to(dtype)
    all_bad = torch.full((255,), math.nan).to(dtype)
    return torch.cat((x, bad[None], all_bad[None]))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_checkpoint_values(pkg, cuda, dtype):
    """Exactly the values of the definition."""
    for x in (edge_values(dtype), torch.randn((33, 1283)).to(dtype), torch.randn((2, 5, 31)).to(dtype),
              torch.randn(7).to(dtype), torch.randn((3000, 4)).to(dtype)):
        packed = pkg.pack_activations(x.to(cuda))
        got = packed.unpack()
        assert got.shape == x.shape and got.dtype == dtype
        want = ref.kept(x).to(dtype)
        assert torch.equal(got.cpu().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
        assert not (got.cpu().isnan() & x.isfinite()).any()
    wide = torch.randn((9, 200), device=cuda).to(dtype)
    assert torch.equal(pkg.pack_activations(wide[:, 3:103]).unpack(),
                       pkg.pack_activations(wide[:, 3:103].contiguous()).unpack())
    assert pkg.pack_activations(wide[:0]).unpack().shape == (0, 200)


def test_one_value_that_is_not_finite(pkg, cuda):
    """It spoils its own gradient alone."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn((5, 128), generator=g).to(cuda, torch.bfloat16)
    dout = torch.randn((5, 64), generator=g).to(cuda, torch.bfloat16)
    bad = x.clone()
    bad[2, 9], bad[3, 64 + 20] = math.inf, math.nan
    grads = []
    for t in (x, bad):
        leaf = t.requires_grad_(True)
        grads.append(torch.autograd.grad(pkg.gated_activation(leaf, checkpoint=8), leaf, dout)[0])
    differ = (grads[0] != grads[1]).nonzero().tolist()
    # (the largest magnitude of their blocks may have been theirs before)
    assert {(r, c) for r, c in differ} >= {(2, 9), (3, 20)}
    assert all(r in (2, 3) for r, _ in differ)
    spoilt = grads[1].isnan().nonzero().tolist()
    assert spoilt == [[2, 9], [2, 73], [3, 20]] or spoilt == [[2, 9], [2, 73], [3, 20], [3, 84]]


# ---- linear layers ---------------------------------------------------------

@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows,width,out,bias', [(1, 1, 1, True), (37, 65, 19, True),
                                                 (130, 128, 64, False), (515, 33, 200, True)])
def test_checkpoint_linear(pkg, cuda, dtype, rows, width, out, bias):
    g = torch.Generator().manual_seed(rows)
    n = lambda *s: torch.randn(s, generator=g).to(dtype)
    x, w, dy = n(rows, width), n(out, width), n(rows, out)
    leaves = [t.to(cuda).requires_grad_(True) for t in ([x, w, n(out)] if bias else [x, w])]
    y = pkg.checkpoint_linear(*leaves)
    grads = torch.autograd.grad(y, leaves, dy.to(cuda))
    X, W, D = x.double(), w.double(), dy.double()
    kept = ref.kept(x)
    b = leaves[2].detach().cpu().double() if bias else torch.zeros(out).double()
    n = lambda k: (k + 8) * ref.F
    close(y, X @ W.T + b, n(width + 1) * (X.abs() @ W.abs().T + b.abs()), 'y')
    close(grads[0], D @ W, n(out) * (D.abs() @ W.abs()), 'dx')
    close(grads[1], D.T @ kept, n(rows) * (D.abs().T @ kept.abs()), 'dweight')
    if bias:
        close(grads[2], D.sum(0), n(rows) * D.abs().sum(0), 'dbias')
    assert torch.equal(y, torch.nn.functional.linear(*leaves))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize('rows,width,out', [
    (1, 1, 8), (31, 40, 16), (32, 128, 256), (33, 129, 264), (64, 33, 512), (255, 300, 8),
    (257, 127, 248), (1000, 260, 520), (5003, 96, 40), (9001, 257, 300 * 8)])
def test_weight_gradients(pkg, cuda, dtype, rows, width, out):
    """The weight's gradient from the checkpoint itself: sizes on both sides of
    steps, tiles and parts of the tokens; gradients of wide pitches."""
    g = torch.Generator().manual_seed(rows)
    x = (torch.randn((rows, width), generator=g) * 2 ** torch.randint(-6, 6, (rows, 1), generator=g)
         ).to(dtype)
    dy = torch.randn((rows, out), generator=g).to(dtype)
    w = torch.randn((out, width), generator=g).to(dtype)
    X, D, kept = x.to(cuda), dy.double(), ref.kept(x)
    leaf = w.to(cuda).requires_grad_(True)
    wide, odd = (torch.full((rows, out + 24), math.nan, dtype=dtype, device=cuda) for _ in range(2))
    results = []
    for grad in (dy.to(cuda), wide[:, 8:out + 8].copy_(dy), odd[:, 3:out + 3].copy_(dy)):
        results.append(torch.autograd.grad(pkg.checkpoint_linear(X, leaf), leaf, grad)[0])
    close(results[0], D.T @ kept, (rows + 8) * ref.F * (D.abs().T @ kept.abs()), 'dweight')
    for r in results[1:]:
        assert torch.equal(r, results[0])


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_bias_gradients(pkg, cuda, dtype):
    for rows, out in ((1, 1), (3, 65), (300, 7), (5001, 130)):
        g = torch.Generator().manual_seed(rows)
        dy = torch.randn((rows, out), generator=g).to(dtype)
        x, w = torch.zeros((rows, 8), device=cuda, dtype=dtype), torch.zeros((out, 8), device=cuda, dtype=dtype)
        b = torch.zeros(out, device=cuda, dtype=dtype, requires_grad=True)
        for grad in (dy.to(cuda), dy.t().contiguous().t().to(cuda)):
            d, = torch.autograd.grad(pkg.checkpoint_linear(x, w, b), b, grad)
            close(d, dy.double().sum(0), (rows + 8) * ref.F * dy.double().abs().sum(0), 'dbias')


def test_values_that_are_not_finite_in_gradients(pkg, cuda):
    """One gradient and one input: their row and column of the weight's gradient."""
    x, dy = torch.randn(70, 40, device=cuda).bfloat16(), torch.randn(70, 24, device=cuda).bfloat16()
    w = torch.zeros(24, 40, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    x[69, 5], dy[69, 9] = math.nan, math.inf
    d, = torch.autograd.grad(pkg.checkpoint_linear(x, w), w, dy)
    bad = ~d.isfinite()
    want = torch.zeros_like(bad)
    want[:, 5] = want[9] = True
    assert torch.equal(bad, want)


def test_checkpoint_linear_layer(pkg, cuda):
    """Leading dimensions, autocast, and what needs no gradient."""
    torch.manual_seed(0)
    layer = pkg.CheckpointLinear(48, 24, device=cuda)
    plain = torch.nn.Linear(48, 24, device=cuda)
    plain.load_state_dict(layer.state_dict())
    x = torch.randn(3, 5, 48, device=cuda, requires_grad=True)
    assert torch.equal(layer(x), plain(x))
    with torch.autocast('cuda', torch.bfloat16):
        y, z = layer(x), plain(x)
    assert y.dtype == torch.bfloat16 and torch.equal(y, z)
    dy = torch.randn_like(y)
    dx, db = torch.autograd.grad(y, (x, layer.bias), dy)
    assert dx.dtype == torch.float32
    ox, ob = torch.autograd.grad(z, (x, plain.bias), dy)
    assert torch.equal(dx, ox) and torch.allclose(db, ob, rtol=2 ** -7, atol=1e-2)
    layer.weight.requires_grad_(False)
    assert torch.equal(torch.autograd.grad(layer(x).sum(), x)[0],
                       torch.autograd.grad(plain(x).sum(), x)[0])
    with torch.no_grad():
        assert not layer(x).requires_grad


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows', [0, 5])
def test_no_outputs(pkg, cuda, dtype, rows):
    """A layer of no channels, as torch's own: empty gradients, and zeros for x."""
    leaves = [torch.ones(s, device=cuda, dtype=dtype, requires_grad=True)
              for s in ((rows, 16), (0, 16), (0,))]
    y = pkg.checkpoint_linear(*leaves)
    assert y.shape == (rows, 0)
    for t, d in zip(leaves, torch.autograd.grad(y, leaves, y.detach())):
        assert d.shape == t.shape and d.dtype == dtype and not d.any()


def test_largest_halves(pkg, cuda):
    """fp16's largest numbers come back from a checkpoint as its largest, not as
    the power of two above it: gradients of silu, whose slope is one there."""
    half = torch.float16
    g = torch.Generator().manual_seed(9)
    x = torch.linspace(64000, 65504, 400).to(half).repeat(3, 2)
    dout = (torch.randn((3, 400), generator=g) / 64).to(half)
    leaf = x.to(cuda).requires_grad_(True)
    out = pkg.gated_activation(leaf, 'silu', checkpoint=8)
    got, = torch.autograd.grad(out, leaf, dout.to(cuda))
    a, b = ref.kept(x.unflatten(-1, (2, -1))).unbind(-2)
    assert a.max() == 65504
    want = torch.cat((dout.double() * b, dout.double() * a), -1).to(half)  # (exact products)
    assert torch.equal(got.cpu(), want)


def test_checkpoints_laid_out_otherwise(pkg, cuda):
    """Bytes that have been moved are the same checkpoint wherever they lie."""
    x = torch.randn((6, 3, 70), device=cuda).bfloat16()
    packed = pkg.pack_activations(x)
    want, data = packed.unpack(), packed.data
    shifted = torch.zeros(data.numel() + 1, dtype=torch.uint8, device=cuda)[1:].view(data.shape)
    for other in (data.t().contiguous().t(), data.cpu().to(cuda), shifted.copy_(data),
                  torch.stack((data, data), 1)[:, 0]):
        assert torch.equal(pkg.PackedActivations(other, packed.shape, packed.dtype).unpack(), want)
