"""linear_int8 and quantize_weight against their definitions: codes and scales
exactly, results to the last rounding."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import block as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(tokens, width, out, dtype, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, width), generator=g) * (0.1 + 3 * torch.rand((tokens, 1), generator=g))
    codes = torch.randint(-127, 128, (out, width), generator=g).to(torch.int8)
    scales = torch.rand(out, generator=g) * 0.02 + 1e-3
    return x.to(dtype), codes, scales, torch.randn(out, generator=g).to(dtype) if bias else None


def check(pkg, cuda, x, codes, scales, bias, got=None):
    if got is None:
        got = pkg.linear_int8(x.to(cuda), codes.to(cuda), scales.to(cuda),
                              None if bias is None else bias.to(cuda))
    assert got.dtype == x.dtype and got.is_contiguous()
    want, bound = ref.linear_int8(x, codes, scales, bias)
    u, tiny = ref.U[x.dtype], ref.TINY[x.dtype]
    off = (got.cpu().double() - want).abs() - bound - u * (want.abs() + bound) - tiny
    assert got.shape == want.shape and bool((off <= 0).all()), off.max()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('tokens', [1, 2, 5, 16, 17, 33, 64, 67, 130, 300])
def test_tokens(pkg, cuda, dtype, tokens):
    for width, out in ((64, 96), (333, 130), (1280, 257)):
        check(pkg, cuda, *make(tokens, width, out, dtype, tokens))


@pytest.mark.parametrize('tokens', [1, 7, 200])
@pytest.mark.parametrize('width', [1, 15, 16, 17, 127, 128, 129, 500, 1025, 2049, 8193])
def test_widths(pkg, cuda, width, tokens):
    check(pkg, cuda, *make(tokens, width, 37, torch.bfloat16, width))


@pytest.mark.parametrize('tokens,width,out', [
    (9, 128, 4064), (16, 3000, 4100), (32, 200, 8193), (20, 300, 20001), (32, 129, 4000),
    (33, 128, 8191), (70, 129, 4097), (300, 333, 2000), (64, 640, 8193), (40, 2050, 50),
    (257, 1100, 1601)])
def test_parts_of_rows(pkg, cuda, tokens, width, out):
    """Rows whose length is divided: evenly, unevenly and with parts that are
    left with nothing; both sides of where tiles grow."""
    check(pkg, cuda, *make(tokens, width, out, torch.float16, width))


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('tokens,width', [
    (1, 2048), (1, 2049), (1, 16384), (1, 16385), (2, 8192), (2, 8193), (3, 4096), (4, 4097),
    (5, 2048), (8, 2048), (8, 2049), (9, 100)])
def test_few_tokens(pkg, cuda, dtype, tokens, width):
    """Both sides of where every block forms the codes itself; rows that begin
    at any address, and one that is not finite."""
    x, *rest = make(tokens, width, 41, dtype, width)
    wide = torch.zeros((tokens, width + 3), dtype=dtype, device=cuda)
    wide[:, 1:-2] = x.to(cuda)
    check(pkg, cuda, x, *rest, got=pkg.linear_int8(wide[:, 1:-2], *(t.to(cuda) for t in rest)))
    if tokens > 1:
        wide[1, width // 2] = float('inf')
        got = pkg.linear_int8(wide[:, 1:-2], *(t.to(cuda) for t in rest))
        assert bool(got[1].isnan().all())
        keep = [i for i in range(tokens) if i != 1]
        check(pkg, cuda, x[keep], *rest, got=got[keep])


@pytest.mark.parametrize('out', [1, 3, 4, 7, 8, 31, 32, 33, 127, 129, 1030])
@pytest.mark.parametrize('tokens', [1, 40])
def test_channels(pkg, cuda, out, tokens):
    for dtype in DTYPES:
        check(pkg, cuda, *make(tokens, 160, out, dtype, out, bias=out % 2 == 1))


@pytest.mark.parametrize('tokens,width,out', [
    (1000, 700, 2100), (2049, 256, 1025), (4100, 130, 600), (512, 300, 3001), (2000, 140, 8003),
    (4100, 130, 2100)])
def test_large(pkg, cuda, tokens, width, out):
    """More tiles than the card has CUs, and ends of tiles both ways."""
    check(pkg, cuda, *make(tokens, width, out, torch.bfloat16, 1))


@pytest.mark.parametrize('tokens', [1, 20, 200])
def test_largest_sums(pkg, cuda, tokens):
    """All codes at their ends: sums of 2^17 products of 127 and 128 fit."""
    width = 1 << 17
    x = torch.ones((tokens, width))
    x[0] = -3.0
    codes = torch.full((3, width), -128, dtype=torch.int8)
    codes[1] = 127
    check(pkg, cuda, x, codes, torch.tensor([0.5, 0.25, 2.0 ** -10]), None)


def test_codes(pkg, cuda):
    """Ties, values at borders of codes one unit to each side, ends of the
    range, zeros and rows that are not finite."""
    rows = []
    for top in (127.0, 64.0, 63.5, 1.0, 1e-3, 3e4, 254.0):
        s = ref.token_codes(torch.tensor([[top]]))[1].item()
        half = torch.arange(-126, 127).double() * s + 0.5 * s
        for y in (half, half * (1 + 2.0 ** -23), half * (1 - 2.0 ** -23)):
            y = y.clamp(-top, top).float()
            y[0] = top
            rows.append(y)
    for dtype in DTYPES:
        x = torch.stack(rows).to(dtype)
        codes, scales = pkg.quantize_weight(x.to(cuda))
        want, s = ref.token_codes(x)
        assert torch.equal(scales.cpu().double(), s[:, 0])
        assert torch.equal(codes.cpu().double(), want)
        assert codes.stride(0) % 128 == 0
    for scale in (0.0, 1e-42, 1e-37, 3e38):
        x = torch.linspace(-1, 1, 77)[None] * scale
        codes, scales = pkg.quantize_weight(x.to(cuda))
        want, s = ref.token_codes(x)
        assert torch.equal(scales.cpu().double(), s[:, 0]) and torch.equal(codes.cpu().double(), want)
    x = torch.randn(4, 50)
    x[1, 3], x[2, 49] = math.inf, math.nan
    _, scales = pkg.quantize_weight(x.to(cuda))
    assert scales.isnan().tolist() == [False, True, True, False]
    c, s = pkg.quantize_weight(torch.randn(6, 50, device=cuda))
    for tokens in (x, x.repeat(20, 1)):
        y = pkg.linear_int8(tokens.to(cuda), c, s)
        assert y.isnan().all(1).tolist() == [False, True, True, False] * (len(tokens) // 4)
        assert not y[0].isnan().any()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_every_width_of_a_row(pkg, cuda, dtype):
    """Codes of rows held by one and by four waves, and read twice."""
    for width in (3, 511, 513, 1025, 2000, 2049, 4097, 8191, 8193, 20000):
        x = torch.randn((5, width)).to(dtype)
        codes, scales = pkg.quantize_weight(x.to(cuda))
        want, s = ref.token_codes(x)
        assert torch.equal(scales.cpu().double(), s[:, 0]) and torch.equal(codes.cpu().double(), want)
        pitch = codes.stride(0)
        whole = codes.as_strided((5, pitch), (pitch, 1))
        assert not whole[:, width:].any()


@pytest.mark.parametrize('tokens', [1, 3, 90])
def test_layouts(pkg, cuda, tokens):
    """Weights at other pitches, not aligned, transposed, cut from wider ones
    whose neighbours must not matter; tokens in parts of rows."""
    x, codes, scales, bias = make(tokens, 100, 75, torch.bfloat16, 3)
    dev = [t.to(cuda) for t in (x, codes, scales, bias)]
    want = pkg.linear_int8(*dev)
    check(pkg, cuda, x, codes, scales, bias, want)
    wide = torch.full((75, 256), 113, dtype=torch.int8, device=cuda)
    for cut in (wide[:, :100], wide[:, 16:116], wide[:, 3:103], wide[:, 156:],
                wide.view(-1)[:75 * 101].view(75, 101)[:, :100],
                torch.empty((100, 75), dtype=torch.int8, device=cuda).t()):
        cut.copy_(dev[1])
        assert torch.equal(pkg.linear_int8(dev[0], cut, *dev[2:]), want)
    rows = torch.full((tokens, 333), math.nan, device=cuda, dtype=torch.bfloat16)
    rows[:, 5:105] = dev[0]
    assert torch.equal(pkg.linear_int8(rows[:, 5:105], *dev[1:]), want)
    assert torch.equal(pkg.linear_int8(dev[0].t().contiguous().t(), *dev[1:]), want)
    spaced = torch.stack((dev[2], dev[2]), 1)[:, 1], torch.stack((dev[3], dev[3]), 1)[:, 0]
    assert torch.equal(pkg.linear_int8(dev[0], dev[1], *spaced), want)
    assert torch.equal(pkg.linear_int8(dev[0].unsqueeze(1), *dev[1:]), want.unsqueeze(1))
    assert torch.equal(pkg.linear_int8(dev[0][0], *dev[1:]), want[0])
    one = pkg.linear_int8(dev[0], wide[:1, 3:103].copy_(dev[1][:1]), dev[2][:1], dev[3][:1])
    assert torch.equal(one, want[:, :1])


def test_nothing(pkg, cuda):
    c, s = pkg.quantize_weight(torch.randn(6, 50, device=cuda))
    assert pkg.linear_int8(torch.zeros((0, 50), device=cuda), c, s).shape == (0, 6)
    assert pkg.linear_int8(torch.zeros((3, 50), device=cuda), c[:0], s[:0]).shape == (3, 0)
    assert pkg.quantize_weight(torch.zeros((0, 50), device=cuda))[0].shape == (0, 50)


def test_layer(pkg, cuda):
    """Int8Linear: near the layer it is made of, fp32 scales after casts, and
    its state kept and loaded."""
    torch.manual_seed(0)
    linear = torch.nn.Linear(200, 90, device=cuda)
    layer = pkg.Int8Linear(linear)
    x = torch.randn(4, 7, 200, device=cuda)
    y, want = layer(x), linear(x)
    # each operand off by at most half of its scale: 1/127 of its largest magnitude (and 2^-8 of
    # that for the scale's own rounding up)
    half = 0.5 * (1 + 2 ** -7) / 127
    ex, ew = half * x.abs().amax(-1, keepdim=True), half * linear.weight.abs().amax(-1)
    bound = ex * linear.weight.abs().sum(-1) + ew * x.abs().sum(-1, keepdim=True) + 200 * ex * ew
    assert bool(((y - want).abs() <= bound + 1e-5).all())
    half = pkg.Int8Linear(linear).to(torch.bfloat16)
    assert half.scales.dtype == torch.float32
    assert torch.equal(half(x.bfloat16()), pkg.linear_int8(x.bfloat16(), layer.codes[:, :200], layer.scales,
                                                           linear.bias.detach().bfloat16()))
    moved = pkg.Int8Linear(linear).cpu().to(cuda)
    assert moved.codes.stride(0) % 128 == 0 and torch.equal(moved(x), y)
    other = pkg.Int8Linear(torch.nn.Linear(200, 90, device=cuda))
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('tokens', [1, 9, 20, 100])
@pytest.mark.parametrize('size,scale', [(1e33, 1e-4), (1e-4, 1e33), (1e-33, 1e-3), (1e33, 1e-36),
                                        (1e-36, 1e33)])
def test_far_scales(pkg, cuda, dtype, tokens, size, scale):
    """The largest and the smallest tokens and channels: nothing on the way leaves
    the range in which the result is, and a scale of zero gives zeros."""
    g = torch.Generator().manual_seed(tokens)
    x = ((0.5 + torch.rand((tokens, 8192), generator=g)) * size).to(dtype)
    codes = torch.randint(100, 128, (70, 8192), generator=g).to(torch.int8)
    scales = scale * (0.5 + torch.rand(70, generator=g))
    scales[5], scales[6] = 0, -scales[6]
    want, _ = ref.linear_int8(x, codes, scales, None)
    assert want.abs().max() < 1e36 and want[:, 0].abs().min() > 1e-33
    check(pkg, cuda, x, codes, scales, None)


@pytest.mark.parametrize('dtype,tokens,width,out', [
    (torch.bfloat16, 4100, 1290, 2100), (torch.float32, 2600, 650, 3333),    # 256 x 256
    (torch.float16, 1024, 600, 8192), (torch.bfloat16, 1100, 513, 7100),     # 128 x 256
    (torch.bfloat16, 1000, 1000, 2100), (torch.float32, 700, 1150, 4099),    # 64 x 128
    (torch.float16, 512, 1300, 3001), (torch.float32, 1030, 1190, 1800),     # 64 x 64
    (torch.bfloat16, 200, 2310, 4090), (torch.float16, 300, 2600, 2000),     # in two parts
    (torch.float16, 67, 5000, 4099), (torch.bfloat16, 67, 2800, 4099),       # 32 x 32 in three
    (torch.bfloat16, 64, 3700, 8001), (torch.float32, 257, 3300, 1601),      # 64 x 32 in four
    (torch.float32, 40, 4700, 201), (torch.float16, 31, 8100, 5003)])        # 32 x 32 in four
def test_long_walks(pkg, cuda, dtype, tokens, width, out):
    """Rows so long that every tile's ring of buffers goes round twice and more,
    with ends of tiles and of rows, on each kind of tile."""
    check(pkg, cuda, *make(tokens, width, out, dtype, width))
