"""The block's operators where no kernel runs: refusals of the C entries and of
the Python calls, what follows a call besides gradients, and layouts of codes;
and on the GPU streams, graphs, repeated calls and calls beside each other."""
from __future__ import annotations

import warnings

import pytest
import torch
from torch.autograd import forward_ad


class NoLaunches:
    """Results of the right shapes, and no gradients."""

    @staticmethod
    def residual_norm_forward(x, *args):
        return torch.empty_like(x), torch.empty_like(x), None, None

    @staticmethod
    def residual_norm(x, *args):
        return torch.empty_like(x), torch.empty_like(x)

    @staticmethod
    def gated_activation_forward(x, *args):
        return x.new_empty((x.shape[0], x.shape[1] // 2)), None

    @staticmethod
    def gated_activation(x, *args):
        return x.new_empty((x.shape[0], x.shape[1] // 2))

    @staticmethod
    def linear_int8(x, codes, row, scales, bias):
        return x.new_empty((x.shape[0], scales.shape[0]))


@pytest.fixture
def block(pkg, monkeypatch):
    """The module with its launches and the check for a GPU left out."""
    from bevfusion_triton_amd import block

    monkeypatch.setattr(block.P, 'require_gpu', lambda *t: None)
    monkeypatch.setattr(block.L, 'block_calls', lambda: NoLaunches)
    return block


@pytest.fixture(autouse=True)
def no_error_left(pkg):
    """The thread's error text is as other tests expect it: a call of nothing
    clears it."""
    yield
    assert pkg.library().bevpool_gated_forward(None, 0, 0, 0, 1, 0, None, None, None) == 0


# ---- the C entries: they return before any HIP call ------------------------

def refused(lib, call, cases):
    for bad, status, text in cases:
        assert call(**bad) == status, bad
        assert text in lib.bevpool_last_error(), bad


def test_residual_norm_entries(pkg):
    lib = pkg.library()

    def forward(x=16, x_dtype=2, update=16, uw=16, scale=16, gate=16, gate_rows=4, weight=16, dtype=2,
                rows=8, width=64, eps=1e-6, total=16, normed=16):
        return lib.bevpool_residual_norm_forward(x, 64, x_dtype, update, 64, uw, scale, gate, 64,
                                                 gate_rows, weight, dtype, rows, width, eps, total,
                                                 normed, None, None, None)

    refused(lib, forward, (
        (dict(dtype=3), -1, b'dtype'), (dict(x_dtype=1), -1, b'fp32'), (dict(rows=-1), -1, b'rows'),
        (dict(width=0), -1, b'width'), (dict(width=8193), -1, b'width'),
        (dict(eps=-1.0), -1, b'eps'), (dict(eps=float('nan')), -1, b'eps'),
        (dict(gate_rows=3), -1, b'divide'), (dict(gate_rows=0), -1, b'without rows'),
        (dict(update=None), -1, b'of an update'), (dict(x=None), -1, b'null'),
        (dict(total=None), -1, b'null'), (dict(normed=None), -1, b'null'),
        (dict(update=None, uw=None, scale=None, gate=None, weight=None), -1, b'neither')))
    assert forward(rows=0, x=None, update=None, gate=None) == 0

    def backward(x=16, update=16, uw=16, gate=16, gate_rows=4, weight=16, dnormed=16, rows=8, dx=16,
                 dupdate=16, dgate=16, duw=16, dscale=None, dweight=16, scratch=16, nbytes=1 << 20):
        return lib.bevpool_residual_norm_backward(
            x, 64, 2, update, 64, uw, None, gate, 64, gate_rows, weight, 0, None, 0, dnormed, 64, 2,
            rows, 64, 1e-6, dx, dupdate, dgate, duw, dscale, dweight, scratch, nbytes, None)

    need = lib.bevpool_residual_norm_backward_scratch_bytes(8, 64, 4, 2, 0)
    refused(lib, backward, (
        (dict(gate_rows=3), -1, b'divide'), (dict(x=None), -1, b'null'), (dict(dx=None), -1, b'null'),
        (dict(dupdate=None), -1, b'null'), (dict(dgate=None), -1, b'null'),
        (dict(dnormed=None), -1, b'null'), (dict(duw=None), -1, b'place'),
        (dict(dweight=None), -1, b'place'), (dict(dscale=16), -1, b'not there'),
        (dict(update=None), -1, b'of an update'), (dict(scratch=None), -3, b'scratch'),
        (dict(nbytes=need - 1), -3, b'scratch'),
        (dict(update=None, uw=None, duw=None, gate=None, weight=None, dweight=None), -1, b'neither')))
    assert need > 0 and lib.bevpool_residual_norm_backward_scratch_bytes(0, 64, 0, 2, 0) == 0


def test_gated_and_checkpoint_entries(pkg):
    lib = pkg.library()

    def forward(x=16, dtype=2, rows=4, width=64, act=0, out=16):
        return lib.bevpool_gated_forward(x, 128, dtype, rows, width, act, out, None, None)

    def backward(x=16, dtype=2, rows=4, width=64, act=0, out=16):
        return lib.bevpool_gated_backward(x, 128, 0, 16, 64, dtype, rows, width, act, out, None)

    def pack(x=16, dtype=2, rows=4, width=64, out=16):
        return lib.bevpool_checkpoint_pack(x, 64, dtype, rows, width, out, None)

    def unpack(x=16, dtype=2, rows=4, width=64, out=16):
        return lib.bevpool_checkpoint_unpack(x, dtype, rows, width, out, None)

    for call in (forward, backward, pack, unpack):
        refused(lib, call, (
            (dict(dtype=-1), -1, b'dtype'), (dict(rows=-1), -1, b'rows'), (dict(width=0), -1, b'width'),
            (dict(width=(1 << 18) + 1), -1, b'width'), (dict(rows=1 << 40), -1, b'grid'),
            (dict(x=None), -1, b'null'), (dict(out=None), -1, b'null')))
        assert call(rows=0, x=None, out=None) == 0
    for call in (forward, backward):
        refused(lib, call, ((dict(act=3), -1, b'activation'), (dict(act=-1), -1, b'activation')))
    pitch = lib.bevpool_checkpoint_pitch
    assert [pitch(w) for w in (0, 1, 32, 33, 1280)] == [0, 48, 48, 80, 1328]


def test_weight_gradient_entries(pkg):
    lib = pkg.library()

    def grad(dy=16, row=64, kept=16, dtype=2, tokens=100, n=64, k=40, dw=16, scratch=16, nbytes=1 << 30):
        return lib.bevpool_checkpoint_weight_grad(dy, row, kept, dtype, tokens, n, k, dw, scratch,
                                                  nbytes, None)

    need = lib.bevpool_checkpoint_weight_grad_scratch_bytes(100, 64, 40)
    refused(lib, grad, (
        (dict(dtype=0), -1, b'16-bit'), (dict(tokens=0), -1, b'tokens'), (dict(n=60), -1, b'multiple of 8'),
        (dict(n=0), -1, b'multiple of 8'), (dict(k=0), -1, b'2^18'), (dict(k=(1 << 18) + 1), -1, b'2^18'),
        (dict(dy=None), -1, b'null'), (dict(kept=None), -1, b'null'), (dict(dw=None), -1, b'null'),
        (dict(dy=8), -1, b'16 bytes'), (dict(row=60), -1, b'16 bytes'), (dict(row=1 << 24), -1, b'16 bytes'),
        (dict(kept=8), -1, b'16 bytes'), (dict(scratch=None), -3, b'scratch'),
        (dict(nbytes=need - 1), -3, b'scratch')))
    assert need == 64 * 40 * 4

    def sums(x=16, dtype=2, rows=9, width=5, out=16, scratch=16, nbytes=1 << 20):
        return lib.bevpool_column_sums(x, 5, dtype, rows, width, out, scratch, nbytes, None)

    need = lib.bevpool_column_sums_scratch_bytes(5)
    refused(lib, sums, (
        (dict(dtype=3), -1, b'dtype'), (dict(rows=-1), -1, b'rows'), (dict(width=0), -1, b'width'),
        (dict(x=None), -1, b'null'), (dict(out=None), -1, b'null'), (dict(scratch=None), -3, b'scratch'),
        (dict(nbytes=need - 1), -3, b'scratch')))
    assert sums(width=1 << 27, nbytes=1 << 60) == -1 and b'grid' in lib.bevpool_last_error()


def test_linear8_entries(pkg):
    lib = pkg.library()

    def product(x=16, dtype=2, weight=16, row=128, scales=16, tokens=3, width=100, channels=5, y=16,
                scratch=16, nbytes=3 * 132):
        return lib.bevpool_linear8(x, 100, dtype, weight, row, scales, None, tokens, width, channels,
                                   y, scratch, nbytes, None)

    refused(lib, product, (
        (dict(dtype=7), -1, b'dtype'), (dict(width=0), -1, b'width'),
        (dict(width=(1 << 17) + 1), -1, b'width'), (dict(tokens=-1), -1, b'tokens'),
        (dict(channels=1 << 31), -1, b'channels'), (dict(x=None), -1, b'null'),
        (dict(weight=None), -1, b'null'), (dict(scales=None), -1, b'null'), (dict(y=None), -1, b'null'),
        (dict(weight=8), -1, b'16 bytes'), (dict(row=100), -1, b'16 bytes'),
        (dict(row=96), -1, b'16 bytes'), (dict(row=1 << 22), -1, b'16 bytes'),
        (dict(scratch=None), -3, b'scratch'), (dict(scratch=8), -3, b'scratch'),
        (dict(nbytes=3 * 132 - 1), -3, b'scratch')))
    assert product(tokens=1, width=1, row=16, channels=1 << 30, nbytes=1 << 20) == -1
    assert b'grid' in lib.bevpool_last_error()
    assert lib.bevpool_linear8_codes(16, 1, 2, 1 << 30, 1, 16, 16, None) == -1
    assert b'grid' in lib.bevpool_last_error()
    assert lib.bevpool_linear8_scratch_bytes(3, 100) == 3 * 132
    assert product(tokens=0, x=None) == 0 and product(channels=0, weight=None) == 0
    assert lib.bevpool_linear8_codes(16, 100, 2, 3, 100, None, 16, None) == -1
    assert b'null' in lib.bevpool_last_error()
    assert [lib.bevpool_linear8_pitch(w) for w in (1, 128, 129)] == [128, 128, 256]


# ---- the Python calls ------------------------------------------------------

def test_cpu_tensors_are_refused(pkg):
    x, w = torch.zeros(3, 8), torch.ones(8)
    for call in (lambda: pkg.residual_norm(x, weight=w), lambda: pkg.gated_activation(x),
                 lambda: pkg.pack_activations(x), lambda: pkg.checkpoint_linear(x, torch.zeros(4, 8)),
                 lambda: pkg.quantize_weight(x),
                 lambda: pkg.linear_int8(x, torch.zeros(4, 8, dtype=torch.int8), torch.ones(4))):
        with pytest.raises(RuntimeError, match='ROCm GPU only'):
            call()


def test_refusals(block):
    x, w, half = torch.zeros(6, 8), torch.ones(8), torch.float16
    norm, gated = block.residual_norm, block.gated_activation
    codes, scales = torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    linear, product = block.checkpoint_linear, block.linear_int8
    for call, kind, text in (
            (lambda: norm(x), ValueError, 'nothing to do'),
            (lambda: norm(x, scale=w, weight=w), ValueError, 'of an update'),
            (lambda: norm(x, x[:5], weight=w), ValueError, 'shape of x'),
            (lambda: norm(x, x, weight=w[:7]), ValueError, 'shape'),
            (lambda: norm(x, x, scale=w.half()), TypeError, 'dtype'),
            (lambda: norm(x.half(), x.bfloat16()), TypeError, 'float32 or'),
            (lambda: norm(x.int(), weight=w), TypeError, 'dtype'),
            (lambda: norm(x, x, gate=x[:4]), ValueError, 'divide'),
            (lambda: norm(x, x, gate=x[:0]), ValueError, 'divide'),
            (lambda: norm(x, x, gate=x[:, :1]), ValueError, 'gate'),
            (lambda: norm(x, x, gate=w.half()), TypeError, 'gate'),
            (lambda: norm(x, weight=w, eps=-1.0), ValueError, 'eps'),
            (lambda: norm(x, weight=w, checkpoint=4), ValueError, 'checkpoint'),
            (lambda: norm(torch.zeros(2, 8193), weight=torch.ones(8193)), ValueError, '8192'),
            (lambda: norm(torch.zeros(()), weight=w), ValueError, 'width'),
            (lambda: gated(x, 'relu'), ValueError, 'kind'),
            (lambda: gated(x[:, :7]), ValueError, 'shape'),
            (lambda: gated(x[:, :0]), ValueError, 'shape'),
            (lambda: gated(x.double()), TypeError, 'dtype'),
            (lambda: gated(x, checkpoint=16), ValueError, 'checkpoint'),
            (lambda: block.pack_activations(x.clone().requires_grad_(True)), RuntimeError, 'no gradient'),
            (lambda: block.pack_activations(x[:, :0]), ValueError, 'width'),
            (lambda: linear(x, torch.zeros(4, 7)), ValueError, 'in'),
            (lambda: linear(x, torch.zeros(4, 8, dtype=half)), TypeError, 'weight'),
            (lambda: linear(x, torch.zeros(4, 8), torch.zeros(3)), ValueError, 'bias'),
            (lambda: block.quantize_weight(w), ValueError, 'out, in'),
            (lambda: block.quantize_weight(x.int()), TypeError, 'dtype'),
            (lambda: product(x, x, scales), TypeError, 'int8'),
            (lambda: product(x[:, :7], codes, scales), ValueError, 'in'),
            (lambda: product(x, codes, scales.half()), TypeError, 'scales'),
            (lambda: product(x, codes, scales[:3]), ValueError, 'scales'),
            (lambda: product(x, codes, scales, scales.half()), TypeError, 'bias'),
            (lambda: product(x, codes, scales, scales[:2]), ValueError, 'bias'),
            (lambda: product(x.clone().requires_grad_(True), codes, scales), RuntimeError,
             'no gradient')):
        with pytest.raises(kind, match=text):
            call()


CALLS = {
    'residual_norm': lambda b, x: b.residual_norm(x, x, weight=torch.ones_like(x[0]))[1],
    'gated_activation': lambda b, x: b.gated_activation(x),
    'checkpoint_linear': lambda b, x: b.checkpoint_linear(x, torch.ones_like(x[:4])),
    'linear_int8': lambda b, x: b.linear_int8(x, torch.ones_like(x[:4], dtype=torch.int8),
                                              torch.ones_like(x[:4, 0])),
}


@pytest.mark.parametrize('name', CALLS)
def test_tangents_are_refused(block, name):
    """A result without a tangent would stand for a derivative of zero."""
    x = torch.randn(6, 8)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match='jvp'):
            CALLS[name](block, dual)
    assert CALLS[name](block, x).shape[0] == 6


@pytest.mark.parametrize('name', CALLS)
def test_a_trace_records_the_call(block, name):
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')  # (sizes as constants)
        traced = torch.jit.trace(lambda x: CALLS[name](block, x), (torch.randn(6, 8),),
                                 check_trace=False)
    assert '^_' in str(traced.graph)


def test_code_rows(block):
    """Codes in place where each row starts at 16 bytes and can be read up to
    16, and copies of all others."""
    store = torch.zeros(10 * 48, dtype=torch.int8)
    whole = store.view(10, 48)
    for view in (whole, whole[:, :33], whole[:, :48], whole[2:, 16:40], whole[:1, :5]):
        codes, row = block._code_rows(view)
        assert codes.data_ptr() == view.data_ptr() and row % 16 == 0
        last = (view.shape[0] - 1) * row + (view.shape[1] + 15) // 16 * 16
        assert codes.storage_offset() + last <= store.numel()
    for view in (whole[:, 1:20], whole.t(), store[:9 * 20].view(9, 20), whole[:, 4:].as_strided(
            (9, 15), (48, 2)), store[480 - 5:].view(1, 5), store.as_strided((12, 20), (40, 1)),
            store.as_strided((3, 8), (0, 1))):
        codes, row = block._code_rows(view)
        assert codes.data_ptr() != view.data_ptr() and torch.equal(codes[:, :view.shape[1]], view)
        assert row % 16 == 0 and row >= view.shape[1]


# ---- on the GPU ------------------------------------------------------------

def operands(cuda, rows=37, width=120, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(rows)
    n = lambda *s: torch.randn(s, generator=g).to(cuda, dtype)
    return {'x': n(rows, width), 'update': n(rows, width), 'w': 1 + 0.2 * n(width), 'gate': n(1, width),
            'linear': n(64, width), 'bias': n(64), 'dx': n(rows, width), 'dhalf': n(rows, width // 2), 'dy': n(rows, 64)}


def steps(pkg, t, codes, checkpoint):
    """One pass through each operator with its gradients."""
    leaves = [t[n].detach().requires_grad_(True)
              for n in ('x', 'update', 'w', 'gate', 'linear', 'bias')]
    x, update, w, gate, linear, bias = leaves
    total, normed = pkg.residual_norm(x, update, update_weight=w, scale=w, gate=gate, weight=w,
                                      checkpoint=checkpoint)
    half = pkg.gated_activation(x, 'gelu', checkpoint=checkpoint)
    y = pkg.checkpoint_linear(x, linear, bias)
    with torch.no_grad():
        z = pkg.linear_int8(t['x'], *codes)
    grads = torch.autograd.grad((total, normed, half, y), leaves, (t['dx'], t['dx'], t['dhalf'], t['dy']))
    return [total.detach(), normed.detach(), half.detach(), y.detach(), z, *grads]


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [None, 8])
def test_the_same_bits_again(pkg, cuda, checkpoint):
    t = operands(cuda, 5000)
    codes = pkg.quantize_weight(t['linear'])
    want = steps(pkg, t, codes, checkpoint)
    for a, b in zip(steps(pkg, t, codes, checkpoint), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize('checkpoint', [None, 8])
def test_graphs(pkg, cuda, checkpoint):
    """Two captured steps replayed between each other and eager ones, with new
    inputs in place."""
    cases = [operands(cuda, rows) for rows in (37, 300)]
    codes = [pkg.quantize_weight(t['linear']) for t in cases]
    for t, c in zip(cases, codes):
        steps(pkg, t, c, checkpoint)
    graphs, results = [], []
    torch.cuda.synchronize()
    for t, c in zip(cases, codes):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(steps(pkg, t, c, checkpoint))
    for turn in range(4):
        for t in cases:
            for n in ('x', 'update', 'dx', 'dy'):
                t[n].copy_(torch.randn_like(t[n]))
        for i in (0, 1, 0) if turn % 2 else (1, 0, 1):
            graphs[i].replay()
        torch.cuda.synchronize()
        for t, c, got in zip(cases, codes, results):
            want = steps(pkg, t, c, checkpoint)
            for k, (a, b) in enumerate(zip(got, want)):
                assert torch.equal(a, b), (turn, k)


@pytest.mark.gpu
def test_streams(pkg, cuda):
    """Calls on a stream of their own, behind work that makes their inputs, and
    two streams at once."""
    t = operands(cuda, 3000)
    codes = pkg.quantize_weight(t['linear'])
    want = steps(pkg, t, codes, 8)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            late = {n: torch.zeros_like(x) for n, x in t.items()}
            for n, x in t.items():
                late[n].copy_(x)
            got.append(steps(pkg, late, codes, 8))
    torch.cuda.synchronize()
    for results in got:
        for a, b in zip(results, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize('name', CALLS)
def test_a_trace_runs_on_other_inputs(pkg, cuda, name):
    x = torch.randn(6, 8, device=cuda)
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')
        traced = torch.jit.trace(lambda x: CALLS[name](pkg, x), (x,), check_trace=False)
    other = x.flip(0).contiguous()
    for _ in range(4):  # (the executor optimises after the first runs)
        assert torch.equal(traced(other), CALLS[name](pkg, other))


@pytest.mark.gpu
def test_a_second_derivative_is_refused(pkg, cuda):
    x = torch.randn(4, 16, device=cuda, requires_grad=True)
    w = torch.ones(16, device=cuda)
    for out in (pkg.residual_norm(x, x, weight=w)[1], pkg.gated_activation(x),
                pkg.checkpoint_linear(x, w[None])):
        g, = torch.autograd.grad(out.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


@pytest.mark.gpu
def test_more_than_2_31_values(pkg, cuda):
    """Offsets past 32 bits: the last rows are those of a call of their own."""
    rows, width = 270_000, 8192  # 2.2 G values
    x = torch.empty((rows, width), device=cuda, dtype=torch.bfloat16)
    x[:] = torch.randn(width, device=cuda).bfloat16()
    x[-3:] = torch.randn((3, width), device=cuda).bfloat16()
    w = torch.ones(width, device=cuda, dtype=torch.bfloat16)
    total, normed = pkg.residual_norm(x, x, update_weight=w, weight=w)
    small = pkg.residual_norm(x[-3:], x[-3:], update_weight=w, weight=w)
    assert torch.equal(total[-3:], small[0]) and torch.equal(normed[-3:], small[1])
    del total, normed
    assert torch.equal(pkg.gated_activation(x)[-3:], pkg.gated_activation(x[-3:]))
    packed = pkg.pack_activations(x)
    assert torch.equal(packed.unpack()[-3:], pkg.pack_activations(x[-3:]).unpack())
    del packed
    leaf = x.requires_grad_(True)
    dy = torch.ones((rows, width // 2), device=cuda, dtype=torch.bfloat16)
    d, = torch.autograd.grad(pkg.gated_activation(leaf, checkpoint=8), leaf, dy)
    tail = x.detach()[-3:].clone().requires_grad_(True)
    e, = torch.autograd.grad(pkg.gated_activation(tail, checkpoint=8), tail, dy[-3:])
    assert torch.equal(d[-3:], e)
    del d, dy
    dy = torch.ones((rows, width), device=cuda, dtype=torch.bfloat16)
    d, = torch.autograd.grad(pkg.residual_norm(leaf, leaf, weight=w, checkpoint=8), leaf, (dy, dy))
    e, = torch.autograd.grad(pkg.residual_norm(tail, tail, weight=w, checkpoint=8), tail,
                             (dy[-3:], dy[-3:]))
    assert torch.equal(d[-3:], e)
    del d, dy, leaf, x
    x = torch.randn((70_000, 96), device=cuda).bfloat16()
    codes, scales = pkg.quantize_weight(torch.randn((40_000, 96), device=cuda))
    with torch.no_grad():
        y = pkg.linear_int8(x, codes, scales)
        assert torch.equal(y[-300:], pkg.linear_int8(x[-300:], codes, scales))


@pytest.mark.gpu
def test_what_is_kept(pkg, cuda):
    """A checkpoint is what the backward pass holds on to: 33 bytes for 32
    values, and the operands themselves are free."""
    x = torch.randn(4096, 1280, device=cuda, dtype=torch.bfloat16)
    held = {}

    def requested():  # (allocated blocks may be larger)
        return torch.cuda.memory_stats()['requested_bytes.all.current']

    for checkpoint in (None, 8):
        leaf = x.clone().requires_grad_(True)
        torch.cuda.synchronize()
        before = requested()
        out = pkg.gated_activation(leaf * 1.0, 'silu', checkpoint=checkpoint)
        held[checkpoint] = requested() - before - out.numel() * 2
        del out
    assert held[None] == 4096 * 1280 * 2
    assert held[8] == 4096 * 2 * 672  # (rows of 640 codes and 20 scales, at 16 bytes)


def test_checkpoints_that_do_not_fit_are_refused(block):
    """Before any kernel reads them: rows of another length, number or type."""
    data = torch.zeros((3, 48), dtype=torch.uint8)  # (of rows of 1 to 32 values)
    for bad, shape in ((data[:, :47], (3, 8)), (data[:2], (3, 8)), (data, (4, 8)), (data, (3, 33)),
                       (data, (3, 2, 8)), (data[0], (8,)), (data, (0, 8)), (data, (3, 0))):
        with pytest.raises(ValueError, match='checkpoint'):
            block.PackedActivations(bad, torch.Size(shape), torch.bfloat16).unpack()
    for bad, dtype in ((data.to(torch.int8), torch.bfloat16), (data, torch.float64)):
        with pytest.raises(TypeError, match='dtype'):
            block.PackedActivations(bad, torch.Size((3, 8)), dtype).unpack()


def test_checkpoints_on_the_host_are_refused(pkg):
    with pytest.raises(RuntimeError, match='ROCm GPU only'):
        pkg.PackedActivations(torch.zeros((3, 48), dtype=torch.uint8), torch.Size((3, 8)),
                              torch.bfloat16).unpack()
