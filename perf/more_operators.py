"""The operators of a transformer block around the attention, as they are
measured: norms fused with gate and residual, the gated activation, linear
layers that keep their input in 8 bits for the backward pass, and products in
8-bit integers for serving.

A case is a dict of plain values:

  kind        'residual'  residual_norm
              'gated'     gated_activation
              'linear'    checkpoint_linear
              'int8'      linear_int8
  dtype, tokens, width    type of the operands, rows, elements of a row
  grad        True: forward and the gradients of every input; False: forward
  checkpoint  True: the backward pass works from 8-bit copies of its inputs
              (blocks of 32 values along a row that share a power of two)

  'residual'  stream: type of the residual stream; gate: 'none', 'element'
              (one for each value) or 'groups' (one row for each of `groups`
              equal parts of the rows); post: norm after the block; scale: a
              residual scale for each channel; norm: norm before the next block
  'gated'     act: 'silu', 'gelu' or 'sigmoid'; width: of the result
  'linear', 'int8'   out: channels of the result; bias
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
SIZE = {'f32': 4, 'f16': 2, 'bf16': 2}
EPS = 1e-6
BLOCK = 32  # values that share a scale in a checkpoint

CAMERAS = 6 * 32 * 88  # tokens of six cameras' feature maps

RESIDUAL = {'kind': 'residual', 'grad': True, 'dtype': 'bf16', 'stream': 'bf16',
            'tokens': CAMERAS, 'width': 1280, 'gate': 'none', 'groups': 1, 'post': True,
            'scale': True, 'norm': True, 'checkpoint': False}
GATED = {'kind': 'gated', 'grad': True, 'dtype': 'bf16', 'tokens': CAMERAS, 'width': 5120,
         'act': 'silu', 'checkpoint': True}
LINEAR = {'kind': 'linear', 'grad': True, 'dtype': 'bf16', 'tokens': CAMERAS, 'width': 1280,
          'out': 1280, 'bias': False, 'checkpoint': True}
INT8 = {'kind': 'int8', 'grad': False, 'dtype': 'bf16', 'tokens': CAMERAS, 'width': 1280,
        'out': 10240, 'bias': False, 'checkpoint': False}


def listed():
    return [
        # the next token of 16 requests, between attention and projections:
        # latency
        dict(RESIDUAL, name='residual_token', grad=False, tokens=16, width=4096),
        # the tokens of six cameras, a gate for each camera, one training step
        dict(RESIDUAL, name='residual_cameras_step', gate='groups', groups=6),
        # the same with the stream in single precision, kept in 8 bits
        dict(RESIDUAL, name='residual_8bit_step', stream='f32', checkpoint=True),
        # a long prompt, a gate for every value, rows that fit no vector
        dict(RESIDUAL, name='residual_odd_infer', grad=False, dtype='f16', stream='f16',
             tokens=30011, width=1283, gate='element'),
        # the next token of 16 requests: latency
        dict(GATED, name='gated_token', grad=False, tokens=16, width=10240, checkpoint=False),
        # the hidden values of six cameras' tokens, kept in 8 bits, one step
        dict(GATED, name='gated_cameras_step'),
        # a part of a BEV map in single precision, odd sizes, one step
        dict(GATED, name='gated_odd_f32_step', dtype='f32', tokens=4097, width=1031, act='gelu',
             checkpoint=False),
        # a projection of six cameras' tokens, one step, its input kept in 8 bits
        dict(LINEAR, name='linear_cameras_step'),
        # a small odd one in half precision
        dict(LINEAR, name='linear_odd_step', dtype='f16', tokens=2701, width=515, out=389,
             bias=True),
        # the next token of one request: the weights' bytes and latency
        dict(INT8, name='int8_token', tokens=1, width=4096, out=6144),
        # the next token of 64 requests, sizes that fit no tile
        dict(INT8, name='int8_batch', dtype='f16', tokens=67, width=5000, out=4099, bias=True),
        # the gated layer's projection of six cameras' tokens
        dict(INT8, name='int8_cameras'),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(['residual', 'residual', 'gated', 'gated', 'linear', 'int8', 'int8'])
    base = {'residual': RESIDUAL, 'gated': GATED, 'linear': LINEAR, 'int8': INT8}[kind]
    case = dict(base, dtype=rng.choice(['bf16', 'bf16', 'f16', 'f32']))
    if kind == 'residual':
        case['stream'] = rng.choice([case['dtype'], 'f32'])
        case['width'] = rng.choice([log_int(64, 8192), 8 * log_int(8, 1024)])
        case['tokens'] = min(log_int(1, 60000), CAMERAS * 1280 // case['width'])
        case['gate'] = rng.choice(['none', 'element', 'groups'])
        if case['gate'] == 'groups':
            case['groups'] = min(case['tokens'], rng.choice([1, 2, 6, 40]))
            case['tokens'] -= case['tokens'] % case['groups']
        case['post'] = rng.random() < 0.7
        case['scale'] = rng.random() < 0.7
        case['norm'] = rng.random() < 0.8
        case['grad'] = rng.random() < 0.6
        case['checkpoint'] = case['grad'] and rng.random() < 0.5
    elif kind == 'gated':
        case['width'] = rng.choice([log_int(64, 16384), 8 * log_int(8, 2048)])
        case['tokens'] = min(log_int(1, 60000),
                             2 * CAMERAS * 5120 // (SIZE[case['dtype']] * case['width']))
        case['act'] = rng.choice(['silu', 'gelu', 'sigmoid'])
        case['grad'] = rng.random() < 0.6
        case['checkpoint'] = case['grad'] and rng.random() < 0.6
    elif kind == 'linear':
        case['width'], case['out'] = log_int(64, 4096), log_int(64, 4096)
        most = CAMERAS * 1280 * 1280 // (case['width'] * case['out'])
        case['tokens'] = min(log_int(16, 30000), most // (8 if case['dtype'] == 'f32' else 1) + 1)
        case['bias'] = rng.random() < 0.5
    else:
        case['width'] = rng.choice([log_int(64, 8192), 16 * log_int(8, 512)])
        case['out'] = rng.choice([log_int(64, 12000), 16 * log_int(8, 750)])
        most = CAMERAS * 1280 * 10240 // (case['width'] * case['out'])
        case['tokens'] = min(rng.choice([log_int(1, 64), log_int(1, 30000)]), most,
                             CAMERAS * 10240 * 2 // (case['out'] * SIZE[case['dtype']]))
        case['bias'] = rng.random() < 0.5
    return case


def work(case):
    size, n, width = SIZE[case['dtype']], case['tokens'], case['width']
    values = n * width
    packed = (BLOCK + 1) / BLOCK
    if case['kind'] == 'residual':
        wide = SIZE[case['stream']]
        gate = {'none': 0, 'element': size, 'groups': 0}[case['gate']]
        moved = 2 * wide + size + (size if case['norm'] else 0) + gate
        if case['grad']:
            kept = 2 * packed if case['checkpoint'] else wide + size
            # (the checkpoint is written and read; gradients of both outputs in, of inputs out)
            moved += kept * (2 if case['checkpoint'] else 1) + 2 * wide + size + 2 * gate
            moved += size if case['norm'] else 0
        return {'bytes': int(values * moved), 'flops': (55 if case['grad'] else 15) * values}
    if case['kind'] == 'gated':
        moved = 3 * size
        if case['grad']:
            moved += 3 * size + (4 * packed if case['checkpoint'] else 2 * size)
        return {'bytes': int(values * moved), 'flops': (30 if case['grad'] else 12) * values}
    if case['kind'] == 'linear':
        ins, outs, weight = values * size, n * case['out'] * size, width * case['out'] * size
        return {'bytes': int(2 * ins + 2 * outs + 3 * weight + 2 * packed * values),
                'flops': 6 * values * case['out']}
    return {'bytes': values * size + width * case['out'] + 4 * case['out']
            + n * case['out'] * size, 'flops': 2 * values * case['out']}


# ---- inputs ----------------------------------------------------------------

def _package():
    from __graft_entry__ import load_package

    return load_package()


def prepare(case, seed):
    dev = torch.device('cuda')
    dtype = DTYPES[case['dtype']]
    gen = torch.Generator(device=dev).manual_seed(seed)
    n, width = case['tokens'], case['width']

    def normal(*shape, scale=1.0, kind=dtype):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(kind)

    state = {'case': case}
    leaves = []
    if case['kind'] == 'residual':
        # (a stream that has grown over some blocks, and a block's output)
        state['x'] = normal(n, width, scale=3.0, kind=DTYPES[case['stream']])
        state['update'] = normal(n, width, scale=0.7)
        if case['gate'] != 'none':
            rows = n if case['gate'] == 'element' else case['groups']
            state['gate'] = normal(rows, width, scale=0.5)
        if case['post']:
            state['update_weight'] = 1 + normal(width, scale=0.2)
        if case['scale']:
            state['scale'] = 0.5 + normal(width, scale=0.1)
        if case['norm']:
            state['weight'] = 1 + normal(width, scale=0.2)
        if case['grad']:
            state['dstream'] = normal(n, width, kind=DTYPES[case['stream']])
            if case['norm']:
                state['dnormed'] = normal(n, width)
        leaves = ['x', 'update', 'gate', 'update_weight', 'scale', 'weight']
    elif case['kind'] == 'gated':
        state['x'] = normal(n, 2 * width, scale=1.5)
        if case['grad']:
            state['dout'] = normal(n, width)
        leaves = ['x']
    elif case['kind'] == 'linear':
        state['x'] = normal(n, width)
        state['weight'] = normal(case['out'], width, scale=width ** -0.5)
        state['dout'] = normal(n, case['out'])
        if case['bias']:
            state['bias'] = normal(case['out'])
        leaves = ['x', 'weight', 'bias']
    else:
        # tokens of different magnitudes, and a layer's weights as they are
        # kept: codes and a scale for each channel, rows at multiples of 64
        # bytes
        size = torch.rand((n, 1), generator=gen, device=dev) * 2 + 0.2
        state['x'] = (torch.randn((n, width), generator=gen, device=dev) * size).to(dtype)
        weight = torch.randn((case['out'], width), generator=gen, device=dev) * width ** -0.5
        scales = weight.abs().amax(1) / 127
        pitch = (width + 63) // 64 * 64
        codes = torch.zeros((case['out'], pitch), dtype=torch.int8, device=dev)[:, :width]
        codes.copy_((weight / scales[:, None]).round())
        state['codes'], state['scales'] = codes, scales
        if case['bias']:
            state['bias'] = normal(case['out'])
    if case['grad']:
        for name in leaves:
            if name in state:
                state[name] = state[name].detach().requires_grad_(True)
    return state


# ---- one pass --------------------------------------------------------------

def run(state):
    kind = state['case']['kind']
    return {'residual': _run_residual, 'gated': _run_gated, 'linear': _run_linear,
            'int8': _run_int8}[kind](state)


RESIDUAL_INPUTS = ('x', 'update', 'gate', 'update_weight', 'scale', 'weight')


def _run_residual(s):
    case = s['case']
    names = [n for n in RESIDUAL_INPUTS if n in s]
    inputs = {n: s[n] for n in names}
    if own:
        x, update = inputs.pop('x'), inputs.pop('update')
        outs = _package().residual_norm(x, update, eps=EPS,
                                        checkpoint=8 if case['checkpoint'] else None, **inputs)
    else:
        outs = _plain_residual(case, **inputs)
    result = dict(zip(('stream', 'normed'), outs if case['norm'] else outs[:1]))
    if case['grad']:
        if not own and case['checkpoint']:  # the formula at what the checkpoint stands for
            for n in ('x', 'update'):
                inputs[n] = _kept(s[n].detach()).requires_grad_(True)
            outs = _plain_residual(case, **inputs)
            wrt = [inputs[n] for n in names]
        else:
            wrt = [s[n] for n in names]
        douts = [s[n] for n in ('dstream', 'dnormed') if n in s]
        grads = torch.autograd.grad([t for t in outs if t is not None], wrt, douts)
        result = {n: t.detach() for n, t in result.items()}
        result.update({'d' + n: g.to(s[n].dtype) for n, g in zip(names, grads)})
    return result


def _run_gated(s):
    case = s['case']
    if own:
        out = _package().gated_activation(s['x'], case['act'],
                                          checkpoint=8 if case['checkpoint'] else None)
    else:
        out = _plain_gated(case, s['x'])
    if not case['grad']:
        return {'out': out}
    if not own and case['checkpoint']:
        n, width = case['tokens'], case['width']
        x = _kept(s['x'].detach().view(n, 2, width)).view(n, 2 * width).requires_grad_(True)
        grad, = torch.autograd.grad(_plain_gated(case, x).to(s['dout'].dtype), x, s['dout'])
    else:
        grad, = torch.autograd.grad(out, s['x'], s['dout'])
    return {'out': out.detach(), 'dx': grad.to(s['x'].dtype)}


def _run_linear(s):
    if own:
        names = [n for n in ('x', 'weight', 'bias') if n in s]
        out = _package().checkpoint_linear(s['x'], s['weight'], s.get('bias'))
        grads = torch.autograd.grad(out, [s[n] for n in names], s['dout'])
        return {'out': out.detach(), **{'d' + n: g for n, g in zip(names, grads)}}
    dtype = s['x'].dtype
    with torch.no_grad():
        x, w, dout = s['x'].float(), s['weight'].float(), s['dout'].float()
        out = torch.matmul(x, w.T)
        if 'bias' in s:
            out = out + s['bias'].float()
        res = {'out': out, 'dx': torch.matmul(dout, w),
               'dweight': torch.matmul(dout.T.contiguous(), _kept(s['x']).float())}
        if 'bias' in s:
            res['dbias'] = dout.sum(0)
        return {n: t.to(dtype) for n, t in res.items()}


def _run_int8(s):
    if own:
        return {'out': _package().linear_int8(s['x'], s['codes'], s['scales'], s.get('bias'))}
    return {'out': _plain_int8(s)}


# ---- plain forms: elementary operations in 32 bits, rounded once -----------

def _power(exponent):
    """2 ** exponent in 64 bits, by its bits: exact (pow and exp2 need not be)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _kept(x):
    """What the 8-bit copy of x stands for (in fp32): blocks of 32 along the
    last dimension share the least power of two p with 127 p >= their largest
    magnitude; multiples of p, ties to even."""
    width = x.shape[-1]
    y = torch.nn.functional.pad(x.float(), (0, -width % BLOCK)).unflatten(-1, (-1, BLOCK))
    mantissa, exponent = torch.frexp(y.abs().amax(-1, keepdim=True))
    exponent = torch.where(mantissa > 127 / 128, exponent - 6, exponent - 7).clamp_min(-126)
    one = _power(exponent).float()
    return ((y / one).round() * one).flatten(-2)[..., :width].contiguous()


def _plain_norm(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_residual(case, x, update, gate=None, update_weight=None, scale=None, weight=None):
    dtype = DTYPES[case['dtype']]
    v = update.float()
    if update_weight is not None:
        v = _plain_norm(v, update_weight)
    if scale is not None:
        v = v * scale.float()
    if gate is not None:
        rows = gate.float()
        if case['gate'] == 'groups':
            rows = rows.repeat_interleave(case['tokens'] // case['groups'], 0)
        v = v * rows
    stream = x.float() + v
    normed = _plain_norm(stream, weight).to(dtype) if weight is not None else None
    return stream.to(DTYPES[case['stream']]), normed


def _plain_gated(case, x):
    a, b = x.float().chunk(2, -1)
    if case['act'] == 'gelu':
        y = 0.5 * a * (1 + torch.erf(a * math.sqrt(0.5)))
    else:
        y = 1 / (1 + torch.exp(-a))
        if case['act'] == 'silu':
            y = a * y
    return (y * b).to(DTYPES[case['dtype']])


def _token_codes(x):
    """(codes, scale) of each row in 64 bits: the least number of 8 mantissa
    bits (as bfloat16 has) with 127 scale >= the row's largest magnitude, at
    least 2^-126."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top / 127)
    scale = (torch.ceil(mantissa * 256) / 256 * _power(exponent)).clamp_min(2.0 ** -126)
    # (the quotient was rounded: a step up where that left it short)
    step = _power(torch.frexp(scale)[1] - 8)
    scale = torch.where(127 * scale < top, scale + step, scale)
    return (x / scale).round(), scale


def _plain_int8(s):
    codes, scale = _token_codes(s['x'])
    # (sums of whole numbers: exact while below 2^24, as they are by far here)
    out = torch.matmul(codes.float(), s['codes'].float().T)
    out = out * scale.float() * s['scales']
    if 'bias' in s:
        out = out + s['bias'].float()
    return out.to(s['x'].dtype)


# ---- the definitions in 64 bits --------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {'residual': _exact_residual, 'gated': _exact_gated, 'linear': _exact_linear,
                'int8': _exact_int8}[case['kind']](case, s)


def _floor_power(x):
    """The largest power of two that is at most x: its bits without those
    behind the point."""
    return (x.contiguous().view(torch.int64) & (0x7ff << 52)).view(torch.float64)


def _exact_kept(x):
    width = x.shape[-1]
    x = x.double()
    out = torch.empty_like(x)
    for i in range(0, width, BLOCK):
        part = x[..., i:i + BLOCK]
        top = part.abs().amax(-1, keepdim=True)
        # the least power of two by trying: 2^-126 and up
        p = _floor_power(top.clamp_min(1e-300) / 127) / 2
        for _ in range(3):
            p = torch.where(127 * p < top, 2 * p, p)
        p = p.clamp_min(2.0 ** -126)
        out[..., i:i + BLOCK] = torch.round(part / p) * p
    return out


def _exact_residual(case, s):
    gate = s['gate'].double() if 'gate' in s else 1.0
    if case['gate'] == 'groups':
        gate = gate.repeat_interleave(case['tokens'] // case['groups'], 0)
    w_u, scale, w = (s[n].double() if n in s else 1.0 for n in ('update_weight', 'scale',
                                                                'weight'))

    def root(t):
        return (t.square().mean(-1, keepdim=True) + EPS) ** -0.5

    def forward(x, u):
        r_u = root(u) if case['post'] else 1.0
        stream = x + scale * gate * (u * r_u * w_u)
        return stream, r_u

    x, u = s['x'].double(), s['update'].double()
    stream, r_u = forward(x, u)
    out = {'stream': stream}
    if case['norm']:
        out['normed'] = stream * root(stream) * w
    if not case['grad']:
        return out
    if case['checkpoint']:
        x, u = _exact_kept(s['x']), _exact_kept(s['update'])
        stream, r_u = forward(x, u)
    g, dw = s['dstream'].double(), None
    if case['norm']:
        dh, r = s['dnormed'].double(), root(stream)
        dw = (dh * stream * r).sum(0)
        g = g + r * (dh * w - stream * r ** 2 * (dh * w * stream).mean(-1, keepdim=True))
    n = u * r_u
    dn = g * scale * gate * w_u
    out['dx'] = g
    out['dupdate'] = r_u * (dn - n * (dn * n).mean(-1, keepdim=True)) if case['post'] else dn
    if 'gate' in s:
        dgate = g * scale * n * w_u
        if case['gate'] == 'groups':
            dgate = dgate.unflatten(0, (case['groups'], -1)).sum(1)
        out['dgate'] = dgate
    if case['post']:
        out['dupdate_weight'] = (g * scale * gate * n).sum(0)
    if case['scale']:
        out['dscale'] = (g * gate * n * w_u).sum(0)
    if case['norm']:
        out['dweight'] = dw
    return out


def _exact_gated(case, s):
    width = case['width']

    def act(t):
        """The function and its slope."""
        if case['act'] == 'gelu':
            p = torch.special.ndtr(t)
            return t * p, p + t * torch.exp(-t * t / 2) / math.sqrt(2 * math.pi)
        p = torch.sigmoid(t)
        if case['act'] == 'sigmoid':
            return p, p * torch.sigmoid(-t)
        return t * p, p + t * p * torch.sigmoid(-t)

    a, b = s['x'][:, :width].double(), s['x'][:, width:].double()
    out = {'out': act(a)[0] * b}
    if case['grad']:
        if case['checkpoint']:
            a, b = _exact_kept(s['x'][:, :width]), _exact_kept(s['x'][:, width:])
        y, slope = act(a)
        dy = s['dout'].double()
        out['dx'] = torch.cat((dy * b * slope, dy * y), 1)
    return out


def _exact_linear(case, s):
    x, w, dy = s['x'].double(), s['weight'].double(), s['dout'].double()
    out = {'out': x @ w.T + (s['bias'].double() if case['bias'] else 0.0), 'dx': dy @ w,
           'dweight': dy.T.contiguous() @ _exact_kept(s['x'])}
    if case['bias']:
        out['dbias'] = dy.sum(0)
    return out


def _exact_int8(case, s):
    x = s['x'].double()
    top = x.abs().amax(1, keepdim=True)
    # bfloat16 numbers around the largest magnitude over 127: the least that reaches it
    near = (top / 127).float().bfloat16().double()
    unit = _floor_power(near.clamp_min(2.0 ** -126)) / 128
    scale = torch.full_like(near, math.inf)
    for i in (2, 1, 0, -1, -2):
        t = near + i * unit
        scale = torch.where((127 * t >= top) & (t > 0), t, scale)
    codes = torch.round(x / scale.clamp_min(2.0 ** -126))
    out = (codes @ s['codes'].double().T) * scale * s['scales'].double()
    return {'out': out + s['bias'].double() if case['bias'] else out}
