"""The token operators that stand after the pooling, as they are measured:
norm and rotation of queries and keys, attention over packed sequences, and
attention of new tokens over caches that share a prefix.

A case is a dict of plain values:

  kind      'rotate'  norm_rotate
            'packed'  attend_packed
            'cached'  attend_cached
  grad      True: forward and the gradients of every input; False: forward
  dtype, q_heads, k_heads, dim   type, heads and size of a head

  'rotate'  tokens; pairs_0, pairs_1, pairs_2: rotated pairs of each axis
            (0: the axis is absent); norm: with weights; interleaved: layout
            of a pair; fw, fh: the tokens are maps of fh rows and fw columns
            (frame, row, column), or text after them where fw is 0 (start:
            position of the first token)
  'packed'  sequences, longest, spread: their numbers of queries, longest *
            (rank / sequences) ** spread (0: all alike), at least 1, in an
            order drawn by the seed; context: keys before a sequence's first
            query; causal
  'cached'  requests, new: requests and the new tokens of each; capacity,
            shortest: slots of a cache, and the least of its keys in use (the
            most is capacity; evenly between, in an order drawn by the seed);
            prefix: shared keys (0: none)
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
SIZE = {'f32': 4, 'f16': 2, 'bf16': 2}

ROTATE = {'kind': 'rotate', 'grad': True, 'dtype': 'bf16', 'tokens': 6 * 32 * 88, 'q_heads': 16,
          'k_heads': 16, 'dim': 80, 'pairs_0': 8, 'pairs_1': 16, 'pairs_2': 16, 'norm': True,
          'interleaved': False, 'fh': 32, 'fw': 88, 'start': 0}
PACKED = {'kind': 'packed', 'grad': True, 'dtype': 'bf16', 'sequences': 6, 'longest': 32 * 88,
          'spread': 0.0, 'context': 0, 'causal': False, 'q_heads': 16, 'k_heads': 16, 'dim': 80}
CACHED = {'kind': 'cached', 'grad': False, 'dtype': 'bf16', 'requests': 64, 'new': 1,
          'capacity': 1024, 'shortest': 1, 'prefix': 6 * 32 * 88, 'q_heads': 32, 'k_heads': 8,
          'dim': 128}


def listed():
    return [
        # the next token of 16 requests after a prompt: latency
        dict(ROTATE, name='rotate_token', grad=False, tokens=16, q_heads=32, k_heads=8, dim=128,
             pairs_0=16, pairs_1=24, pairs_2=24, fh=0, fw=0, start=20011),
        # the tokens of six cameras' feature maps, one training step
        dict(ROTATE, name='rotate_cameras_step'),
        # a BEV map of 180 x 180 in single precision, as the pooling leaves it
        dict(ROTATE, name='rotate_bev_f32_step', dtype='f32', tokens=180 * 180, q_heads=8,
             k_heads=8, dim=64, pairs_0=0, pairs_1=16, pairs_2=16, fh=180, fw=180),
        # a long prompt's queries and keys, rotated only, a part of each head,
        # in the layout of neighbouring elements; sizes that fit nothing
        dict(ROTATE, name='rotate_odd_infer', grad=False, dtype='f16', tokens=30011, q_heads=7,
             k_heads=1, dim=72, pairs_0=27, pairs_1=0, pairs_2=0, norm=False, interleaved=True,
             fh=0, fw=0),
        # a few short prompts, one step: launches and latency
        dict(PACKED, name='packed_short_step', dtype='f16', sequences=5, longest=77, spread=2.0,
             causal=True, q_heads=8, k_heads=2, dim=64),
        # attention within each of six cameras' maps, one training step
        dict(PACKED, name='packed_cameras_step'),
        # prompts of very different lengths, one training step
        dict(PACKED, name='packed_prompts_step', sequences=11, longest=4096, spread=1.7,
             causal=True, q_heads=16, k_heads=4, dim=128),
        # one long prompt, forward
        dict(PACKED, name='packed_long_infer', grad=False, sequences=1, longest=32768,
             causal=True, q_heads=8, k_heads=1, dim=128),
        # windows of a BEV map in single precision, one step
        dict(PACKED, name='packed_f32_step', dtype='f32', sequences=9, longest=900, q_heads=4,
             k_heads=4, dim=32),
        # one request's next token after a prompt of odd length: latency
        dict(CACHED, name='cached_token', requests=1, capacity=4099, shortest=4099, prefix=0),
        # 64 questions about one scene: six cameras' tokens shared by all
        dict(CACHED, name='cached_scene'),
        # drafted tokens of 24 requests with long caches of their own
        dict(CACHED, name='cached_drafts', dtype='f16', requests=24, new=4, capacity=16384,
             shortest=300, prefix=0, dim=64),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        kind = rng.choice(['rotate', 'packed', 'cached'])
        k_heads = rng.choice([1, 2, 3, 4, 8, 16])
        heads = {'dtype': rng.choice(['bf16', 'bf16', 'f16', 'f32']), 'k_heads': k_heads,
                 'q_heads': k_heads * rng.choice([1, 2, 4, 7, 8]),
                 'dim': rng.choice([32, 64, 72, 80, 96, 128])}
        if kind == 'rotate':
            case = dict(ROTATE, **heads)
            case['grad'] = rng.random() < 0.6
            case['tokens'] = log_int(1, 40000)
            case['norm'] = rng.random() < 0.7
            case['interleaved'] = rng.random() < 0.3
            half = case['dim'] // 2
            if rng.random() < 0.5:  # maps
                case['fh'], case['fw'] = rng.randint(8, 64), rng.randint(16, 128)
                case['pairs_0'] = half // 5
                case['pairs_1'] = case['pairs_2'] = (half - case['pairs_0']) // 2
            else:
                case['fh'] = case['fw'] = 0
                # (single precision: as far as the plain form's own angles go)
                case['start'] = log_int(1, 30000 if case['dtype'] != 'f32' else 64)
                case['tokens'] = min(case['tokens'], 300 if case['dtype'] == 'f32' else 40000)
                case['pairs_0'] = rng.choice([half, half - 3, half // 2])
                case['pairs_1'] = case['pairs_2'] = 0
        elif kind == 'packed':
            case = dict(PACKED, **heads)
            case['grad'] = rng.random() < 0.6
            case['sequences'] = log_int(1, 40)
            case['longest'] = log_int(8, 16384)
            case['spread'] = rng.choice([0.0, 1.0, 2.0])
            case['causal'] = rng.random() < 0.6
            case['context'] = rng.choice([0, 0, log_int(1, 2048)])
        else:
            case = dict(CACHED, **heads)
            case['requests'] = log_int(1, 128)
            case['new'] = rng.choice([1, 1, 1, 2, 5])
            case['capacity'] = log_int(64, 32768)
            case['shortest'] = rng.randint(max(1, case['new']), case['capacity'])
            case['prefix'] = rng.choice([0, log_int(100, 32768)])
        if _fits(case):
            return case


def _fits(case):
    """No dearer than the largest listed ones: scores of the plain form, and
    bytes of a cache."""
    if case['kind'] == 'rotate':
        return (case['tokens'] * (case['q_heads'] + case['k_heads']) * case['dim']
                <= 6 * 32 * 88 * 32 * 80)
    if case['kind'] == 'packed':
        longest = case['longest']
        scores = case['sequences'] * case['q_heads'] * longest * (longest + case['context'])
        return scores * (case['dim'] if case['dtype'] == 'f32' else 32) <= (
            32 * (2.9e9 if case['grad'] else 8.5e9))
    keys = case['requests'] * case['capacity'] + case['prefix']
    scores = case['requests'] * case['new'] * case['q_heads'] * (case['capacity'] + case['prefix'])
    return (keys * case['k_heads'] * case['dim'] * SIZE[case['dtype']]
            <= 24 * 16384 * 8 * 64 * 2 and scores <= 3e8)


# ---- sizes -----------------------------------------------------------------

def _lengths(case):
    n = case['sequences']
    return [max(1, round(case['longest'] * ((i + 1) / n) ** case['spread'])) for i in range(n)]


def _cache_lengths(case):
    n, low, high = case['requests'], case['shortest'], case['capacity']
    low = max(low, case['new'])
    return [high - (high - low) * i // max(1, n - 1) for i in range(n)]


def _pairs(case):
    return [case[k] for k in ('pairs_0', 'pairs_1', 'pairs_2') if case[k]]


def work(case):
    size, dim, hq, hk = SIZE[case['dtype']], case['dim'], case['q_heads'], case['k_heads']
    if case['kind'] == 'rotate':
        values = case['tokens'] * (hq + hk) * dim
        passes = 5 if case['grad'] else 2  # x, y; and dy, x again, dx
        return {'bytes': passes * values * size, 'flops': (24 if case['grad'] else 9) * values}
    if case['kind'] == 'packed':
        lengths, context = _lengths(case), case['context']
        tokens = sum(lengths)
        keys = tokens + context * len(lengths)
        pairs = sum(n * context + (n * (n + 1) // 2 if case['causal'] else n * n)
                    for n in lengths)
        q, kv = tokens * hq * dim, 2 * keys * hk * dim
        moved = 2 * q + kv
        if case['grad']:
            moved += 3 * q + 2 * kv  # out, dout and dq; k, v and their gradients
        return {'bytes': moved * size, 'flops': (14 if case['grad'] else 4) * dim * hq * pairs}
    keys, new, rows = sum(_cache_lengths(case)), case['new'], case['requests'] * case['new']
    pairs = (keys - case['requests'] * (new - 1) / 2) * new + rows * case['prefix']
    return {'bytes': int((2 * (keys + case['prefix']) * hk + 2 * rows * hq) * dim * size),
            'flops': int(4 * dim * hq * pairs)}


# ---- inputs ----------------------------------------------------------------

def _package():
    from __graft_entry__ import load_package

    return load_package()


def _frequencies(case):
    """10000 ** (-i / pairs), a ladder of its own for each axis."""
    return torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
                      for n in _pairs(case)]).float()


def _positions(case):
    i = torch.arange(case['tokens'])
    if case['fw']:
        maps = torch.stack((i // (case['fh'] * case['fw']), i // case['fw'] % case['fh'],
                            i % case['fw']), 1)
        return maps[:, [case['pairs_0'] > 0, True, True]]
    return (case['start'] + i)[:, None].expand(-1, len(_pairs(case))).contiguous()


def prepare(case, seed):
    dev = torch.device('cuda')
    dtype = DTYPES[case['dtype']]
    gen = torch.Generator(device=dev).manual_seed(seed)
    order = random.Random(seed)
    hq, hk, dim = case['q_heads'], case['k_heads'], case['dim']

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dtype)

    def starts(lengths):
        return torch.tensor([0] + lengths).cumsum(0).to(dev, torch.int32)

    state = {'case': case}
    if case['kind'] == 'rotate':
        # queries and keys are parts of one projection's rows, as a model has them
        rows = normal(case['tokens'], (hq + 2 * hk) * dim)
        state['q'] = rows[:, :hq * dim].view(-1, hq, dim)
        state['k'] = rows[:, hq * dim:(hq + hk) * dim].view(-1, hk, dim)
        state['positions'] = _positions(case).to(dev, torch.int32)
        state['frequencies'] = _frequencies(case).to(dev)
        if case['norm']:
            state['q_weight'] = 1 + normal(dim, scale=0.2)
            state['k_weight'] = 1 + normal(dim, scale=0.2)
        if case['grad']:
            state['dq'], state['dk'] = normal(case['tokens'], hq, dim), normal(case['tokens'], hk,
                                                                              dim)
    elif case['kind'] == 'packed':
        lengths = _lengths(case)
        order.shuffle(lengths)
        keys = [n + case['context'] for n in lengths]
        state['q'] = normal(sum(lengths), hq, dim)
        state['k'] = normal(sum(keys), hk, dim)
        state['v'] = normal(sum(keys), hk, dim)
        state['q_starts'], state['k_starts'] = starts(lengths), starts(keys)
        if case['grad']:
            state['dout'] = normal(sum(lengths), hq, dim)
    else:
        lengths = _cache_lengths(case)
        order.shuffle(lengths)
        state['q'] = normal(case['requests'], case['new'], hq, dim)
        state['k'] = normal(case['requests'], case['capacity'], hk, dim)
        state['v'] = normal(case['requests'], case['capacity'], hk, dim)
        state['lengths'] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        if case['prefix']:
            state['prefix_k'] = normal(case['prefix'], hk, dim)
            state['prefix_v'] = normal(case['prefix'], hk, dim)
    if case['grad']:
        for name in ('q', 'k', 'v', 'q_weight', 'k_weight'):
            if name in state:
                state[name] = state[name].detach().requires_grad_(True)
    return state


# ---- one pass --------------------------------------------------------------

def run(state):
    case = state['case']
    return {'rotate': _run_rotate, 'packed': _run_packed, 'cached': _run_cached}[case['kind']](state)


def _run_rotate(s):
    case = s['case']
    weights = {k: s[k] for k in ('q_weight', 'k_weight') if k in s}
    if own:
        q, k = _package().norm_rotate(s['q'], s['k'], s['positions'], s['frequencies'],
                                      _pairs(case), interleaved=case['interleaved'], **weights)
    else:
        q = _plain_rotate(s, s['q'], weights.get('q_weight'))
        k = _plain_rotate(s, s['k'], weights.get('k_weight'))
    out = {'q': q, 'k': k}
    if case['grad']:
        names = ['q', 'k'] + list(weights)
        grads = torch.autograd.grad((q, k), [s[n] for n in names], (s['dq'], s['dk']))
        out.update({'d' + n: g for n, g in zip(names, grads)})
    return {n: t.detach() for n, t in out.items()}


def _run_packed(s):
    case = s['case']
    if own:
        out = _package().attend_packed(s['q'], s['k'], s['v'], s['q_starts'], s['k_starts'],
                                       causal=case['causal'])
    else:
        out = _plain_packed(s)
    if not case['grad']:
        return {'out': out}
    grads = torch.autograd.grad(out, (s['q'], s['k'], s['v']), s['dout'])
    return {'out': out.detach(), 'dq': grads[0], 'dk': grads[1], 'dv': grads[2]}


def _run_cached(s):
    if own:
        return {'out': _package().attend_cached(s['q'], s['k'], s['v'], s['lengths'],
                                                s.get('prefix_k'), s.get('prefix_v'))}
    return {'out': _plain_cached(s)}


# ---- plain forms: elementary operations in 32 bits, rounded once -----------

def _plain_rotate(s, x, weight):
    case = s['case']
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
    sizes = torch.tensor(_pairs(case))
    axis = torch.repeat_interleave(torch.arange(len(sizes)), sizes).to(x.device)
    angle = (s['positions'].float()[:, axis] * s['frequencies'])[:, None, :]
    cos, sin = angle.cos(), angle.sin()
    n = angle.shape[-1]
    if case['interleaved']:
        a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :n], y[..., n:2 * n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., 2 * n:]), -1).to(x.dtype)


def _attend(scores, seen, values):
    """softmax of the seen scores times values; rows that see nothing give 0."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.detach().amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    return torch.matmul(p, values) / p.sum(-1, keepdim=True).clamp_min(1e-37)


def _plain_packed(s):
    case = s['case']
    hq, hk, dim = case['q_heads'], case['k_heads'], case['dim']
    dev = s['q'].device

    def padded(starts, most):
        n = starts[1:] - starts[:-1]
        i = torch.arange(most, device=dev)
        return n, (starts[:-1, None] + i).clamp_max(starts[-1] - 1).long(), i < n[:, None]

    nq, q_rows, q_in = padded(s['q_starts'], case['longest'])
    nk, k_rows, k_in = padded(s['k_starts'], case['longest'] + case['context'])
    (S, Lq), Lk = q_rows.shape, k_rows.shape[1]
    q = s['q'].float()[q_rows].view(S, Lq, hk, hq // hk, dim).permute(0, 2, 3, 1, 4)
    k = s['k'].float()[k_rows].permute(0, 2, 3, 1).unsqueeze(2)
    v = s['v'].float()[k_rows].permute(0, 2, 1, 3).unsqueeze(2)
    scores = torch.matmul(q, k) * dim ** -0.5
    seen = k_in[:, None, :]
    if case['causal']:
        last = torch.arange(Lq, device=dev)[None, :] + (nk - nq)[:, None]
        seen = seen & (torch.arange(Lk, device=dev) <= last[:, :, None])
    out = _attend(scores, seen[:, None, None], v)
    return out.permute(0, 3, 1, 2, 4).reshape(S, Lq, hq, dim)[q_in].to(s['q'].dtype)


def _plain_cached(s):
    case = s['case']
    B, n, hq, dim = s['q'].shape
    hk = case['k_heads']
    cap = case['capacity']
    dev = s['q'].device
    q = s['q'].float().view(B, n, hk, hq // hk, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(B, hk, -1, dim)
    scores = torch.matmul(q, s['k'].float().permute(0, 2, 3, 1))
    last = s['lengths'][:, None] - n + torch.arange(n, device=dev)
    seen = torch.arange(cap, device=dev) <= last[:, :, None]
    seen = seen[:, None, None].expand(B, 1, hq // hk, n, cap).reshape(B, 1, -1, cap)
    scores = scores.masked_fill(~seen, -math.inf)
    if case['prefix']:
        shared = torch.matmul(q.transpose(0, 1).reshape(hk, -1, dim),
                              s['prefix_k'].float().permute(1, 2, 0))
        shared = shared.view(hk, B, -1, case['prefix']).transpose(0, 1)
        scores = torch.cat((shared, scores), -1)
    p = torch.exp((scores - scores.amax(-1, keepdim=True)) * dim ** -0.5)
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p[..., -cap:], s['v'].float().permute(0, 2, 1, 3))
    if case['prefix']:
        rows = p[..., :-cap].transpose(0, 1).reshape(hk, -1, case['prefix'])
        shared = torch.matmul(rows, s['prefix_v'].float().transpose(0, 1))
        out = out + shared.view(hk, B, -1, dim).transpose(0, 1)
    out = out.view(B, hk, hq // hk, n, dim).permute(0, 3, 1, 2, 4)
    return out.reshape(B, n, hq, dim).to(s['q'].dtype)


# ---- the definitions in 64 bits --------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {'rotate': _exact_rotate, 'packed': _exact_packed,
                'cached': _exact_cached}[case['kind']](case, s)


def _exact_rotate(case, s):
    """Each pair as a complex number, times exp(i angle); the gradient by the
    conjugate."""
    pos, freq, turns = s['positions'].double(), s['frequencies'].double(), []
    for axis, n in enumerate(_pairs(case)):
        i = sum(_pairs(case)[:axis])
        turns.append(pos[:, axis, None] * freq[i:i + n])
    angle = torch.cat(turns, 1)[:, None]
    turn, n = torch.polar(torch.ones_like(angle), angle), angle.shape[-1]

    def rotate(y, by):
        flat = y[..., :2 * n]
        if case['interleaved']:
            z = torch.view_as_complex(flat.reshape(*flat.shape[:-1], n, 2)) * by
            flat = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(flat[..., :n], flat[..., n:]) * by
            flat = torch.cat((z.real, z.imag), -1)
        return torch.cat((flat, y[..., 2 * n:]), -1)

    out, grads, weights = {}, {}, {}
    for name in ('q', 'k'):
        x = s[name].double()
        w, r = 1.0, 1.0
        if case['norm']:
            w = s[name + '_weight'].double()
            r = (x.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
        out[name] = rotate(x * r * w, turn)
        if case['grad']:
            g = rotate(s['d' + name].double(), turn.conj())
            if case['norm']:
                weights[f'd{name}_weight'] = (g * x * r).sum((0, 1))
                g = r * (g * w) - x * r ** 3 * (g * w * x).mean(-1, keepdim=True)
            grads['d' + name] = g
    return {**out, **grads, **weights}


def _exact_packed(case, s):
    q, k, v = s['q'].double(), s['k'].double(), s['v'].double()
    group = case['q_heads'] // case['k_heads']
    scale = 1.0 / math.sqrt(case['dim'])
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    q_at, k_at = s['q_starts'].tolist(), s['k_starts'].tolist()
    for n in range(case['sequences']):
        a, b, c, d = q_at[n], q_at[n + 1], k_at[n], k_at[n + 1]
        for h in range(case['q_heads']):
            g = h // group
            for i in range(a, b, 8192):  # (rows at a time, for the memory)
                e = min(b, i + 8192)
                x = q[i:e, h] @ k[c:d, g].T * scale
                if case['causal']:
                    over = torch.ones_like(x, dtype=torch.bool).triu((d - c) - (b - a) + i - a + 1)
                    x[over] = -math.inf
                p = x.softmax(-1)
                out[i:e, h] = p @ v[c:d, g]
                if case['grad']:
                    do = s['dout'][i:e, h].double()
                    t = do @ v[c:d, g].T
                    ds = p * (t - (p * t).sum(-1, keepdim=True)) * scale
                    dq[i:e, h] = ds @ k[c:d, g]
                    dk[c:d, g] += ds.T @ q[i:e, h]
                    dv[c:d, g] += p.T @ do
    return {'out': out, 'dq': dq, 'dk': dk, 'dv': dv} if case['grad'] else {'out': out}


def _exact_cached(case, s):
    q = s['q'].double()
    group = case['q_heads'] // case['k_heads']
    out = torch.zeros_like(q)
    lengths = s['lengths'].tolist()
    for b in range(case['requests']):
        k, v = s['k'][b, :lengths[b]].double(), s['v'][b, :lengths[b]].double()
        if case['prefix']:
            k = torch.cat((s['prefix_k'].double(), k))
            v = torch.cat((s['prefix_v'].double(), v))
        k, v = (t.repeat_interleave(group, 1).transpose(0, 1).contiguous() for t in (k, v))
        for i in range(case['new']):
            n = k.shape[1] - (case['new'] - 1 - i)
            p = (torch.matmul(k[:, :n], q[b, i, :, :, None])[..., 0] / case['dim'] ** 0.5).softmax(-1)
            out[b, i] = (p[:, :, None] * v[:, :n]).sum(1)
    return {'out': out}
