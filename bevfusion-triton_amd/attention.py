"""Token operators on MI355X: norm and rotation of queries and keys, and
attention over packed sequences.

What a transformer over camera and BEV tokens needs after the pooling, as HIP
kernels behind the same C ABI (``include/bevpool.h``); the reference has no
counterpart.

  * :func:`norm_rotate`      RMS norm of each head and rotary positions with
                             several axes (frame, row, column), one pass
  * :func:`axis_frequencies` the usual frequency ladders for it
  * :func:`attend_packed`    attention over packed sequences of different
                             lengths, causal or not, grouped heads
  * :func:`attend_cached`    its form for serving: new tokens of many requests
                             over their caches and a prefix that all share

The first two have gradients.  Operands are fp32, fp16 or bf16 (rows, heads,
dim) tensors; any strides are taken, so parts of one projection's output need
no copy (attention copies an operand whose rows or heads do not start at
multiples of 16 bytes; a cache that does not is refused).  Calls run on torch's current stream, allocate with
torch's allocator and never wait for the device.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import _pipeline as P

_POSITION_KINDS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
MAX_AXES = 4


def axis_frequencies(pairs, base=10000.0, *, shared=False, device=None):
    """Frequencies (radians per unit of position) of ``sum(pairs)`` rotated
    pairs, ``pairs[i]`` of them turned by axis i: ``base ** (-j / n)``.  Each
    axis has a ladder of its own (j, n within the axis), or, with ``shared``,
    all share one over all the pairs in order."""
    pairs = [int(n) for n in pairs]
    if any(n < 0 for n in pairs):
        raise ValueError('pairs must not be negative')
    ladders = [sum(pairs)] if shared else pairs
    parts = [float(base) ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in ladders]
    return torch.cat(parts).to(device, torch.float32)


def _check_rows(name, x, dims=3):
    if x.dim() != dims:
        raise ValueError(f'{name} must have {dims} dimensions (..., heads, dim).')
    if x.dtype not in L.DTYPE_CODES:
        raise TypeError(f'{name} must have dtype torch.float16, torch.float32, or torch.bfloat16.')


def _check_same(name, x, like):
    if x.dtype != like.dtype:
        raise TypeError(f'{name} must have the dtype of q ({like.dtype}).')
    if x.device != like.device:
        raise ValueError(f'{name} must be on the device of q ({like.device}).')


def _unit(x):
    """x with unit stride along its last dimension."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _strides(x):
    return (x.data_ptr(), *x.stride()[:2]) if x is not None else (0, 0, 0)


def _run(call, device, what):
    """call(library, stream) on the device's current stream.  (Where the device
    is current already, as it mostly is, without the context manager.)"""
    if device.index == torch._C._cuda_getDevice():
        status = call(L.library(), torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            status = call(L.library(), L.stream_handle(device))
    L.check(status, what)


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _recorded():
    """Whether something other than a gradient follows the calls: tangents,
    which the autograd functions refuse (a result without one would stand for
    a derivative of zero), or a trace, which records the functions as they are
    (it does not see the library's calls)."""
    return forward_ad._current_level >= 0 or torch._C._get_tracing_state() is not None


# ---- norm and rotation -----------------------------------------------------

def _norm_rotate(q, k, q_weight, k_weight, positions, frequencies, pairs, eps, interleaved):
    tokens, q_heads, dim = q.shape
    k_heads = k.shape[1] if k is not None else 0
    q_out = q.new_empty(q.shape)
    k_out = None if k is None else k.new_empty(k.shape)
    _run(lambda lib, s: lib.bevpool_norm_rotate_forward(
        *_strides(q), q_heads, *_strides(k), k_heads, L.DTYPE_CODES[q.dtype], tokens, dim,
        *_rotation(positions, frequencies, pairs, interleaved), L.ptr(q_weight), L.ptr(k_weight),
        eps, L.ptr(q_out), L.ptr(k_out), s), q.device, 'bevpool_norm_rotate_forward')
    return q_out, k_out


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, frequencies, pairs, eps, interleaved):
        tokens, q_heads, dim = q.shape
        k_heads = k.shape[1] if k is not None else 0
        ctx.call = (tokens, q_heads, k_heads, dim, q.dtype, pairs, eps, interleaved)
        # (a rotation alone needs no input for its gradient)
        ctx.save_for_backward(q if q_weight is not None else None,
                              k if k_weight is not None else None, q_weight, k_weight, positions,
                              frequencies)
        return _norm_rotate(q, k, q_weight, k_weight, positions, frequencies, pairs, eps,
                            interleaved)

    @staticmethod
    @once_differentiable  # (the gradients are no functions of the graph's)
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, positions, frequencies = ctx.saved_tensors
        tokens, q_heads, k_heads, dim, dtype, pairs, eps, interleaved = ctx.call
        dev = positions.device

        # (None: of a k that is not there; an output that nothing was computed
        # from has a gradient of zeros)
        dq_out, dk_out = (g if g is None else _unit(g if g.dtype == dtype else g.to(dtype))
                          for g in (dq_out, dk_out))
        dq, dk = (g if g is None else g.new_empty(g.shape) for g in (dq_out, dk_out))
        dqw = torch.empty_like(q_weight) if q_weight is not None else None
        dkw = torch.empty_like(k_weight) if k_weight is not None else None
        lib = L.library()
        nbytes = lib.bevpool_norm_rotate_backward_scratch_bytes(dim)
        normed = dqw is not None or dkw is not None
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if normed else None
        _run(lambda lib, s: lib.bevpool_norm_rotate_backward(
            *_strides(q), q_heads, *_strides(k), k_heads, *_strides(dq_out), *_strides(dk_out),
            L.DTYPE_CODES[dtype], tokens, dim,
            *_rotation(positions, frequencies, pairs, interleaved), L.ptr(q_weight),
            L.ptr(k_weight), eps, L.ptr(dq), L.ptr(dk), L.ptr(dqw), L.ptr(dkw), L.ptr(scratch),
            nbytes if normed else 0, s), dev, 'bevpool_norm_rotate_backward')
        return dq, dk, dqw, dkw, None, None, None, None, None


def _rotation(positions, frequencies, pairs, interleaved):
    return (L.ptr(positions), _POSITION_KINDS[positions.dtype],
            positions.stride(0) if positions.shape[0] else 0, L.ptr(frequencies),
            _counts(pairs), len(pairs), int(interleaved))


@functools.lru_cache(maxsize=64)
def _counts(pairs):
    return (ctypes.c_int32 * max(1, len(pairs)))(*pairs)


def norm_rotate(q, k, positions, frequencies, pairs=None, *, q_weight=None, k_weight=None,
                eps=1e-6, interleaved=False):
    """RMS norm of queries and keys for each head (where a weight is given),
    then rotation by positions with several axes; returns (q, k) contiguous.

    q (tokens, q_heads, dim) and k (tokens, k_heads, dim) or None, dim even and
    at most 256.  positions (tokens,) or (tokens, axes), int32, int64 or
    float32.  frequencies (P,) fp32, 2 P <= dim; ``pairs[i]`` of them (in
    order, ``sum(pairs) == P``; default: all, one axis) turn by axis i.  Pair p
    is the elements (p, P + p) of a head, or (2p, 2p + 1) with
    ``interleaved``; the elements from 2 P on are not turned.  q_weight,
    k_weight (dim,): n = x / sqrt(mean(x^2) + eps) * weight in fp32.
    Gradients flow to q, k and the weights."""
    _check_rows('q', q)
    tokens, _, dim = q.shape
    if k is not None:
        _check_rows('k', k)
        _check_same('k', k, q)
        if k.shape[0] != tokens or k.shape[2] != dim:
            raise ValueError('q and k must agree on tokens and dim.')
    elif k_weight is not None:
        raise ValueError('k_weight without k.')
    if dim % 2 or not 2 <= dim <= 256:
        raise ValueError('dim must be even and at most 256.')
    if positions.dim() == 1:
        positions = positions.unsqueeze(1)
    if positions.dim() != 2 or positions.shape[0] != tokens:
        raise ValueError('positions must have shape [tokens] or [tokens, axes].')
    if positions.dtype not in _POSITION_KINDS:
        raise TypeError('positions must have dtype torch.int32, torch.int64 or torch.float32.')
    if frequencies.dim() != 1 or frequencies.dtype != torch.float32:
        raise ValueError('frequencies must be a 1-d float32 tensor.')
    pairs = (int(frequencies.shape[0]),) if pairs is None else tuple(int(n) for n in pairs)
    if len(pairs) > MAX_AXES or any(n < 0 for n in pairs):
        raise ValueError(f'pairs must be at most {MAX_AXES} numbers, none negative.')
    if sum(pairs) != frequencies.shape[0] or 2 * sum(pairs) > dim:
        raise ValueError('pairs must sum to the number of frequencies, at most dim / 2.')
    if positions.shape[1] < len(pairs):
        raise ValueError('positions must have a column for each axis.')
    if not eps >= 0:
        raise ValueError('eps must not be negative.')
    for name, w in (('q_weight', q_weight), ('k_weight', k_weight)):
        if w is not None:
            if tuple(w.shape) != (dim,):
                raise ValueError(f'{name} must have shape [dim].')
            _check_same(name, w, q)
    P.require_gpu(q, positions, frequencies, *[t for t in (k, q_weight, k_weight) if t is not None])
    for name, t in (('positions', positions), ('frequencies', frequencies)):
        if t.device != q.device:
            raise ValueError(f'{name} must be on the device of q ({q.device}).')
    weights = [w if w is None else w.contiguous() for w in (q_weight, k_weight)]
    run = _NormRotate.apply if _wants_grad(q, k, *weights) or _recorded() else _norm_rotate
    return run(_unit(q), _unit(k) if k is not None else None, *weights, _unit(positions),
               frequencies.contiguous(), pairs, float(eps), bool(interleaved))


# ---- attention over packed sequences ---------------------------------------

def _aligned(x, group=1):
    """x (rows, heads, dim) with unit stride along dim, every row and head at a
    multiple of 16 bytes, and strides whose multiples over a tile (64 rows,
    the heads of a group) the kernels form in 32 bits: itself, or a copy."""
    size = x.element_size()
    row, head, one = x.stride()
    row, head = row * size, head * size
    if (one == 1 and row % 16 == 0 and head % 16 == 0 and row < 1 << 24
            and head * group < 1 << 30 and x.data_ptr() % 16 == 0):
        return x
    # (not contiguous(): a dimension of one keeps whatever stride it has there)
    return x.clone(memory_format=torch.contiguous_format)


def _check_heads(q, k, v):
    for name, x in (('k', k), ('v', v)):
        _check_same(name, x, q)
    if k.shape != v.shape:
        raise ValueError('k and v must have the same shape.')
    dim = q.shape[-1]
    if k.shape[-1] != dim:
        raise ValueError('q and k must have the same dim.')
    if dim % 8 or not 8 <= dim <= 128:
        raise ValueError('dim must be a multiple of 8, at most 128.')
    if q.shape[-2] < 1 or k.shape[-2] < 1 or q.shape[-2] % k.shape[-2]:
        raise ValueError('the number of query heads must be a multiple of that of key heads.')


def _check_scale(scale, dim):
    scale = float(dim) ** -0.5 if scale is None else float(scale)
    if not 1e-30 <= scale < float('inf'):
        raise ValueError('scale must be positive (1e-30 or more) and finite.')
    return scale


def _check_starts(name, starts, like):
    if starts.dim() != 1 or starts.shape[0] < 1:
        raise ValueError(f'{name} must have shape [sequences + 1].')
    if starts.dtype not in (torch.int32, torch.int64):
        raise TypeError(f'{name} must have dtype torch.int32 or torch.int64.')
    if starts.device != like.device:
        raise ValueError(f'{name} must be on the device of q ({like.device}).')
    if starts.dtype == torch.int32 and starts.is_contiguous():
        return starts
    return starts.to(torch.int32).contiguous()


def _attend_packed(q, k, v, q_starts, k_starts, causal, scale, rest=None):
    out = q.new_empty(q.shape)
    lse = q.new_empty(q.shape[:2], dtype=torch.float32)
    _run(lambda lib, s: lib.bevpool_attention_forward(
        *_strides(q), *_strides(k), *_strides(v), L.DTYPE_CODES[q.dtype], q.shape[0], k.shape[0],
        q.shape[1], k.shape[1], q.shape[2], L.ptr(q_starts), L.ptr(k_starts),
        q_starts.shape[0] - 1, int(causal), scale, L.ptr(out), L.ptr(rest), L.ptr(lse), s), q.device,
        'bevpool_attention_forward')
    return out, lse


class _AttendPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_starts, k_starts, causal, scale):
        # (16-bit types: the output's rounding, for the gradients)
        rest = q.new_empty(q.shape) if q.element_size() == 2 else None
        out, lse = _attend_packed(q, k, v, q_starts, k_starts, causal, scale, rest)
        ctx.save_for_backward(q, k, v, out, rest, lse, q_starts, k_starts)
        ctx.call = (causal, scale)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable  # (the gradients are no functions of the graph's)
    def backward(ctx, dout, _):
        q, k, v, out, rest, lse, q_starts, k_starts = ctx.saved_tensors
        causal, scale = ctx.call
        if dout.dtype != q.dtype:
            dout = dout.to(q.dtype)
        dout = _aligned(dout, q.shape[1] // k.shape[1])
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        nbytes = L.library().bevpool_attention_backward_scratch_bytes(
            q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], L.DTYPE_CODES[q.dtype],
            q_starts.shape[0] - 1)
        scratch = q.new_empty(nbytes, dtype=torch.uint8)
        _run(lambda lib, s: lib.bevpool_attention_backward(
            *_strides(q), *_strides(k), *_strides(v), L.ptr(out), L.ptr(rest), *_strides(dout), L.ptr(lse),
            L.DTYPE_CODES[q.dtype], q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2],
            L.ptr(q_starts), L.ptr(k_starts), q_starts.shape[0] - 1, int(causal), scale, L.ptr(dq),
            L.ptr(dk), L.ptr(dv), L.ptr(scratch), nbytes, s), q.device,
            'bevpool_attention_backward')
        return dq, dk, dv, None, None, None, None


def attend_packed(q, k, v, q_starts, k_starts=None, *, causal=False, scale=None,
                  return_lse=False):
    """Attention within packed sequences of different lengths.

    q (q_total, q_heads, dim), k and v (k_total, k_heads, dim), q_heads a
    multiple of k_heads (query head h reads key head h // (q_heads /
    k_heads)), dim a multiple of 8 up to 128.  Sequence i has the queries
    [q_starts[i], q_starts[i + 1]) and the keys [k_starts[i], k_starts[i + 1])
    (default: as the queries); both are int32 or int64 tensors on the device
    (of values that fit 32 bits), ascending from 0, and are never read back.  With ``causal``, query j of a
    sequence sees its keys up to j + (keys - queries): the last query sees
    all.  out = softmax(scale * q k) v (scale: dim ** -0.5); a query that sees
    no key or is in no sequence gives zeros and passes no gradient.  Values of
    other sequences and of rows of none never matter, but a key or value that is
    not finite may reach the queries of its own sequence that do not see it
    (weights of zero times infinity, as where all keys are multiplied), and a
    query or gradient that is not the keys that it does not see.  With
    ``return_lse`` also the logarithm of each query's sum of exponentials,
    (q_total, q_heads) fp32 (-inf without keys, no gradient)."""
    for name, x in (('q', q), ('k', k), ('v', v)):
        _check_rows(name, x)
    _check_heads(q, k, v)
    scale = _check_scale(scale, q.shape[2])
    P.require_gpu(q, k, v)
    q_starts = _check_starts('q_starts', q_starts, q)
    if k_starts is None:
        if k.shape[0] != q.shape[0]:
            raise ValueError('without k_starts, q and k must have the same number of tokens.')
        k_starts = q_starts
    else:
        k_starts = _check_starts('k_starts', k_starts, q)
    if k_starts.shape != q_starts.shape:
        raise ValueError('q_starts and k_starts must have the same length.')
    run = _AttendPacked.apply if _wants_grad(q, k, v) or _recorded() else _attend_packed
    out, lse = run(_aligned(q, q.shape[1] // k.shape[1]), _aligned(k), _aligned(v), q_starts,
                   k_starts, bool(causal), scale)
    return (out, lse) if return_lse else out


# ---- new tokens over caches ------------------------------------------------

def _cache_fits(x, strides):
    per = 16 // x.element_size()
    return (strides[-1] == 1 and x.data_ptr() % 16 == 0 and not any(s % per for s in strides[:-1])
            and strides[-3] < per << 20)


def _cache(name, x, dims):
    """x, or a view of it in which dimensions of one, whose stride leads
    nowhere, have a stride that the kernels take."""
    _check_rows(name, x, dims)
    if x.numel() and not _cache_fits(x, x.stride()):
        used = [s if n > 1 else 0 for n, s in zip(x.shape[:-1], x.stride())] + [x.stride(-1)]
        if _cache_fits(x, used):
            return x.as_strided(x.shape, used)
        raise ValueError(f'{name}: rows and heads must start at multiples of 16 bytes, rows less '
                         'than 16 MiB apart.')
    return x


def _attend_cached(q, rows, k, v, lengths, prefix_k, prefix_v, scale):
    """rows: q (requests, tokens, q_heads, dim) as aligned rows."""
    requests, tokens, q_heads, dim = q.shape
    capacity, k_heads = k.shape[1:3]
    prefix = prefix_k.shape[0] if prefix_k is not None else 0
    out = q.new_empty(q.shape)
    nbytes = L.library().bevpool_attention_cached_scratch_bytes(
        requests, tokens, capacity, prefix, q_heads, k_heads, dim)
    scratch = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _run(lambda lib, s: lib.bevpool_attention_cached(
        *_strides(rows), L.ptr(k), *k.stride()[:3], L.ptr(v), *v.stride()[:3],
        *_strides(prefix_k), *_strides(prefix_v), L.ptr(lengths), L.DTYPE_CODES[q.dtype],
        requests, tokens, capacity, prefix, q_heads, k_heads, dim, scale, L.ptr(out),
        L.ptr(scratch), nbytes, s), q.device, 'bevpool_attention_cached')
    return out


class _AttendCached(torch.autograd.Function):
    """For tangents and traces alone: there is no gradient."""
    @staticmethod
    def forward(ctx, q, rows, k, v, lengths, prefix_k, prefix_v, scale):
        return _attend_cached(q, rows, k, v, lengths, prefix_k, prefix_v, scale)


def attend_cached(q, k, v, lengths, prefix_k=None, prefix_v=None, *, scale=None):
    """Attention of new tokens over caches, with a prefix that all requests
    share.

    q (requests, tokens, q_heads, dim), or (requests, q_heads, dim) for single
    tokens; k, v (requests, capacity, k_heads, dim): each request's own cache,
    its new tokens' keys and values already in it.  lengths (requests,), int32
    or int64 on the device (of values that fit 32 bits): the keys in use, the
    new tokens' among them (taken as within [0, capacity]).  prefix_k, prefix_v (prefix, k_heads, dim) or
    None.  New token i sees the whole prefix and the first lengths - (tokens -
    1 - i) keys of its request's cache; what lies past a length is never read.
    A row that sees nothing gives zeros; a new token's key or value that is not
    finite may reach the tokens before it.  Returns q's shape, contiguous.  Heads
    and scale are as in :func:`attend_packed`.  No gradient."""
    single = q.dim() == 3
    if single:
        q = q.unsqueeze(1)
    _check_rows('q', q, 4)
    k, v = _cache('k', k, 4), _cache('v', v, 4)
    _check_heads(q, k, v)
    requests, tokens, q_heads, dim = q.shape
    if k.shape[0] != requests:
        raise ValueError('q and k must have the same number of requests.')
    if tokens < 1:
        raise ValueError('q must hold at least one token of each request.')
    if (prefix_k is None) != (prefix_v is None):
        raise ValueError('prefix_k and prefix_v go together.')
    if prefix_k is not None:
        prefix_k, prefix_v = _cache('prefix_k', prefix_k, 3), _cache('prefix_v', prefix_v, 3)
        for name, x in (('prefix_k', prefix_k), ('prefix_v', prefix_v)):
            _check_same(name, x, q)
            if x.shape[1:] != k.shape[2:] or x.shape != prefix_k.shape:
                raise ValueError(f'{name} must have shape [prefix, k_heads, dim].')
    scale = _check_scale(scale, dim)
    if lengths.dim() != 1 or lengths.shape[0] != requests:
        raise ValueError('lengths must have shape [requests].')
    if lengths.dtype not in (torch.int32, torch.int64):
        raise TypeError('lengths must have dtype torch.int32 or torch.int64.')
    P.require_gpu(q, k, v, lengths)
    if lengths.device != q.device:
        raise ValueError(f'lengths must be on the device of q ({q.device}).')
    if _wants_grad(q, k, v, prefix_k, prefix_v):
        raise RuntimeError('attend_cached has no gradient; call it under torch.no_grad()')
    rows = _aligned(q.reshape(requests * tokens, q_heads, dim))
    if lengths.dtype != torch.int32 or not lengths.is_contiguous():
        lengths = lengths.to(torch.int32).contiguous()
    run = _AttendCached.apply if _recorded() else _attend_cached
    out = run(q, rows, k, v, lengths, prefix_k, prefix_v, scale)
    return out[:, 0] if single else out
