"""Operators of the block around the attention on MI355X: what a transformer on
camera and BEV tokens does between its attention layers, as HIP kernels behind
the same C ABI (``include/bevpool.h``); the reference has no counterpart.

  * :func:`residual_norm`      norms after and before a block, fused with the
                               residual, its gate and its scale
  * :func:`gated_activation`   act(a) b of a projection's two halves
  * :func:`checkpoint_linear`  a linear layer that keeps its input in 8 bits
  * :func:`pack_activations`   such an 8-bit checkpoint by itself
  * :func:`linear_int8`        products in 8-bit integers, for serving, of
                               weights from :func:`quantize_weight`

The first three have gradients.  With ``checkpoint=8`` the backward pass works
from 8-bit copies of what the forward read, for wide rows a little over half of
the memory of 16-bit ones (33 bytes for 32 values, a row's rounded up to whole
blocks and then to 16 bytes: narrow rows gain less or nothing).  Blocks of 32 values along
a row share the least power of two p with 127 p >= their largest magnitude, and
each is rounded to a multiple of p (ties to even; in fp16 at most to its largest
number).  A value that is not finite comes back as NaN, and no other does.

Rows are the leading dimensions; their strides are free, a row's values are
copied where they are not neighbours.  Calls run on torch's current stream,
allocate with torch's allocator and never wait for the device.
"""
from __future__ import annotations

import math

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import _pipeline as P
from .attention import _recorded, _run, _unit, _wants_grad

ACTIVATIONS = {'silu': 0, 'gelu': 1, 'sigmoid': 2}
MAX_RESIDUAL_WIDTH = 8192
MAX_GATED_WIDTH = 1 << 18
MAX_INT8_WIDTH = 1 << 17


def _rows(x):
    """x as (rows, width) with unit stride along the width."""
    if x.dim() != 2:
        x = x.unsqueeze(0) if x.dim() == 1 else x.flatten(0, -2)
    return _unit(x)


def _row(x):
    """(address, row stride) for a call; of nothing: (0, 0)."""
    return (x.data_ptr(), x.stride(0)) if x is not None else (0, 0)


def _check_type(name, x):
    if x.dtype not in L.DTYPE_CODES:
        raise TypeError(f'{name} must have dtype torch.float16, torch.float32, or torch.bfloat16.')


def _check_beside(name, t, dtype, device):
    if t.dtype != dtype:
        raise TypeError(f'{name} must have dtype {dtype}.')
    if t.device != device:
        raise ValueError(f'{name} must be on the device of x ({device}).')


def _vector(name, t, size, dtype, device, shape='width'):
    """t (size,), contiguous; None is None."""
    if t is None:
        return None
    _check_beside(name, t, dtype, device)
    if t.shape != (size,):
        raise ValueError(f'{name} must have shape [{shape}].')
    return t if t.is_contiguous() else t.contiguous()


def _check_checkpoint(checkpoint):
    if checkpoint not in (None, 8):
        raise ValueError('checkpoint must be None or 8.')
    return checkpoint is not None


# ---- residual and norms ----------------------------------------------------

class _ResidualNorm(torch.autograd.Function):
    """For traces, and to refuse tangents; csrc/block_calls.cpp has the node that
    follows other calls."""
    @staticmethod
    def forward(ctx, x, update, update_weight, scale, gate, weight, dtype, eps, keep):
        total, normed, x_kept, update_kept = L.block_calls().residual_norm_forward(
            x, update, update_weight, scale, gate, weight, dtype, eps, keep)
        if not keep:
            x_kept, update_kept = x if weight is not None else None, update
        ctx.save_for_backward(x_kept, update_kept, update_weight, scale, gate, weight)
        ctx.call = (*x.shape, x.dtype, dtype, eps, keep, update is not None)
        ctx.set_materialize_grads(False)
        return total, normed

    @staticmethod
    @once_differentiable
    def backward(ctx, dtotal, dnormed):
        return (*L.block_calls().residual_norm_backward(dtotal, dnormed, *ctx.saved_tensors, *ctx.call),
                None, None, None)


def residual_norm(x, update=None, *, update_weight=None, scale=None, gate=None, weight=None,
                  eps=1e-6, checkpoint=None):
    """A block's output joins the residual stream, and the next block's input
    is normed, in one pass; returns (sum, normed).

        n      = update / sqrt(mean(update^2) + eps) * update_weight
                 (without update_weight: update)
        sum    = x + scale * gate * n
        normed = sum / sqrt(mean(sum^2) + eps) * weight
                 (None without weight; in fp32, of the sum before its rounding)

    x (..., width): the stream, fp32 or the type of the others; update
    (..., width): the block's output, or None: the norm alone, of x, which is
    then the sum.  update_weight, scale, weight (width,).  gate: of x's shape,
    or (groups, width), a row for each of `groups` equal parts of the rows in
    order, or (width,).  width at most 8192.

    With eps of 0 a row of zeros is NaN, as the formula has it.

    Gradients flow to all of them.  ``checkpoint=8`` keeps 8-bit copies of x
    and update for them instead of x and update; the gradients are those at
    the values that the copies stand for."""
    keep = _check_checkpoint(checkpoint)
    _check_type('x', x)
    P.require_gpu(x)
    if x.dim() < 1:
        raise ValueError('x must have shape [..., width].')
    shape, device = x.shape, x.device
    width = shape[-1]
    if not 1 <= width <= MAX_RESIDUAL_WIDTH:
        raise ValueError(f'width must be in [1, {MAX_RESIDUAL_WIDTH}].')
    if update is None:
        if not (update_weight is scale is gate is None):
            raise ValueError('update_weight, scale and gate are of an update.')
        if weight is None:
            raise ValueError('neither an update nor a weight: nothing to do.')
        _check_type('weight', weight)
        dtype = weight.dtype
    else:
        _check_type('update', update)
        dtype = update.dtype
        _check_beside('update', update, dtype, device)
        if update.shape != shape:
            raise ValueError('update must have the shape of x.')
    if x.dtype not in (dtype, torch.float32):
        raise TypeError(f'x must have dtype torch.float32 or that of the others ({dtype}).')
    if not eps >= 0:
        raise ValueError('eps must not be negative.')
    update_weight = _vector('update_weight', update_weight, width, dtype, device)
    scale = _vector('scale', scale, width, dtype, device)
    weight = _vector('weight', weight, width, dtype, device)
    if gate is not None:
        _check_beside('gate', gate, dtype, device)
        if gate.shape != shape and not (gate.dim() in (1, 2) and gate.shape[-1] == width):
            raise ValueError('gate must have the shape of x, [groups, width] or [width].')
        gate = _rows(gate)
        rows, groups = x.numel() // width, gate.shape[0]
        if groups < min(rows, 1) or groups and rows % groups:
            raise ValueError('the rows of gate must divide those of x.')
    args = (_rows(x), None if update is None else _rows(update), update_weight, scale, gate, weight,
            dtype, float(eps))
    if _recorded():
        total, normed = _ResidualNorm.apply(*args, keep)
    else:
        total, normed = L.block_calls().residual_norm(*args, keep, _wants_grad(*args[:6]))
    if len(shape) == 2:
        return x if total is None else total, normed
    return (x if total is None else total.view(shape),
            normed if normed is None else normed.view(shape))


# ---- gated activation ------------------------------------------------------

class _Gated(torch.autograd.Function):
    """As _ResidualNorm."""
    @staticmethod
    def forward(ctx, x, kind, keep):
        out, kept = L.block_calls().gated_activation_forward(x, kind, keep)
        ctx.save_for_backward(kept if keep else x)
        ctx.call = (*out.shape, x.dtype, kind, keep)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        return *L.block_calls().gated_activation_backward(dout, *ctx.saved_tensors, *ctx.call), None, None


def gated_activation(x, kind='silu', *, checkpoint=None):
    """act(a) * b of the two halves a, b of x's rows: x (..., 2 width) ->
    (..., width).  kind: 'silu' a / (1 + exp(-a)), 'gelu' (of the normal
    distribution's integral) or 'sigmoid'.  width at most 2^18.  The gradient
    flows to x; ``checkpoint=8`` keeps an 8-bit copy of x for it instead of x,
    each half in blocks of its own."""
    keep = _check_checkpoint(checkpoint)
    _check_type('x', x)
    if kind not in ACTIVATIONS:
        raise ValueError(f'kind must be one of {", ".join(ACTIVATIONS)}.')
    if x.dim() < 1 or x.shape[-1] % 2 or not 2 <= x.shape[-1] <= 2 * MAX_GATED_WIDTH:
        raise ValueError(f'x must have shape [..., 2 width], width in [1, {MAX_GATED_WIDTH}].')
    P.require_gpu(x)
    rows, kind = _rows(x), ACTIVATIONS[kind]
    if _recorded():
        out = _Gated.apply(rows, kind, keep)
    else:
        out = L.block_calls().gated_activation(rows, kind, keep, _wants_grad(x))
    return out if x.dim() == 2 else out.view(*x.shape[:-1], x.shape[-1] // 2)


# ---- 8-bit checkpoints -----------------------------------------------------

class PackedActivations:
    """An 8-bit checkpoint of a tensor: :meth:`unpack` gives the values that it
    stands for, in the tensor's type and shape.  ``data``: a row of bytes for each
    row, 33 for 32 values, rounded up to 16 (48 at least)."""

    def __init__(self, data, shape, dtype):
        self.data, self.shape, self.dtype = data, shape, dtype

    def unpack(self):
        data, shape = self.data, tuple(self.shape)
        P.require_gpu(data)
        if data.dtype != torch.uint8 or self.dtype not in L.DTYPE_CODES:
            raise TypeError('a checkpoint has bytes of dtype torch.uint8, of values of dtype '
                            'torch.float16, torch.float32, or torch.bfloat16.')
        width = shape[-1] if shape else 0
        pitch = L.library().bevpool_checkpoint_pitch(width)
        if not 1 <= width <= MAX_GATED_WIDTH or data.shape != (math.prod(shape[:-1]), pitch):
            raise ValueError(f'data must have shape [rows, {pitch}] for a checkpoint of {shape}.')
        if not data.is_contiguous() or data.data_ptr() % 16:
            data = data.clone(memory_format=torch.contiguous_format)
        out = data.new_empty(shape, dtype=self.dtype)
        _run(lambda lib, s: lib.bevpool_checkpoint_unpack(
            L.ptr(data), L.DTYPE_CODES[self.dtype], data.shape[0], width, L.ptr(out), s),
            data.device, 'bevpool_checkpoint_unpack')
        return out


def _pack(x):
    return L.block_calls().pack(_rows(x))


class _Pack(torch.autograd.Function):
    """For tangents and traces alone: there is no gradient."""
    @staticmethod
    def forward(ctx, x):
        return _pack(x)


def pack_activations(x):
    """x (..., width) as :class:`PackedActivations`, blocks of 32 values along
    the width (at most 2^18).  Values are rounded to 7 bits of their block's
    largest; what they stand for fp16 and bf16 hold exactly, so unpacking rounds
    no more (fp16: 65,536 is 65,504).  No gradient."""
    _check_type('x', x)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_GATED_WIDTH:
        raise ValueError(f'x must have shape [..., width], width in [1, {MAX_GATED_WIDTH}].')
    P.require_gpu(x)
    if _wants_grad(x):
        raise RuntimeError('pack_activations has no gradient; call it under torch.no_grad()')
    data = _Pack.apply(x) if _recorded() else _pack(x)
    return PackedActivations(data, x.shape, x.dtype)


def _from_checkpoint(dtype, n, k):
    """Whether the gradient of a weight (n, k) is formed from the checkpoint
    itself: where it is so small that the tokens have to be divided over the
    card's CUs, up to half a tile of 256 x 256 for each.  Above, what the
    checkpoint stands for and a library product are faster.  us of the one and
    of the other: 16,896 tokens of 1280 x 1280 84 and 220, of 1280 x 5120 278 and
    322, of 10240 x 1280 584 and 522; 4,096 of 4096 x 4096 166 and 137.  For fewer
    tokens the one is slower too, and keeps no 16-bit copy: 300, 2,048 and 4,096 of
    1280 x 1280 27 and 19, 37 and 31, 45 and 47; 512 and 4,096 of 2048 x 4096 41 and
    27, 96 and 84; 300 and 4,096 of 256 x 256 24 and 28, 25 and 37."""
    return (dtype != torch.float32 and 0 < n <= 1 << 20 and n % 8 == 0
            and -(-n // 256) * -(-k // 256) <= 128)


class _CheckpointLinear(torch.autograd.Function):
    """As _ResidualNorm."""
    @staticmethod
    def forward(ctx, x, weight, bias, direct):
        # (the weight's gradient alone needs x)
        ctx.save_for_backward(_pack(x) if ctx.needs_input_grad[1] else None, weight)
        ctx.call = (*x.shape, x.dtype, direct)
        return nn.functional.linear(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return *L.block_calls().checkpoint_linear_backward(dy, *ctx.saved_tensors, *ctx.call,
                                                         *ctx.needs_input_grad[:3]), None


def _checkpoint_linear(x, weight, bias):
    direct = _from_checkpoint(x.dtype, *weight.shape)
    if _recorded():
        return _CheckpointLinear.apply(x, weight, bias, direct)
    return L.block_calls().checkpoint_linear(x, weight, bias, direct)


def checkpoint_linear(x, weight, bias=None):
    """x weight^T + bias as torch.nn.functional.linear, x (..., in), weight
    (out, in), bias (out,), of one type; but what is kept of x for the
    weight's gradient is an 8-bit copy, and the gradient is that at the values
    it stands for.  The others are exact.  Follows autocast."""
    _check_type('x', x)
    P.require_gpu(x)
    autocast = torch.is_autocast_enabled('cuda')
    if autocast:
        kind = torch.get_autocast_dtype('cuda')
        x, weight = x.to(kind), weight.to(kind)
        bias = bias if bias is None else bias.to(kind)
    _check_beside('weight', weight, x.dtype, x.device)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError('x must have shape [..., in] and weight [out, in].')
    if not 1 <= x.shape[-1] <= MAX_GATED_WIDTH:
        raise ValueError(f'in must be in [1, {MAX_GATED_WIDTH}].')
    bias = _vector('bias', bias, weight.shape[0], x.dtype, x.device, 'out')
    if not _wants_grad(x, weight, bias) and not _recorded():
        return nn.functional.linear(x, weight, bias)
    if autocast:  # (the operands have their types)
        with torch.autocast('cuda', enabled=False):
            y = _checkpoint_linear(_rows(x), weight, bias)
    else:
        y = _checkpoint_linear(_rows(x), weight, bias)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])


class CheckpointLinear(nn.Linear):
    """A linear layer through :func:`checkpoint_linear`."""

    def forward(self, x):
        return checkpoint_linear(x, self.weight, self.bias)


# ---- products in 8-bit integers --------------------------------------------

def quantize_weight(weight):
    """(codes, scales) of weight (out, in) for :func:`linear_int8`: each
    channel's scale is the least number of 8 bits (as bf16 has) with 127 scale
    >= its largest magnitude, its codes the multiples of the scale next to its
    values (ties to even).  codes (out, in) int8, rows at multiples of 128 bytes; scales
    (out,) fp32.  A channel with a value that is not finite has a scale of NaN."""
    _check_type('weight', weight)
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_INT8_WIDTH:
        raise ValueError(f'weight must have shape [out, in], in in [1, {MAX_INT8_WIDTH}].')
    P.require_gpu(weight)
    weight = _unit(weight.detach())
    out, width = weight.shape
    codes = weight.new_empty((out, L.library().bevpool_linear8_pitch(width)), dtype=torch.int8)
    scales = weight.new_empty(out, dtype=torch.float32)
    _run(lambda lib, s: lib.bevpool_linear8_codes(
        *_row(weight), L.DTYPE_CODES[weight.dtype], out, width, L.ptr(codes), L.ptr(scales), s),
        weight.device, 'bevpool_linear8_codes')
    return codes[:, :width], scales


def _code_rows(codes):
    """(codes, row stride): rows at multiples of 16 bytes that can be read up
    to one; codes itself, or a copy."""
    out, width = codes.shape
    row, one = codes.stride()
    need = (width + 15) // 16 * 16
    if out == 1:
        row = need
    end = codes.storage_offset() + (out - 1) * row + need
    if ((one == 1 or width == 1) and need <= row < 1 << 22 and row % 16 == 0
            and codes.data_ptr() % 16 == 0 and end <= codes.untyped_storage().nbytes()):
        return codes, row
    copy = codes.new_zeros((out, need))
    copy[:, :width] = codes
    return copy, need


class _LinearInt8(torch.autograd.Function):
    """For tangents and traces alone: there is no gradient."""
    @staticmethod
    def forward(ctx, x, codes, row, scales, bias):
        return L.block_calls().linear_int8(x, codes, row, scales, bias)


def linear_int8(x, codes, scales, bias=None):
    """x (codes * scales)^T + bias with products in 8-bit integers: x (..., in)
    fp32, fp16 or bf16, codes (out, in) int8 and scales (out,) fp32 as
    :func:`quantize_weight` gives them, bias (out,) of x's type or None ->
    (..., out).  in is at most 2^17.

    Each token gets a scale (the least number of 8 bits, as bf16 has, with 127 scale >= its
    largest magnitude) and codes, the nearest multiples of it (ties to even);
    the sums of products of codes are exact, and are multiplied by both scales
    in fp32.  A token with a value that is not finite gives NaN.  Rows of codes
    that do not start at multiples of 16 bytes are copied at each call.  No
    gradient."""
    _check_type('x', x)
    P.require_gpu(x)
    if codes.dim() != 2 or codes.dtype != torch.int8:
        raise TypeError('codes must have dtype torch.int8 and shape [out, in].')
    channels, width = codes.shape
    if not 1 <= width <= MAX_INT8_WIDTH:
        raise ValueError(f'in must be in [1, {MAX_INT8_WIDTH}].')
    if x.dim() < 1 or x.shape[-1] != width:
        raise ValueError('x must have shape [..., in], in as codes have it.')
    device = x.device
    if codes.device != device:
        raise ValueError(f'codes must be on the device of x ({device}).')
    scales = _vector('scales', scales, channels, torch.float32, device, 'out')
    bias = _vector('bias', bias, channels, x.dtype, device, 'out')
    if _wants_grad(x, scales, bias):
        raise RuntimeError('linear_int8 has no gradient; call it under torch.no_grad()')
    codes, row = _code_rows(codes) if channels else (codes, 0)
    run = _LinearInt8.apply if _recorded() else L.block_calls().linear_int8
    y = run(_rows(x), codes, int(row), scales, bias)  # (a trace has sizes as tensors)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], channels)


class Int8Linear(nn.Module):
    """A linear layer for serving through :func:`linear_int8`, made of one in
    another type: ``Int8Linear(nn.Linear(...))``.  Its scales stay fp32
    whatever the module is cast to."""

    def __init__(self, linear):
        super().__init__()
        self.in_features, self.out_features = linear.in_features, linear.out_features
        codes, scales = quantize_weight(linear.weight)
        # (whole rows, which stay where they begin when the module is moved)
        self.register_buffer('codes', codes.as_strided((codes.shape[0], codes.stride(0)),
                                                       codes.stride()))
        self.register_buffer('scales', scales)
        self.register_buffer('bias', None if linear.bias is None else linear.bias.detach().clone())

    def _apply(self, fn, *args, **kwargs):
        scales = self.scales
        super()._apply(fn, *args, **kwargs)
        if self.scales.dtype != torch.float32:
            self.scales = scales.to(self.scales.device)
        return self

    def forward(self, x):
        if torch.is_autocast_enabled('cuda'):
            x = x.to(torch.get_autocast_dtype('cuda'))
        bias = self.bias if self.bias is None else self.bias.to(x.dtype)
        return linear_int8(x, self.codes[:, :self.in_features], self.scales, bias)
