"""The operators of the block around the attention from their definitions, in 64
bits on the CPU, with the distance from them that a result computed as the
kernels state may have (test infrastructure).

Bounds: u is half the spacing of a result's type relative to its value, F the
same of fp32, in which everything else is held.  They are first-order worst
cases of every rounding on the way, evaluated with sums of magnitudes; nothing
is fitted.  A sum of n terms in fp32 is off by at most n F times the sum of
their magnitudes, in whatever order.
"""
from __future__ import annotations

import math

import torch

from .tokens import F, TINY, U

BLOCK = 32


def kept(x):
    """What the 8-bit checkpoint of x stands for, in 64 bits."""
    width = x.shape[-1]
    y = torch.nn.functional.pad(x.double(), (0, -width % BLOCK)).unflatten(-1, (-1, BLOCK))
    finite = y.isfinite()
    top = torch.where(finite, y, 0.0).abs().amax(-1, keepdim=True)
    p = torch.full_like(top, 2.0 ** -126)
    for _ in range(247):  # (doubled until it is enough, up to 2^121)
        p = torch.where(127 * p < top, 2 * p, p)
    y = (torch.where(finite, y, math.nan) / p).round().clamp(-127, 127) * p
    y = y.flatten(-2)[..., :width]
    if x.dtype == torch.float16:
        y = y.clamp(-65504, 65504)
    return y


def token_codes(x):
    """(codes, scale) of each row, in 64 bits: by trying every bf16 number next
    to the quotient."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    near = (top / 127).float().view(torch.int32) >> 16  # upper halves: bf16 numbers
    scale = torch.full_like(top, math.inf)
    for i in (2, 1, 0, -1):
        s = ((near + i).clamp_min(0x80) << 16).view(torch.float32).double()
        scale = torch.where(127 * s >= top, s, scale)
    scale = torch.where(top.isfinite(), scale, math.nan)
    return (x / scale).round(), scale


# ---- residual and norms ----------------------------------------------------

def _norm(x, weight, eps):
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight


def residual_norm(x, update, update_weight, scale, gate, weight, eps):
    """(sum, normed) in 64 bits, differentiable; gate a row for each of x's."""
    total = x
    if update is not None:
        n = update if update_weight is None else _norm(update, update_weight, eps)
        total = x + (1.0 if scale is None else scale) * (1.0 if gate is None else gate) * n
    return total, None if weight is None else _norm(total, weight, eps)


def residual_bounds(x, update, update_weight, scale, gate, weight, eps, x_dtype, dtype, dtotal=None,
                    dnormed=None, groups=None):
    """{name: bound} for the results of inputs in 64 bits; the gradients' bounds
    are absolute, before the last rounding (u |value| is added by the caller)."""
    W, rows = x.shape[-1], x.shape[0]
    one = torch.ones((), dtype=torch.float64)
    w_u, s, g, w = (one if t is None else t.abs() for t in (update_weight, scale, gate, weight))
    if update is None:
        n, r_u, v = torch.zeros_like(x), one, torch.zeros_like(x)
    else:
        r_u = one
        if update_weight is not None:
            r_u = 1 / torch.sqrt(update.square().mean(-1, keepdim=True) + eps)
        n = update * r_u
        v = n.abs() * w_u * s * g
    total, normed = residual_norm(x, update, update_weight, scale, gate, weight, eps)
    big = x.abs() + v                       # what the sum is made of
    e_sum = (W / 2 + 24) * F * v + F * total.abs()
    out = {'sum': e_sum}
    r = 1 / torch.sqrt(total.square().mean(-1, keepdim=True) + eps)
    # relative error of r: half of that of the mean of squares
    e_r = (W / 2 + 16) * F + (total.abs() * e_sum).mean(-1, keepdim=True) * r * r
    if weight is not None:
        out['normed'] = w * r * (e_sum + total.abs() * (e_r + 4 * F))
    if dtotal is None and dnormed is None:
        return out
    D = torch.zeros_like(x) if dtotal is None else dtotal.abs()
    e_g = 2 * F * D
    H = torch.zeros_like(x) if dnormed is None else dnormed.abs() * w
    if weight is not None and dnormed is not None:
        M = (H * big).mean(-1, keepdim=True)
        size = D + r * (H + big * r * r * M)
        # G = D + r (H - x' r^2 mean(H x')): r three times, the mean's W products, x' twice
        e_g = 3 * e_r * size + (W + 24) * F * size + r ** 3 * (
            e_sum * M + total.abs() * (H * e_sum).mean(-1, keepdim=True))
        out['dweight'] = (dnormed.abs() * r * (e_sum + total.abs() * (e_r + (rows + 8) * F))).sum(0)
        G = size
    else:
        G = D
    out['dx'] = e_g
    if update is None:
        return out
    c = w_u * s * g * torch.ones_like(x)
    e_n = ((W / 2 + 16) * F) * n.abs() if update_weight is not None else 0 * n
    t = c * e_g + 6 * F * c * G
    if update_weight is not None:
        m = (c * G * n.abs()).mean(-1, keepdim=True)
        out['dupdate'] = r_u * (t + n.abs() * (t * n.abs()).mean(-1, keepdim=True)
                                + (2 * W + 48) * F * (c * G + n.abs() * m))
    else:
        out['dupdate'] = t
    part = e_g * n.abs() + G * e_n + 8 * F * G * n.abs()  # of G n
    total_rows = (rows + 16) * F
    q = ((part + total_rows * G * n.abs()) * g * torch.ones_like(x)).sum(0)
    if update_weight is not None:
        out['dupdate_weight'] = q * s
    if scale is not None:
        out['dscale'] = q * w_u
    if gate is not None:
        each = (part + total_rows * G * n.abs()) * s * w_u
        out['dgate'] = each if groups is None else each.unflatten(0, (groups, -1)).sum(1)
    return out


# ---- gated activation ------------------------------------------------------

# (torch's own normal integral and the slope of its sigmoid cancel in the
# tails, which leaves them 1e-16 off whatever their size)
def normal(a):
    return 0.5 * torch.special.erfc(-a / math.sqrt(2))


def sigmoid(a):
    e = torch.exp(torch.where(a < 0, a, -a))  # (of a slope at zero, as abs has none)
    return torch.where(a < 0, e, torch.ones_like(e)) / (1 + e)


def act(a, kind):
    if kind == 'gelu':
        return a * normal(a)
    return a * sigmoid(a) if kind == 'silu' else sigmoid(a)


def gated(x, kind):
    a, b = x.chunk(2, -1)
    return act(a, kind) * b


def gated_bounds(x, kind, dout=None):
    """{name: bound} before the last rounding."""
    a, b = (t.abs() for t in x.chunk(2, -1))
    sa = x.chunk(2, -1)[0]
    floor = 2.0 ** -120  # (what underflows on the way)
    if kind == 'gelu':
        # arguments -a / sqrt(2) and -a^2 / 2 rounded: a^2 F of the functions; erfc to 16 units
        rel = (2 * a * a + 64) * F
        y = a * normal(sa)
        slope = normal(sa) + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    else:
        # exp(-|a|): its argument rounded, |a| F of it; functions to 2 units
        rel = (2 * a + 24) * F
        p, q = sigmoid(sa), sigmoid(-sa)
        y = a * p if kind == 'silu' else p
        slope = p + a * p * q if kind == 'silu' else 2 * p * q
    out = {'out': rel * y * b + floor * (1 + a) * b}
    if dout is not None:
        g = dout.abs()
        out['dx'] = torch.cat((2 * rel * slope * g * b + floor * (1 + a) * g * b,
                               rel * y * g + floor * (1 + a) * g), -1)
    return out


# ---- products in 8-bit integers --------------------------------------------

def linear_int8(x, codes, scales, bias):
    """(value, bound before the last rounding) in 64 bits."""
    q, s = token_codes(x)
    y = (q @ codes.double().T) * s * scales.double()
    bound = 4 * F * y.abs()
    if bias is not None:
        y = y + bias.double()
        bound = bound + F * y.abs()
    return y, bound


__all__ = ['BLOCK', 'F', 'TINY', 'U', 'act', 'gated', 'gated_bounds', 'kept', 'linear_int8',
           'residual_bounds', 'residual_norm', 'token_codes']
