"""The token operators from their definitions, in 64 bits on the CPU, with the
distance from them that a result computed as the kernels state may have (test
infrastructure).

Bounds: u is half the spacing of the operands' type relative to a value (a
result's last rounding, and the rounding of weights and of score gradients to
the type before a matrix product), F the same of fp32, in which everything
else is held.  They are first-order worst cases of every rounding on the way,
evaluated with the sums of absolute values at hand; nothing is fitted.
"""
from __future__ import annotations

import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F = 2.0 ** -24
# smallest step of the type: results and weights below its normal range
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


# ---- norm and rotation -----------------------------------------------------

def pair_of(dim, pairs, interleaved):
    """(pair, sign partner) of every element: element d belongs to pair
    index[d] (-1: none) with the other element partner[d]; first[d] is True
    for the pair's first element."""
    n = sum(pairs)
    index, partner, first = [-1] * dim, list(range(dim)), [True] * dim
    for p in range(n):
        a, b = (2 * p, 2 * p + 1) if interleaved else (p, n + p)
        index[a] = index[b] = p
        partner[a], partner[b] = b, a
        first[b] = False
    return index, partner, first


def angles(positions, frequencies, pairs):
    """(tokens, P) angles in 64 bits."""
    pos = positions.double().reshape(positions.shape[0], -1)
    axis = [i for i, n in enumerate(pairs) for _ in range(n)]
    if not axis:
        return pos.new_zeros((pos.shape[0], 0))
    return pos[:, axis] * frequencies.double()


def norm_rotate(x, positions, frequencies, pairs, weight=None, eps=1e-6, interleaved=False):
    """(tokens, heads, dim) in 64 bits, differentiable; and the bound's scale,
    the sum of the magnitudes that each element is made of."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    index, partner, first = pair_of(x.shape[-1], pairs, interleaved)
    angle = angles(positions, frequencies, pairs)
    angle = torch.cat((angle, angle.new_zeros((angle.shape[0], 1))), 1)[:, None, index]
    sign = torch.tensor([-1.0 if f else 1.0 for f in first], dtype=torch.float64)
    turned = torch.tensor([i >= 0 for i in index])
    other = torch.where(turned, sign * y[..., partner] * angle.sin(), torch.zeros(()).double())
    return y * angle.cos() + other, (y.abs() + y[..., partner].abs()).detach()


# ---- attention -------------------------------------------------------------

def attend_rows(q, k, v, limits, scale):
    """One head: q (n, D), k, v (m, D) in 64 bits; row i sees keys
    [0, limits[i]).  Masked keys take no part, whatever they hold."""
    n, m = q.shape[0], k.shape[0]
    seen = torch.arange(m)[None] < torch.as_tensor(limits)[:, None]
    used = seen.any(0) if n else torch.zeros(m, dtype=torch.bool)
    k = torch.where(used[:, None], k, torch.zeros(()).double())
    s = torch.where(seen, scale * q @ k.T, torch.full((), -math.inf).double())
    top = s.amax(-1, keepdim=True) if m else s.new_full((n, 1), -math.inf)
    top = torch.where(top == -math.inf, torch.zeros(()).double(), top).detach()
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones(()).double(), total)
    lse = (torch.log(total) + top)[:, 0]
    return p, lse, used


def attend_packed(q, k, v, q_starts, k_starts, causal, scale, dout=None, dtype=torch.float64):
    """{name: (value, bound)} of out, lse and, with dout, dq, dk, dv for
    results in `dtype` (64 bits: the values alone matter)."""
    u, tiny = U.get(dtype, 0.0), TINY.get(dtype, 0.0)
    q, k, v = q.double(), k.double(), v.double()
    D, heads, group = q.shape[2], q.shape[1], q.shape[1] // k.shape[1]
    res = {n: (torch.zeros_like(t), torch.zeros_like(t))
           for n, t in (('out', q), ('dq', q), ('dk', k), ('dv', v))}
    res['lse'] = (torch.full(q.shape[:2], -math.inf).double(), torch.zeros(q.shape[:2]).double())
    q_at, k_at = q_starts.tolist(), k_starts.tolist()
    for s in range(len(q_at) - 1):
        a, b, c, d = q_at[s], q_at[s + 1], k_at[s], k_at[s + 1]
        nq, nk = b - a, d - c
        if nq <= 0:
            continue
        limits = [min(nk, max(0, i + 1 + nk - nq)) if causal else nk for i in range(nq)]
        for h in range(heads):
            g = h // group
            Q, K, V = q[a:b, h], k[c:d, g], v[c:d, g]
            p, lse, used = attend_rows(Q, K, V, limits, scale)
            V = torch.where(used[:, None], V, torch.zeros(()).double())
            K = torch.where(used[:, None], K, torch.zeros(()).double())
            out = p @ V
            # scores: D products and sums in fp32, the scale and the maximum's subtraction, all
            # relative to the sum of magnitudes; exp2 to 2 units; sums over nk keys
            err_s = (scale * Q.abs() @ K.abs().T) * (D + 6) * F + 4 * F
            err_p = p * (err_s + (p * err_s).sum(-1, keepdim=True) + (nk / 8 + 4) * F)
            tol = err_p @ V.abs() + (u + (nk / 8 + 4) * F) * (p @ V.abs()) + tiny * V.abs().sum(0)
            res['out'][0][a:b, h] = out
            res['out'][1][a:b, h] = tol + u * out.abs() + tiny
            res['lse'][0][a:b, h] = lse
            fin = torch.where(lse == -math.inf, torch.zeros(()).double(), lse.abs())
            res['lse'][1][a:b, h] = (p * err_s).sum(-1) + (nk / 8 + 8) * F + 4 * F * fin
            if dout is None:
                continue
            G = dout[a:b, h].double()
            dP = G @ V.T
            delta = (p * dP).sum(-1, keepdim=True)
            dS = p * (dP - delta)
            # delta comes from the rounded output
            err_delta = (G.abs() * (res['out'][1][a:b, h] + (D + 2) * F * out.abs())).sum(
                -1, keepdim=True)
            err_dp = G.abs() @ V.abs().T * (D + 2) * F
            e_lse = res['lse'][1][a:b, h][:, None]
            err_ds = (p * (err_s + e_lse + 4 * F)) * (dP - delta).abs() + p * (err_dp + err_delta)
            err_ds = err_ds + (u + 4 * F) * dS.abs() + tiny * (p > 0)
            n = max(nq * group, nk) / 8 + 4
            value, bound = res['dq']
            value[a:b, h] = scale * dS @ K
            bound[a:b, h] = scale * ((err_ds + n * F * dS.abs()) @ K.abs())
            value, bound = res['dk']
            value[c:d, g] += scale * dS.T @ Q
            bound[c:d, g] += scale * ((err_ds + n * F * dS.abs()).T @ Q.abs())
            value, bound = res['dv']
            value[c:d, g] += p.T @ G
            e = p * (err_s + e_lse + 4 * F) + (u + n * F) * p + tiny * (p > 0)
            bound[c:d, g] += e.T @ G.abs()
    for n in ('dq', 'dk', 'dv'):
        value, bound = res[n]
        bound += u * value.abs() + tiny
    return res


def attend_cached(q, k, v, lengths, prefix_k, prefix_v, scale, dtype):
    """(value, bound) of out (requests, tokens, heads, dim): every row as a
    packed sequence of one query over its prefix and its own keys."""
    B, n, heads, dim = q.shape
    value, bound = torch.zeros(q.shape).double(), torch.zeros(q.shape).double()
    for b in range(B):
        for i in range(n):
            own = min(max(int(lengths[b]), 0), k.shape[1]) - (n - 1 - i)
            own = max(own, 0)
            kk, vv = k[b, :own], v[b, :own]
            if prefix_k is not None:
                kk, vv = torch.cat((prefix_k, kk)), torch.cat((prefix_v, vv))
            res = attend_packed(q[b, i][None], kk, vv, torch.tensor([0, 1]),
                                torch.tensor([0, kk.shape[0]]), False, scale, dtype=dtype)
            value[b, i], bound[b, i] = (t[0] for t in res['out'])
    # the parts' weights: two exponentials and products more
    return value, bound + 16 * F * bound / U[dtype]
