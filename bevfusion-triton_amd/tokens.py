"""Attention over camera and BEV tokens: the layer that runs the token operators
together.

:class:`TokenAttention` projects tokens to queries, keys and values, norms and
rotates queries and keys by the tokens' positions (:func:`norm_rotate`), and
attends within packed sequences (:func:`attend_packed`: training and whole
prompts) or from new tokens over caches and a shared scene
(:func:`attend_cached`: one token at a time).  ``examples/bev_tokens.py`` takes
it from the pooled BEV map to answers about one scene.
"""
from __future__ import annotations

import torch
from torch import nn

from .attention import attend_cached, attend_packed, axis_frequencies, norm_rotate


class TokenAttention(nn.Module):
    """Attention of ``q_heads`` heads of ``head_dim`` over ``k_heads`` shared
    key heads, on tokens of ``dim`` channels.  ``pairs`` rotated pairs for each
    axis of the positions (frame, row, column; or one)."""

    def __init__(self, dim, q_heads, k_heads, head_dim, pairs, *, base=10000.0, eps=1e-6,
                 device=None, dtype=None):
        super().__init__()
        kind = {'device': device, 'dtype': dtype}
        self.q_heads, self.k_heads, self.head_dim = q_heads, k_heads, head_dim
        self.pairs, self.eps = tuple(pairs), eps
        self.qkv = nn.Linear(dim, (q_heads + 2 * k_heads) * head_dim, bias=False, **kind)
        self.out = nn.Linear(q_heads * head_dim, dim, bias=False, **kind)
        self.q_norm = nn.Parameter(torch.ones(head_dim, **kind))
        self.k_norm = nn.Parameter(torch.ones(head_dim, **kind))
        self.base = base
        # (a plain attribute: fp32 whatever the module is cast to)
        self.frequencies = axis_frequencies(self.pairs, base, device=device)

    def _apply(self, fn, *args, **kwargs):
        super()._apply(fn, *args, **kwargs)
        device = self.q_norm.device
        if self.frequencies.is_meta:  # (no values there to move)
            self.frequencies = axis_frequencies(self.pairs, self.base, device=device)
        else:
            self.frequencies = self.frequencies.to(device)
        return self

    def project(self, x, positions):
        """Normed and rotated queries and keys, and values, of x (tokens, dim)
        at positions (tokens, axes): (tokens, heads, head_dim) each."""
        rows = self.qkv(x).unflatten(-1, (-1, self.head_dim))
        q, k, v = rows.split((self.q_heads, self.k_heads, self.k_heads), -2)
        # (under autocast the projection is 16-bit and the weights are not)
        q, k = norm_rotate(q, k, positions, self.frequencies, self.pairs,
                           q_weight=self.q_norm.to(q.dtype), k_weight=self.k_norm.to(k.dtype),
                           eps=self.eps)
        return q, k, v

    def forward(self, x, positions, starts, *, causal=False):
        """x (tokens, dim), positions (tokens, axes) and starts (sequences + 1)
        of packed sequences -> (tokens, dim)."""
        q, k, v = self.project(x, positions)
        return self.out(attend_packed(q, k, v, starts, causal=causal).flatten(1))

    @torch.no_grad()
    def scene(self, x, positions):
        """(keys, values) of tokens that many requests share: the prefix of
        :meth:`step`."""
        _, k, v = self.project(x, positions)
        return k, v.contiguous()

    @torch.no_grad()
    def step(self, x, positions, cache_k, cache_v, lengths, prefix=(None, None)):
        """New tokens x (requests, new, dim) at positions (requests, new, axes):
        their keys and values go into the caches (requests, capacity, k_heads,
        head_dim) behind the ``lengths`` (requests,) that are there, which grow
        by ``new``; then the tokens attend to ``prefix``, to what their
        request's cache held and to themselves.  The host does not know the
        lengths: where a cache has no room left, the new tokens take its last
        slots, and its length stays at the capacity.  Returns (requests, new,
        dim)."""
        requests, new = x.shape[:2]
        capacity = cache_k.shape[1]
        if new > capacity:
            raise ValueError(f'{new} new tokens do not fit caches of {capacity}.')
        q, k, v = self.project(x.flatten(0, 1), positions.flatten(0, 1))
        held = lengths.clamp(0, capacity - new)
        slots = held[:, None] + torch.arange(new, device=x.device)
        rows = torch.arange(requests, device=x.device)[:, None]
        cache_k[rows, slots] = k.unflatten(0, (requests, new))
        cache_v[rows, slots] = v.unflatten(0, (requests, new))
        torch.add(held, new, out=lengths)
        out = attend_cached(q.unflatten(0, (requests, new)), cache_k, cache_v, lengths, *prefix)
        return self.out(out.flatten(2))
