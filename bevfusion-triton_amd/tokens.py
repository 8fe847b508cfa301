"""Attention over camera and BEV tokens: the layer that runs the token operators
together.

:class:`TokenAttention` projects tokens to queries, keys and values, norms and
rotates queries and keys by the tokens' positions (:func:`norm_rotate`), and
attends within packed sequences (:func:`attend_packed`: training and whole
prompts) or from new tokens over caches and a shared scene
(:func:`attend_cached`: one token at a time).  ``examples/bev_tokens.py`` takes
it from the pooled BEV map to answers about one scene.

:class:`TokenBlock` is that layer within a transformer's block: norms, gates and
residuals (:func:`residual_norm`) and the gated layer (:func:`gated_activation`),
with 8-bit checkpoints for training and 8-bit products for serving.
"""
from __future__ import annotations

import torch
from torch import nn

from .attention import attend_cached, attend_packed, axis_frequencies, norm_rotate
from .block import CheckpointLinear, Int8Linear, gated_activation, residual_norm


class TokenAttention(nn.Module):
    """Attention of ``q_heads`` heads of ``head_dim`` over ``k_heads`` shared
    key heads, on tokens of ``dim`` channels.  ``pairs`` rotated pairs for each
    axis of the positions (frame, row, column; or one).  ``linear``: the class of
    its projections."""

    def __init__(self, dim, q_heads, k_heads, head_dim, pairs, *, base=10000.0, eps=1e-6,
                 device=None, dtype=None, linear=nn.Linear):
        super().__init__()
        kind = {'device': device, 'dtype': dtype}
        self.q_heads, self.k_heads, self.head_dim = q_heads, k_heads, head_dim
        self.pairs, self.eps = tuple(pairs), eps
        self.qkv = linear(dim, (q_heads + 2 * k_heads) * head_dim, bias=False, **kind)
        self.out = linear(q_heads * head_dim, dim, bias=False, **kind)
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


class TokenBlock(nn.Module):
    """A transformer's block on a residual stream of ``dim`` channels:
    :class:`TokenAttention`, then a gated layer of ``hidden`` values
    (``activation`` as in :func:`gated_activation`), each with a norm before, a
    norm after, a residual scale for each channel and an optional gate:

        x = x + gate * scale * norm(layer(norm(x)))

    The norm after one layer, its residual and the norm before the next are one
    pass.  The stream may be fp32 beside 16-bit parameters, or of their type.
    ``checkpoint=8`` keeps 8-bit copies for the backward pass in place of the
    inputs of the linear layers, of the gated activation and of the norms.
    :meth:`quantize` is for serving."""

    def __init__(self, dim, q_heads, k_heads, head_dim, pairs, hidden, *, activation='silu',
                 checkpoint=None, base=10000.0, eps=1e-6, device=None, dtype=None):
        super().__init__()
        if checkpoint not in (None, 8):
            raise ValueError('checkpoint must be None or 8.')
        kind = {'device': device, 'dtype': dtype}
        linear = nn.Linear if checkpoint is None else CheckpointLinear
        self.attention = TokenAttention(dim, q_heads, k_heads, head_dim, pairs, base=base, eps=eps,
                                        linear=linear, **kind)
        self.up = linear(dim, 2 * hidden, bias=False, **kind)
        self.down = linear(hidden, dim, bias=False, **kind)
        self.activation, self.checkpoint, self.eps = activation, checkpoint, eps
        for layer in ('attention', 'gated'):
            for name in ('norm', 'out_norm', 'scale'):
                setattr(self, f'{layer}_{name}', nn.Parameter(torch.ones(dim, **kind)))

    def _norm(self, x):
        """The attention's input: in the parameters' type, or autocast's, or that
        of a 16-bit stream."""
        kind = self.attention_norm.dtype if x.dtype == torch.float32 else x.dtype
        if torch.is_autocast_enabled('cuda'):
            kind = torch.get_autocast_dtype('cuda')
        x = x if x.dtype == torch.float32 else x.to(kind)
        return residual_norm(x, weight=self.attention_norm.to(kind), eps=self.eps,
                             checkpoint=self.checkpoint)[1]

    def _join(self, x, update, out_norm, scale, gate, norm):
        """The stream with a layer's output, and the next one's input."""
        update_weight, scale, gate, norm = (t if t is None else t.to(update.dtype)
                                            for t in (out_norm, scale, gate, norm))
        if x.dtype != torch.float32:
            x = x.to(update.dtype)
        return residual_norm(x, update, update_weight=update_weight, scale=scale, gate=gate,
                             weight=norm, eps=self.eps, checkpoint=self.checkpoint)

    def _gated(self, x, h, gate):
        y = self.down(gated_activation(self.up(h), self.activation, checkpoint=self.checkpoint))
        return self._join(x, y, self.gated_out_norm, self.gated_scale, gate, None)[0]

    def forward(self, x, positions, starts, *, causal=False, gates=(None, None)):
        """The stream x (tokens, dim) of packed sequences (positions and starts
        as in :class:`TokenAttention`) behind the block.  gates: of the
        attention's and of the gated layer's output, each None, (tokens, dim) or
        (groups, dim), a row for each of `groups` equal parts of the tokens."""
        y = self.attention(self._norm(x), positions, starts, causal=causal)
        x, h = self._join(x, y, self.attention_out_norm, self.attention_scale, gates[0],
                          self.gated_norm)
        return self._gated(x, h, gates[1])

    @torch.no_grad()
    def scene(self, x, positions):
        """(keys, values) of stream tokens that many requests share: the prefix
        of :meth:`step`."""
        return self.attention.scene(self._norm(x), positions)

    @torch.no_grad()
    def step(self, x, positions, cache_k, cache_v, lengths, prefix=(None, None), *,
             gates=(None, None)):
        """New tokens x (requests, new, dim) behind the block; caches, lengths
        and prefix as in :meth:`TokenAttention.step`.  gates: None, of x's shape,
        or (groups, dim), a row for each of `groups` equal parts of the tokens."""
        y = self.attention.step(self._norm(x), positions, cache_k, cache_v, lengths, prefix)
        x, h = self._join(x, y, self.attention_out_norm, self.attention_scale, gates[0],
                          self.gated_norm)
        return self._gated(x, h, gates[1])

    @torch.no_grad()
    def quantize(self):
        """Puts 8-bit integer products (:class:`Int8Linear`) in the place of the
        block's linear layers, for serving: there is no gradient any more.
        Returns the block."""
        for module, name in ((self.attention, 'qkv'), (self.attention, 'out'), (self, 'up'),
                             (self, 'down')):
            if not isinstance(getattr(module, name), Int8Linear):
                setattr(module, name, Int8Linear(getattr(module, name)))
        return self
