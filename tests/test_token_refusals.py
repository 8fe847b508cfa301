"""Argument checks of the token operators' C entries: they return the
documented status and message before any HIP call, so no GPU is needed."""
from __future__ import annotations

import ctypes


def test_norm_rotate(pkg):
    """Argument checks return before any HIP call."""
    lib = pkg.library()
    i32 = lambda *v: (ctypes.c_int32 * max(1, len(v)))(*v)

    def forward(dtype=0, tokens=4, dim=64, kind=0, pairs=(32,), eps=1e-6, k_heads=0, kw=None):
        return lib.bevpool_norm_rotate_forward(1, 64, 64, 1, None, 0, 0, k_heads, dtype, tokens,
                                               dim, 1, kind, 1, 1, i32(*pairs), len(pairs), 0,
                                               None, kw, eps, 1, None, None)

    for bad, text in ((dict(dtype=5), b'dtype'), (dict(tokens=-1), b'negative'),
                      (dict(dim=63), b'even'), (dict(dim=258), b'256'),
                      (dict(pairs=(33,)), b'fit'), (dict(pairs=(20, 20)), b'fit'),
                      (dict(kind=3), b'position type'), (dict(eps=float('nan')), b'eps'),
                      (dict(k_heads=2), b'null'), (dict(kw=1), b'no heads')):
        assert forward(**bad) == -1, bad
        assert text in lib.bevpool_last_error(), bad
    assert lib.bevpool_norm_rotate_backward(
        None, 0, 0, 1, None, 0, 0, 0, 1, 64, 64, None, 0, 0, 0, 4, 64, 1, 0, 1, 1, i32(32), 1, 0,
        1, None, 1e-6, 1, None, 1, None, None, 0, None) == -1  # a weight, but no rows
    assert lib.bevpool_norm_rotate_backward(
        1, 64, 64, 1, None, 0, 0, 0, 1, 64, 64, None, 0, 0, 0, 4, 64, 1, 0, 1, 1, i32(32), 1, 0,
        1, None, 1e-6, 1, None, 1, None, 1, 16, None) == -3


def test_attention(pkg):
    """Argument checks return before any HIP call."""
    lib = pkg.library()

    def forward(dtype=2, q_total=4, k_total=4, q_heads=4, k_heads=2, dim=64, scale=0.125, q=16,
                row=256, starts=16, rest=None):
        return lib.bevpool_attention_forward(q, row, dim, 16, 128, dim, 16, 128, dim, dtype,
                                             q_total, k_total, q_heads, k_heads, dim, starts,
                                             starts, 1, 0, scale, 16, rest, None, None)

    for bad, text in ((dict(dtype=3), b'dtype'), (dict(q_total=-1), b'negative'),
                      (dict(q_heads=3), b'no multiple'), (dict(k_heads=0), b'no multiple'),
                      (dict(dim=60), b'multiple of 8'), (dict(dim=256), b'multiple of 8'),
                      (dict(scale=-1.0), b'scale'), (dict(scale=float('nan')), b'scale'),
                      (dict(q_total=1 << 30), b'too many'), (dict(k_total=1 << 30), b'too many'),
                      (dict(q=None), b'q: null'), (dict(q=8), b'16 bytes'),
                      (dict(row=255), b'16 bytes'), (dict(rest=8), b'out_rest'), (dict(starts=None), b'null starts')):
        assert forward(**bad) == -1, bad
        assert text in lib.bevpool_last_error(), bad
    args = (16, 256, 64, 16, 128, 64, 16, 128, 64, 16, 16, 16, 256, 64, 16, 2, 4, 4, 4, 2, 64, 16, 16,
            1, 0, 0.125, 16, 16, 16)
    assert lib.bevpool_attention_backward_scratch_bytes(4, 4, 4, 2, 64, 2, 1) == 256
    assert lib.bevpool_attention_backward(*args, None, 0, None) == -3
    assert b'scratch' in lib.bevpool_last_error()


def test_cached_attention(pkg):
    lib = pkg.library()

    def call(dtype=2, requests=2, tokens=1, capacity=64, prefix=0, q_heads=4, k_heads=2, dim=64,
             scale=0.125, q=16, k=16, request=64 * 128, pk=None, lengths=16, scratch=None, nbytes=0):
        return lib.bevpool_attention_cached(
            q, 256, 64, k, request, 128, 64, 16, request, 128, 64, pk, 128, 64, pk, 128, 64,
            lengths, dtype, requests, tokens, capacity, prefix, q_heads, k_heads, dim, scale, 16,
            scratch, nbytes, None)

    for bad, text in ((dict(dtype=3), b'dtype'), (dict(tokens=0), b'bad sizes'),
                      (dict(capacity=-1), b'bad sizes'), (dict(q_heads=3), b'bad sizes'),
                      (dict(requests=1 << 30), b'bad sizes'), (dict(dim=20), b'multiple of 8'),
                      (dict(scale=0.0), b'scale'), (dict(lengths=None), b'lengths'),
                      (dict(q=None), b'q: null'), (dict(k=8), b'16 bytes'),
                      (dict(request=64 * 128 + 4), b'16 bytes'), (dict(prefix=9), b'prefix_k')):
        assert call(**bad) == -1, bad
        assert text in lib.bevpool_last_error(), bad
    need = lib.bevpool_attention_cached_scratch_bytes(2, 1, 5000, 0, 4, 2, 64)
    assert need > 0 and need % ((64 + 2) * 4 * 2 * 4) == 0
    assert call(capacity=5000, scratch=16, nbytes=need - 1) == -3
    assert lib.bevpool_attention_cached_scratch_bytes(2, 1, 64, 0, 4, 2, 64) == 0


def test_heads_of_a_group_within_reach(pkg):
    """Any head of a group may begin a tile of rows, also where there are more
    than a tile has rows: the strides of all of them count."""
    lib = pkg.library()

    def backward(group, q_head, dout_head):
        row = 64 * group
        return lib.bevpool_attention_backward(
            16, row, q_head, 16, 64, 64, 16, 64, 64, 16, None, 16, row, dout_head, 16, 2, 4, 4, group,
            1, 64, 16, 16, 1, 0, 0.125, 16, 16, 16, None, 0, None)

    far = (1 << 23) - 8  # elements: just under 16 MiB
    for group in (65, 256, 1024):
        for heads in ((far, 64), (64, far)):
            assert backward(group, *heads) == -1, (group, heads)
            assert b'heads of a group' in lib.bevpool_last_error()
    reach = (1 << 30) // 256 // 2
    assert backward(256, reach, 64) == -1
    assert b'heads of a group' in lib.bevpool_last_error()
    # within reach: the next check (no scratch) answers
    for group, head in ((256, reach - 8), (4, far), (1024, 64)):
        assert backward(group, head, head) == -3, (group, head)
