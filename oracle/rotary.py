"""CPU oracle of rotary positions and of the write into a paged cache, in
float64 (no reference implementation in this form; test infrastructure).

  (u, v) -> L (u cos a - v sin a, v cos a + u sin a), a = position * frequency

on pairs (i, i + r/2) or (2i, 2i + 1) of the first r elements of a head.

Beside every result stands a bound of what the kernel's arithmetic may add:
the angle's rest (at most pi/4) is rounded to fp32 (2^-25), its cosine and
sine are off by 2 steps at most (2^-22 for values up to 1), one rounding by L,
one of each product and one of the sum: 8 * 2^-23 of L (|u| + |v|).

Pins (tests/test_oracle_rotary.py): complex multiplication, the rows of the
framework's other rotations, and float64 autograd.
"""
from __future__ import annotations

import torch

ERR = 2.0 ** -20


def turn(x, positions, inv_freq, interleaved=False, scale=1.0, inverse=False):
    """x [..., heads, D], positions [...], inv_freq [r / 2]: (result, bound)."""
    half = inv_freq.numel()
    a = (positions.double()[..., None] * inv_freq.double())[..., None, :]
    c, s = scale * torch.cos(a), scale * torch.sin(a) * (-1 if inverse else 1)
    y, err = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    if interleaved:
        iu, iv = torch.arange(0, 2 * half, 2), torch.arange(1, 2 * half, 2)
    else:
        iu, iv = torch.arange(half), torch.arange(half, 2 * half)
    u, v = y[..., iu], y[..., iv]
    bound = ERR * scale * (u.abs() + v.abs())
    y[..., iu], y[..., iv] = u * c - v * s, v * c + u * s
    err[..., iu], err[..., iv] = bound, bound
    return y, err


def append(cache, rows, err, slots, scale=None):
    """rows [tokens, heads, D] (and their bounds) into their slots of cache
    [pages, page, heads, D]: (whole cache, bound), for e4m3 before rounding."""
    whole = cache.double().flatten(0, 1).clone()
    bound = torch.zeros_like(whole)
    if scale is not None:
        rows, err = rows / scale.double()[:, None], err / scale.double()[:, None]
        err = err + rows.abs() * 2.0 ** -24
        rows = rows.clamp(-448, 448)
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < whole.size(0):
            whole[slot], bound[slot] = rows[t], err[t]
    return whole.view(cache.shape), bound.view(cache.shape)
