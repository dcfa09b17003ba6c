"""CPU oracle of rotary positions and of the write into a paged cache, in
float64 (no reference implementation in this form; test infrastructure).

  (u, v) -> L (u cos a - v sin a, v cos a + u sin a), a = position * frequency

on pairs (i, i + r/2) or (2i, 2i + 1) of the first r elements of a head.

Beside every result stands a bound of what the kernel's arithmetic may add,
for positions up to 2^29.  With h = 2^-25, half a step of fp32 below 1, the
angle's rest r (at most pi/4) is off by h when it is rounded, its square z by
2 h z.  Cosine: 1 + z p with |p| <= 1/2, p off by 0.63 h (its last step, 1/24's
rounding): 0.39 h, z 0.62 h, the sum's rounding h, the rest 0.71 h, in all
2.8 h.  Sine: r + z r p with |p| <= 1/6, p off by 0.52 h: 0.26 h, z r twice
rounded 0.33 h, the end of the series 0.06 h, the sum h, the rest 0.88 h, in all
2.8 h.  Then each is rounded by the product with L (2 h of it), the products
with u and v (2 h of them); the last rounding is the output's.  In all 2.8 h +
4 h of L (|u| + |v|).

Pins (tests/test_oracle_rotary.py): complex multiplication, the rows of the
framework's other rotations, and float64 autograd.
"""
from __future__ import annotations

import torch

TURN = 2.8 * 2.0 ** -25  # of a cosine or sine
ERR = TURN + 4 * 2.0 ** -25


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
