"""CPU oracle of the attention of new tokens over a paged key-value cache, in
float64 (no reference implementation in this form; test infrastructure).

Beside every result stands a bound of what the kernel's arithmetic may add.
u = 2^-24.  A score is a product of D terms added in fp32 and two more
roundings: ds = (D + 8) u scale sum |q k|, and its part of the exponent a
rounding of what it is taken from (u of the largest |score|, twice).  A weight
is off by that, by its exponential (4 u) and by its parts (two of fp16 2^-21,
three of bf16 u, among the roundings at the end).  The sums of n weights
pass at most 32 additions in a product, n / 16 in a lane and 64 between lanes,
waves and parts.  The result is off by what the weights are, twice (the sum
that it is divided by has the same bound), and a few roundings.

Pins (tests/test_oracle_paged_attention.py): torch's softmax attention over
dense keys, and sums over parts joined by their lse.
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24
SPLIT = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -21, torch.float32: 0.0}


def gather(cache, row, length):
    """Positions 0 .. length - 1 of a sequence: (values [length, Hkv, D] in
    float64, which of them are in a page that exists)."""
    pages, page, hkv, d = cache.shape
    out = torch.zeros(length, hkv, d, dtype=torch.float64)
    there = torch.zeros(length, dtype=torch.bool)
    for j in range(0, length, page):
        e = int(row[j // page])
        n = min(page, length - j)
        if 0 <= e < pages:
            out[j:j + n] = cache[e, :n].double()
            there[j:j + n] = True
    return out, there


def attention(q, k_cache, v_cache, table, lens, scale=None, window=0, k_scale=None,
              v_scale=None):
    """q [B, T, Hq, D]: dict of o, lse and their bounds o_err, lse_err."""
    dtype = q.dtype
    q = q.double()
    B, T, Hq, D = q.shape
    Hkv, page = k_cache.size(2), k_cache.size(1)
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    o, o_err = torch.zeros(B, T, Hq, D, dtype=torch.float64), torch.zeros(B, T, Hq, D,
                                                                       dtype=torch.float64)
    lse = torch.full((B, T, Hq), -math.inf, dtype=torch.float64)
    lse_err = torch.zeros(B, T, Hq, dtype=torch.float64)
    for b in range(B):
        length = max(0, min(int(lens[b]), table.size(1) * page if k_cache.size(0) else 0))
        k, there = gather(k_cache, table[b], length)
        v, _ = gather(v_cache, table[b], length)
        if k_scale is not None:
            k = k * k_scale.double()[:, None]
        if v_scale is not None:
            v = v * v_scale.double()[:, None]
        for t in range(T):
            at = length - T + t
            seen = there & (torch.arange(length) <= at)
            if window:
                seen &= torch.arange(length) > at - window
            if not seen.any():
                continue
            ks = k[seen].repeat_interleave(G, 1).transpose(0, 1)  # [Hq, n, D]
            vs = v[seen].repeat_interleave(G, 1).transpose(0, 1)
            n = ks.size(1)
            s = scale * (ks @ q[b, t][:, :, None])[..., 0]
            ds = (D + 8) * U * abs(scale) * (ks.abs() @ q[b, t].abs()[:, :, None])[..., 0]
            delta = ds.amax(-1) + 4 * U * s.abs().amax(-1) + 8 * U
            depth = (n / 16 + 96) * U
            rel = torch.expm1(2 * delta) + SPLIT[dtype] + 2 * depth + 8 * U
            p = torch.softmax(s, -1)[:, None]
            o[b, t] = (p @ vs)[:, 0]
            o_err[b, t] = (p @ vs.abs())[:, 0] * rel[:, None]
            lse[b, t] = torch.logsumexp(s, -1)
            lse_err[b, t] = delta + depth + 4 * U * (1 + lse[b, t].abs())
    return {"o": o, "o_err": o_err, "lse": lse, "lse_err": lse_err}
