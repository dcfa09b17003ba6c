"""CPU oracle of the gated linear recurrence, token by token in float64 (no
reference implementation exists; test infrastructure).

  r = sigmoid(a_t), i = sigmoid(b_t), l = -c softplus(lam) r,
  h_t = exp(l) h_{t-1} + sqrt(1 - exp(2 l)) i x_t

Beside every result stands a bound of what fp32 arithmetic may add to it
(`Err`): each operation's relative error is at most a few units u = 2^-24,
and the bounds follow the same recurrences.  EPS collects the roundings of
one gate: exp(-a) with |a| <= 8 carries (|a| + 2) u from its argument and the
hardware's exponential, the reciprocal, the product with -c softplus(lam)
(itself 4 u), the series of expm1 (5e-8 = 0.8 u truncation, 3 u rounding) and
the square root add 12 u at most, so 24 u cover a gate.

A decay alpha = exp(l) carries keep(l) = |l| EPS + 6 u of itself, however small
it is: l's own relative error (18 u of EPS) and that of the exponential's
argument (1.3 u) are multiplied by |l|; near 1 alpha - 1 = l + l^2 / 2 + ...
carries EPS, and |alpha - 1| <= 1.14 alpha |l| down to l = -1/4, where the
exponential takes over (2 u); the product with the state and the joins of tiles
and waves round a few more times.

Pins (tests/test_oracle_recurrence.py): the closed form for constant gates,
cumulative sums and products for open ones, float64 autograd and central
differences for the gradients.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

U = 2.0 ** -24
EPS = 24 * U


def keep(ell):
    """Relative error of a decay, with its product."""
    return ell.abs() * EPS + 6 * U


def gates(a, b, lam, c):
    """(r, i, l, alpha, s) in float64."""
    a, b, lam = a.double(), b.double(), lam.double()
    r, i = torch.sigmoid(a), torch.sigmoid(b)
    ell = -c * F.softplus(lam) * r
    return r, i, ell, torch.exp(ell), torch.sqrt(-torch.expm1(2 * ell))


def runs(cu, total):
    """[(start, end)] with the kernels' clamping."""
    at = [min(max(int(v), 0), total) for v in cu]
    return list(zip(at[:-1], at[1:]))


def forward(x, a, b, lam, c, h0, cu):
    """x, a, b [tokens, D]; h0 [N, D] or None; cu N + 1 values.  Returns a dict
    of float64 tensors: h, before (h_{t-1}), final, and their error bounds
    h_err, before_err, final_err.  Tokens outside every sequence hold NaN."""
    r, i, ell, alpha, s = gates(a, b, lam, c)
    add = s * i * x.double()
    total, D = x.shape
    out = {k: torch.full((total, D), float("nan"), dtype=torch.float64)
           for k in ("h", "before", "h_err", "before_err")}
    n = len(cu) - 1
    start = torch.zeros(n, D, dtype=torch.float64) if h0 is None else h0.double()
    final, final_err = start.clone(), torch.zeros(n, D, dtype=torch.float64)
    for q, (t0, t1) in enumerate(runs(cu, total)):
        h, e = start[q].clone(), torch.zeros(D, dtype=torch.float64)
        for t in range(t0, t1):
            out["before"][t], out["before_err"][t] = h, e
            e = alpha[t] * (e + h.abs() * keep(ell[t])) + add[t].abs() * EPS
            h = alpha[t] * h + add[t]
            e = e + 2 * U * h.abs()
            out["h"][t], out["h_err"][t] = h, e
        if t1 > t0:
            final[q], final_err[q] = h, e
    out.update(final=final, final_err=final_err)
    return out


def backward(dy, x, a, b, lam, c, h0, dfinal, cu):
    """Gradients and error bounds, in float64: dx, da, db [tokens, D], dlam [D],
    dh0 [N, D], each with its *_err."""
    fwd = forward(x, a, b, lam, c, h0, cu)
    r, i, ell, alpha, s = gates(a, b, lam, c)
    x, dy, lam = x.double(), dy.double(), lam.double()
    total, D = x.shape
    n = len(cu) - 1
    G = torch.full((total, D), float("nan"), dtype=torch.float64)
    Ge = G.clone()
    q = torch.zeros(n, D, dtype=torch.float64) if dfinal is None else dfinal.double().clone()
    qe = torch.zeros_like(q)
    for k, (t0, t1) in enumerate(runs(cu, total)):
        for t in range(t1 - 1, t0 - 1, -1):
            G[t] = dy[t] + q[k]
            Ge[t] = qe[k] + 2 * U * G[t].abs() + 2 * U * q[k].abs()
            q[k] = alpha[t] * G[t]
            qe[k] = alpha[t] * (Ge[t] + G[t].abs() * keep(ell[t]))
    l_s = torch.where(s > 0, ell / s, torch.zeros_like(s))  # tends to 0 with the gate
    part_h, part_u = alpha * fwd["before"] * ell, i * x * alpha * alpha * l_s
    # E = (dL/dl) l; part_h holds a decay once, part_u twice (s has less than
    # half of a decay's error: alpha^2 |l| <= s^2 / 2).
    E = G * (part_h - part_u)
    Ee = ((part_h - part_u).abs() * Ge + G.abs() * (alpha * ell).abs() * fwd["before_err"]
          + G.abs() * (part_h.abs() * (ell.abs() + 2) + part_u.abs() * (2 * ell.abs() + 2)) * EPS)
    out = {"dx": G * s * i, "db": G * s * x * i * (1 - i), "da": E * (1 - r), "dh0": q,
           "dh0_err": qe}
    out["dx_err"] = s * i * Ge + out["dx"].abs() * 2 * EPS
    out["db_err"] = (s * x * i * (1 - i)).abs() * Ge + out["db"].abs() * 3 * EPS
    out["da_err"] = (1 - r) * Ee + out["da"].abs() * EPS
    # dlam = sum E sigmoid(lam) / softplus(lam); at most 64 + tokens / 64
    # additions lie between a term and the sum.
    ratio = torch.where(lam < -30, torch.ones_like(lam), torch.sigmoid(lam) / F.softplus(lam))
    live = torch.zeros(total, dtype=torch.bool)
    for t0, t1 in runs(cu, total):
        live[t0:t1] = True
    out["dlam"] = E[live].sum(0) * ratio
    out["dlam_err"] = (Ee[live].sum(0) + E[live].abs().sum(0) * (64 + total / 64) * U) * ratio
    return out


def update(x, a, b, lam, c, pool, slots, accepted, cu):
    """x, a, b [tokens, D]; pool [slots, D]; slots a list of slot numbers or of
    lists of them (a column for each token), or None; accepted a list or None.
    Returns (y [tokens, D], new pool) with error bounds (y_err, pool_err)."""
    r, i, ell, alpha, s = gates(a, b, lam, c)
    add = s * i * x.double()
    y = torch.full(x.shape, float("nan"), dtype=torch.float64)
    y_err, start = y.clone(), pool.double()
    new, new_err = start.clone(), torch.zeros_like(start)
    lines = pool.size(0)
    for q, (t0, t1) in enumerate(runs(cu, x.size(0))):
        row = [q] if slots is None else slots[q]
        wide = isinstance(row, (list, tuple)) and slots is not None
        row = list(row) if wide else [row] if slots is not None else [q]
        col = 0 if accepted is None else min(max(accepted[q] - 1, 0), len(row) - 1)
        first = row[col]
        ok = 0 <= first < lines
        h = start[first].clone() if ok else torch.zeros_like(lam, dtype=torch.float64)
        e = torch.zeros_like(h)
        for t in range(t0, t1):
            e = alpha[t] * (e + h.abs() * keep(ell[t])) + add[t].abs() * EPS
            h = alpha[t] * h + add[t]
            e = e + 2 * U * h.abs()
            y[t], y_err[t] = h, e
            k = t - t0
            if wide and k < len(row) and 0 <= row[k] < lines:
                new[row[k]], new_err[row[k]] = h, e
        if not wide and ok and t1 > t0:
            new[first], new_err[first] = h, e
    return y, y_err, new, new_err
