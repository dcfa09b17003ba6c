"""CPU oracle of the step from one block to the next, in float64 (no reference
implementation exists; test infrastructure).

  n = x rstd1 w1', v = n silu(z), h = residual + scale v, y = h rstd2 w2'

with w' = weight or 1 + weight, parts that are None left out, and the
gradients of all inputs.  Beside every result stands a bound of what fp32
arithmetic may add (`*_err`), u = 2^-24: a sum over N elements passes at most
64 additions in a lane and 16 across lanes and waves (80 u of the sum of
magnitudes), a gate's sigmoid at |z| <= 8 carries 14 u.

Pins (tests/test_oracle_residual_norm.py): torch's RMSNorm, float64 autograd
and central differences.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24
SUM = 80 * U
GATE = 14 * U


def _wide(t):
    return None if t is None else t.double()


def forward(x, res, post, gate, scale, pre, eps, unit_offset=False):
    """x, res, gate [rows, N]; weights [N].  Returns a dict of float64 tensors:
    h, y, r1, r2 and what the backward pass uses, with error bounds."""
    x, res, post, gate, scale, pre = map(_wide, (x, res, post, gate, scale, pre))
    off = 1.0 if unit_offset else 0.0
    o = {}
    rel = 2 * U  # relative error of v
    if post is not None:
        o["r1"] = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        o["xh"] = x * o["r1"]
        o["w1"] = post + off
        n = o["xh"] * o["w1"]
        rel += SUM + 6 * U
    else:
        n = x
    v = n
    if gate is not None:
        o["sg"] = torch.sigmoid(gate)
        v = n * gate * o["sg"]
        rel += GATE
    o["n"], o["v"], o["z"] = n, v, gate
    o["s"] = torch.ones_like(x[0]) if scale is None else scale
    o["h"] = res + o["s"] * v
    o["h_err"] = (o["s"] * v).abs() * rel + 2 * U * o["h"].abs()
    o["v_rel"] = rel
    if pre is not None:
        ms = o["h"].square().mean(-1, keepdim=True)
        o["r2"] = 1 / torch.sqrt(ms + eps)
        # relative error of r2: half of that of the mean of squares
        o["r2_rel"] = (o["h"].abs() * o["h_err"]).mean(-1, keepdim=True) / (ms + eps) + SUM
        o["w2"] = pre + off
        o["y"] = o["h"] * o["r2"] * o["w2"]
        o["y_err"] = (o["r2"] * o["w2"]).abs() * o["h_err"] + o["y"].abs() * (o["r2_rel"] + 6 * U)
    return o


def backward(dh, dy, x, res, post, gate, scale, pre, eps, unit_offset=False):
    """Gradients dx, dres, dgate, dpost, dscale, dpre (those of given parts),
    with error bounds."""
    o = forward(x, res, post, gate, scale, pre, eps, unit_offset)
    x = x.double()
    rows = x.size(0)
    sums = (64 + rows / 16) * U  # additions between a row's term and the column sum
    g = torch.zeros_like(x) if dh is None else dh.double()
    e = torch.zeros_like(x)
    out = {}
    if pre is not None:
        dyf = torch.zeros_like(x) if dy is None else dy.double()
        hh = o["h"] * o["r2"]
        hh_err = o["h_err"] * o["r2"] + hh.abs() * (o["r2_rel"] + 2 * U)
        out["dpre"] = (dyf * hh).sum(0)
        out["dpre_err"] = (dyf.abs() * hh_err).sum(0) + (dyf * hh).abs().sum(0) * sums
        wd = o["w2"] * dyf
        m = (wd * hh).mean(-1, keepdim=True)
        m_err = ((wd.abs() * hh_err).mean(-1, keepdim=True)
                 + (wd * hh).abs().mean(-1, keepdim=True) * SUM)
        inner = wd.abs() + (hh * m).abs()
        g = g + o["r2"] * (wd - hh * m)
        e = (o["r2"] * (hh.abs() * m_err + hh_err * m.abs() + inner * (6 * U + o["r2_rel"]))
             + 2 * U * g.abs())
    out["dres"], out["dres_err"] = g, e
    if scale is not None:
        out["dscale"] = (g * o["v"]).sum(0)
        out["dscale_err"] = ((e * o["v"].abs() + (g * o["v"]).abs() * (o["v_rel"] + 2 * U)).sum(0)
                             + (g * o["v"]).abs().sum(0) * sums)
    g, e = g * o["s"], e * o["s"].abs() + (g * o["s"]).abs() * U
    if gate is not None:
        z, sg = o["z"], o["sg"]
        slope = sg * (1 + z * (1 - sg))
        # 1 + z (1 - sg) cancels near its zero: its own error is absolute.
        slope_err = slope.abs() * GATE + sg * (1 + (z * (1 - sg)).abs()) * 2 * GATE
        out["dgate"] = g * o["n"] * slope
        out["dgate_err"] = ((o["n"] * slope).abs() * e + (g * o["n"]).abs() * slope_err
                            + out["dgate"].abs() * o["v_rel"])
        g, e = g * z * sg, e * (z * sg).abs() + (g * z * sg).abs() * GATE
    if post is not None:
        out["dpost"] = (g * o["xh"]).sum(0)
        term = (g * o["xh"]).abs()
        out["dpost_err"] = ((e * o["xh"].abs() + term * (SUM + 6 * U)).sum(0)
                            + term.sum(0) * sums)
        wg, we = g * o["w1"], e * o["w1"].abs()
        m = (wg * o["xh"]).mean(-1, keepdim=True)
        m_err = ((we * o["xh"].abs()).mean(-1, keepdim=True)
                 + (wg * o["xh"]).abs().mean(-1, keepdim=True) * 2 * SUM)
        g = o["r1"] * (wg - o["xh"] * m)
        e = o["r1"] * (we + o["xh"].abs() * m_err
                       + (wg.abs() + (o["xh"] * m).abs()) * (2 * SUM + 8 * U))
    out["dx"], out["dx_err"] = g, e
    return out
