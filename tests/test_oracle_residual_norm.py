"""Pins of oracle/residual_norm.py (CPU): torch's RMSNorm, float64 autograd and
central differences."""
import itertools

import pytest
import torch
import torch.nn.functional as F

from oracle import residual_norm as orn

EPS = 1e-6


def _rand(seed, M, N):
    g = torch.Generator().manual_seed(seed)
    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)
    return {"x": r(M, N), "res": r(M, N), "post": r(N), "gate": r(M, N), "scale": r(N),
            "pre": r(N), "dh": r(M, N), "dy": r(M, N)}


def _plain(p, off):
    """(h, y) from torch's library functions."""
    N = p["x"].size(-1)
    v = p["x"]
    if p["post"] is not None:
        v = F.rms_norm(v, (N,), p["post"] + off, EPS)
    if p["gate"] is not None:
        v = v * F.silu(p["gate"])
    if p["scale"] is not None:
        v = v * p["scale"]
    h = p["res"] + v
    return h, (F.rms_norm(h, (N,), p["pre"] + off, EPS) if p["pre"] is not None else None)


CHOICES = list(itertools.product([False, True], repeat=4))


@pytest.mark.parametrize("post,gate,scale,pre", CHOICES)
@pytest.mark.parametrize("offset", [False, True])
def test_forward_and_gradients_match_torch(post, gate, scale, pre, offset):
    p = _rand(1, 3, 7)
    for name, keep in (("post", post), ("gate", gate), ("scale", scale), ("pre", pre)):
        if not keep:
            p[name] = None
    args = [p[k] for k in ("x", "res", "post", "gate", "scale", "pre")]
    o = orn.forward(*args, EPS, offset)
    h, y = _plain(p, 1.0 if offset else 0.0)
    torch.testing.assert_close(o["h"], h)
    if pre:
        torch.testing.assert_close(o["y"], y)
    names = [k for k in ("x", "res", "post", "gate", "scale", "pre") if p[k] is not None]
    leaves = {k: p[k].clone().requires_grad_() for k in names}
    h, y = _plain({**p, **leaves}, 1.0 if offset else 0.0)
    loss = (h * p["dh"]).sum() + ((y * p["dy"]).sum() if pre else 0)
    want = torch.autograd.grad(loss, [leaves[k] for k in names])
    got = orn.backward(p["dh"], p["dy"] if pre else None, *args, EPS, offset)
    for k, w in zip(names, want):
        torch.testing.assert_close(got["d" + k], w, rtol=1e-9, atol=1e-11)


def test_gradients_match_differences():
    p = _rand(2, 2, 5)
    keys = ("x", "res", "post", "gate", "scale", "pre")
    got = orn.backward(p["dh"], p["dy"], *[p[k] for k in keys], EPS)
    step = 1e-6
    for k in keys:
        for at in range(0, p[k].numel(), 2):
            ends = []
            for sign in (1, -1):
                moved = p[k].clone()
                moved.view(-1)[at] += sign * step
                o = orn.forward(*[moved if q == k else p[q] for q in keys], EPS)
                ends.append(float((o["h"] * p["dh"]).sum() + (o["y"] * p["dy"]).sum()))
            want = (ends[0] - ends[1]) / (2 * step)
            assert got["d" + k].reshape(-1)[at].item() == pytest.approx(want, rel=1e-6, abs=1e-8)


def test_a_missing_gradient_counts_as_zero():
    p = _rand(3, 2, 6)
    args = [p[k] for k in ("x", "res", "post", "gate", "scale", "pre")]
    zero = torch.zeros_like(p["dh"])
    for dh, dy in ((None, p["dy"]), (p["dh"], None)):
        got = orn.backward(dh, dy, *args, EPS)
        want = orn.backward(zero if dh is None else dh, zero if dy is None else dy, *args, EPS)
        for k in ("dx", "dres", "dgate", "dpost", "dscale", "dpre"):
            torch.testing.assert_close(got[k], want[k])
