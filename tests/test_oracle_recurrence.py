"""Pins of oracle/recurrence.py (CPU): closed forms, float64 autograd and
central differences."""
import math

import pytest
import torch

from oracle import recurrence as orc


def _rand(seed, total, D, n):
    g = torch.Generator().manual_seed(seed)
    x, a, b, dy = (torch.randn(total, D, generator=g, dtype=torch.float64) for _ in range(4))
    lam = torch.randn(D, generator=g, dtype=torch.float64) * 2 - 3
    h0, df = (torch.randn(n, D, generator=g, dtype=torch.float64) for _ in range(2))
    return x, a, b, dy, lam, h0, df


def test_constant_gates_have_the_geometric_closed_form():
    # alpha and the input constant: h_t = alpha^t h_0 + (1 - alpha^t) / (1 - alpha) s i x
    T, lam, c = 40, torch.tensor([-4.0, 0.5]), 8.0
    a, b, x = torch.full((T, 2), 0.3), torch.full((T, 2), -0.7), torch.full((T, 2), 1.5)
    h0 = torch.tensor([[2.0, -1.0]])
    h = orc.forward(x, a, b, lam, c, h0, [0, T])["h"]
    for ch in range(2):
        r = 1 / (1 + math.exp(-0.3))
        alpha = math.exp(-c * math.log1p(math.exp(float(lam[ch]))) * r)
        inp = math.sqrt(1 - alpha * alpha) / (1 + math.exp(0.7)) * 1.5
        for t in (1, 7, T):
            want = alpha ** t * float(h0[0, ch]) + (1 - alpha ** t) / (1 - alpha) * inp
            assert h[t - 1, ch].item() == pytest.approx(want, rel=1e-6)


def test_a_closed_decay_gate_keeps_the_state_and_an_open_one_forgets_it():
    x = torch.randn(5, 1)
    inf = torch.full((5, 1), float("inf"))
    keep = orc.forward(x, -inf, inf, torch.tensor([0.0]), 8.0, torch.tensor([[3.0]]), [0, 5])
    assert torch.equal(keep["h"], torch.full((5, 1), 3.0, dtype=torch.float64))
    lose = orc.forward(x, inf, inf, torch.tensor([60.0]), 8.0, torch.tensor([[3.0]]), [0, 5])
    torch.testing.assert_close(lose["h"], x.double())  # alpha = exp(-480): s = 1


def test_sequences_do_not_touch_each_other_and_rows_outside_are_not_computed():
    x, a, b, _, lam, h0, _ = _rand(1, 12, 3, 4)
    cu = [1, 4, 4, 9, 11]
    out = orc.forward(x, a, b, lam, 8.0, h0, cu)
    for q, (t0, t1) in enumerate(zip(cu[:-1], cu[1:])):
        one = orc.forward(x[t0:t1], a[t0:t1], b[t0:t1], lam, 8.0, h0[q:q + 1], [0, t1 - t0])
        assert torch.equal(out["h"][t0:t1], one["h"])
        assert torch.equal(out["final"][q], one["final"][0])
    assert torch.equal(out["final"][1], h0[1])
    assert out["h"][[0, 11]].isnan().all()


def _loss(x, a, b, lam, h0, dy, df, cu, c):
    """The sum that the gradients belong to, from plain differentiable torch."""
    r, i = torch.sigmoid(a), torch.sigmoid(b)
    alpha = torch.exp(-c * torch.log1p(torch.exp(lam)) * r)
    add = torch.sqrt(1 - alpha ** 2) * i * x
    loss = 0.0
    for q, (t0, t1) in enumerate(zip(cu[:-1], cu[1:])):
        h = h0[q]
        for t in range(t0, t1):
            h = alpha[t] * h + add[t]
            loss = loss + (h * dy[t]).sum()
        loss = loss + (h * df[q]).sum()
    return loss


@pytest.mark.parametrize("c", [8.0, 0.7])
def test_gradients_match_autograd(c):
    cu = [0, 1, 1, 14, 20]
    x, a, b, dy, lam, h0, df = _rand(2, 20, 5, 4)
    leaves = [t.clone().requires_grad_() for t in (x, a, b, lam, h0)]
    want = torch.autograd.grad(_loss(*leaves, dy, df, cu, c), leaves)
    got = orc.backward(dy, x, a, b, lam, c, h0, df, cu)
    for name, w in zip(("dx", "da", "db", "dlam", "dh0"), want):
        torch.testing.assert_close(got[name], w, rtol=1e-9, atol=1e-11)


def test_gradients_match_differences():
    cu = [0, 7, 9]
    x, a, b, dy, lam, h0, df = _rand(3, 9, 2, 2)
    got = orc.backward(dy, x, a, b, lam, 8.0, h0, df, cu)
    args, step = [x, a, b, lam, h0], 1e-5
    for name, k in (("dx", 0), ("da", 1), ("db", 2), ("dlam", 3), ("dh0", 4)):
        for at in range(0, args[k].numel(), 3):
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in args]
                moved[k].view(-1)[at] += sign * step
                ends.append(float(_loss(*moved, dy, df, cu, 8.0)))
            want = (ends[0] - ends[1]) / (2 * step)
            assert got[name].reshape(-1)[at].item() == pytest.approx(want, rel=2e-6, abs=2e-8)


def test_closed_gate_gradients_are_the_finite_limits():
    # a = -1000: r underflows to 0 in float64, s = 0; nothing is NaN and da is 0.
    x, a, b, dy, lam, h0, df = _rand(4, 3, 2, 1)
    got = orc.backward(dy, x, torch.full_like(a, -1000.0), b, lam, 8.0, h0, df, [0, 3])
    for name in ("dx", "da", "db", "dlam", "dh0"):
        assert got[name].isfinite().all()
    assert (got["da"] == 0).all() and (got["dx"] == 0).all()
    torch.testing.assert_close(got["dh0"][0], dy.sum(0) + df[0])


def test_update_is_the_forward_pass_token_by_token():
    x, a, b, _, lam, h0, _ = _rand(5, 6, 4, 2)
    want = orc.forward(x, a, b, lam, 8.0, h0, [0, 3, 6])
    pool = torch.cat([h0, torch.zeros(5, 4, dtype=torch.float64)])
    slots = [[0, 2, 3], [1, 4, 5]]
    y, _, new, _ = orc.update(x, a, b, lam, 8.0, pool, slots, [1, 1], [0, 3, 6])
    torch.testing.assert_close(y, want["h"])
    torch.testing.assert_close(new[[0, 2, 3, 1, 4, 5]], want["h"])  # a slot after every token
    # two accepted tokens: the next window starts from column 1
    y2, _, _, _ = orc.update(x, a, b, lam, 8.0, new, slots, [2, 3], [0, 3, 6])
    start = torch.stack([want["h"][1], want["h"][5]])
    torch.testing.assert_close(y2, orc.forward(x, a, b, lam, 8.0, start, [0, 3, 6])["h"])
    # a slot outside the pool starts from zero and is not written
    y3, _, same, _ = orc.update(x[:1], a[:1], b[:1], lam, 8.0, pool, [-1], None, [0, 1])
    torch.testing.assert_close(y3, orc.forward(x[:1], a[:1], b[:1], lam, 8.0, None, [0, 1])["h"])
    assert torch.equal(same, pool)
