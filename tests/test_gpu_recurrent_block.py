"""A recurrent block as it is used: causal conv1d, gated linear recurrence, and
the block-to-block norm.  Served: a packed prefill, then single tokens over the
same state slots, eager and from a captured graph.  Trained: forward and
backward through both operators against float64 autograd."""
import pytest
import torch

from oracle import conv1d as oc
from oracle import recurrence as orc
from oracle import residual_norm as orn
from rounding_tol import assert_within

pytestmark = pytest.mark.gpu

C, EPS, W = 8.0, 1e-6, 4
BF16 = torch.bfloat16


def _rand(g, *shape, dtype=BF16, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g).clamp_(-4, 4) * std + mean).to(dtype)


def _layer(g, D, dev):
    p = {"conv": _rand(g, D, W, std=0.5), "wa": _rand(g, D), "ba": _rand(g, D), "wb": _rand(g, D),
         "bb": _rand(g, D), "wz": _rand(g, D), "post": _rand(g, D, std=0.1, mean=1.0),
         "scale": _rand(g, D, std=0.1, mean=0.5), "pre": _rand(g, D, std=0.1, mean=1.0)}
    p["lam"] = torch.log(torch.expm1(10.0 ** (-4 * torch.rand(D, generator=g)))).float()
    return {k: v.to(dev) for k, v in p.items()}


def _step(p, u, res, conv, pool, slots, cu, longest):
    """One layer over the tokens of u (packed sequences, or one token each
    where longest is 1); what it computed, for the checks."""
    from torch_npu_ops_amd import _xk_torch as xt, ops
    x = ops.npu_causal_conv1d_update_v2(u, conv, p["conv"], True, None, slots, cu, longest, -1,
                                        state_rule=1)
    a, b, z = x * p["wa"] + p["ba"], x * p["wb"] + p["bb"], u * p["wz"]
    if longest == 1:
        y = xt.npu_gated_linear_recurrence_update(x, a, b, p["lam"], pool, C, slots)
    else:
        at = slots.long()
        y, fin, _ = xt.npu_gated_linear_recurrence(x[None], a[None], b[None], p["lam"], C,
                                                   pool[at], True, cu)
        y, pool[at] = y[0], fin
    h, out, _, _ = xt.npu_gated_residual_rms_norm(y, res, p["post"], z, p["scale"], p["pre"], EPS)
    return dict(u=u, res=res, x=x, a=a, b=b, z=z, y=y, h=h, out=out)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("D", [258, 1024])
def test_prefill_then_single_tokens(dev, D, graph):
    g = torch.Generator().manual_seed(D)
    lens, more = [37, 1, 130, 16], 6
    n, total = len(lens), sum(lens)
    layers = [_layer(g, D, dev) for _ in range(2)]
    slots = torch.tensor([4, 0, 5, 2], dtype=torch.int32, device=dev)
    convs = [torch.zeros(6, D, W - 1, dtype=BF16, device=dev) for _ in layers]
    pools = [torch.zeros(6, D, device=dev) for _ in layers]
    for pool in pools:
        pool[[1, 3]] = 7.0  # slots of others
    ends = torch.tensor([0] + lens).cumsum(0)
    cu = ends.int().to(dev)
    one = torch.arange(n + 1, dtype=torch.int32, device=dev)
    tokens = [_rand(g, total, D).to(dev)] + [_rand(g, n, D).to(dev) for _ in range(more)]

    def stack(u, where, longest):
        got, res = [], u
        for p, conv, pool in zip(layers, convs, pools):
            got.append(_step(p, u, res, conv, pool, slots, where, longest))
            u, res = got[-1]["out"], got[-1]["h"]
        return got
    runs = [stack(tokens[0], cu, max(lens))]
    if graph:
        still = tokens[1].clone()
        kept = [t.clone() for t in convs + pools]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            stack(still, one, 1)
        torch.cuda.current_stream().wait_stream(side)
        for t, k in zip(convs + pools, kept):
            t.copy_(k)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            live = stack(still, one, 1)
        for u in tokens[1:]:
            still.copy_(u)
            captured.replay()
            runs.append([{k: v.clone() for k, v in layer.items()} for layer in live])
            torch.cuda.synchronize()
    else:
        runs += [stack(u, one, 1) for u in tokens[1:]]

    for pool in pools:
        assert (pool[[1, 3]] == 7.0).all()
    for k, (p, pool) in enumerate(zip(layers, pools)):
        p = {name: v.cpu() for name, v in p.items()}
        for s in range(n):
            def whole(name):
                first = runs[0][k][name][int(ends[s]):int(ends[s + 1])]
                return torch.cat([first] + [r[k][name][s:s + 1] for r in runs[1:]]).cpu()
            u, x, a, b, y = (whole(name) for name in ("u", "x", "a", "b", "y"))
            want = oc.causal_conv1d_update_v2(
                u, torch.zeros(1, D, W - 1, dtype=BF16), p["conv"], None, True, None,
                torch.tensor([0, len(u)], dtype=torch.int32), len(u), state_rule=1)[0]
            # Four products and SiLU in fp32, one rounding to bf16.
            torch.testing.assert_close(x.float(), want.float(), rtol=2.0 ** -7, atol=1e-5)
            ref = orc.forward(x, a, b, p["lam"], C, None, [0, len(u)])
            assert_within(y, ref["h"], ref["h_err"], f"layer {k} sequence {s}")
            assert_within(pool[int(slots[s])], ref["final"][0], ref["final_err"][0], "state")
            o = orn.forward(y, whole("res"), p["post"], whole("z"), p["scale"], p["pre"], EPS)
            assert_within(whole("h"), o["h"], o["h_err"], "h")
            assert_within(whole("out"), o["y"], o["y_err"], "out")


class _Recurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, lam, h0, cu):
        from torch_npu_ops_amd import _xk_torch as xt
        y, fin, states = xt.npu_gated_linear_recurrence(x, a, b, lam, C, h0, True, cu, True)
        ctx.save_for_backward(x, a, b, lam, states, h0, cu)
        return y, fin

    @staticmethod
    def backward(ctx, dy, dfin):
        from torch_npu_ops_amd import _xk_torch as xt
        x, a, b, lam, states, h0, cu = ctx.saved_tensors
        return *xt.npu_gated_linear_recurrence_bwd(dy, x, a, b, lam, states, C, h0, dfin, cu), None


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, post, gate, scale, pre):
        from torch_npu_ops_amd import _xk_torch as xt
        h, y, r1, r2 = xt.npu_gated_residual_rms_norm(x, res, post, gate, scale, pre, EPS)
        ctx.save_for_backward(x, res, r1, r2, post, gate, scale, pre)
        return h, y

    @staticmethod
    def backward(ctx, dh, dy):
        from torch_npu_ops_amd import _xk_torch as xt
        dx, dres, dgate, dpost, dscale, dpre = xt.npu_gated_residual_rms_norm_bwd(
            dh, dy, *ctx.saved_tensors)
        return dx, dres, dpost, dgate, dscale, dpre


def _recurrence64(x, a, b, lam, h0, cu):
    r, i = torch.sigmoid(a), torch.sigmoid(b)
    ell = -C * torch.nn.functional.softplus(lam) * r
    add = torch.sqrt(-torch.expm1(2 * ell)) * i * x
    ys, fins = [], []
    for s, (t0, t1) in enumerate(zip(cu[:-1], cu[1:])):
        h = h0[s]
        for t in range(t0, t1):
            h = torch.exp(ell[0, t]) * h + add[0, t]
            ys.append(h)
        fins.append(h)
    return torch.stack(ys)[None], torch.stack(fins)


def _norm64(x, res, post, gate, scale, pre):
    def rms(v):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
    h = res + scale * (rms(x) * post * torch.nn.functional.silu(gate))
    return h, rms(h) * pre


def test_training_step_of_two_layers(dev):
    # fp32.  An operator's result is off by at most 2e-5 of its terms' size (the
    # oracles' bounds, some 250 units of 2^-24); through four operators and
    # back, 1.6e-4; a sum over the tokens may be smaller than its terms by a
    # few times, so the largest element of each gradient times 1e-3 covers it.
    g = torch.Generator().manual_seed(3)
    D, lens = 96, [60, 1, 33]
    ends = [0] + torch.tensor(lens).cumsum(0).tolist()
    T = ends[-1]
    leaves = {"u": torch.randn(1, T, D, generator=g), "h0": torch.randn(2, len(lens), D, generator=g)}
    for k in range(2):
        p = _layer(g, D, "cpu")
        leaves.update({f"{n}{k}": v.float() for n, v in p.items() if n != "conv"})
    cot = [torch.randn(1, T, D, generator=g) for _ in range(2)]
    cot.append(torch.randn(2, len(lens), D, generator=g))

    def loss(p, recurrence, norm, cu, cot):
        u, res, total = p["u"], p["u"], 0.0
        for k in range(2):
            q = {n: p[f"{n}{k}"] for n in ("wa", "ba", "wb", "bb", "wz", "lam", "post", "scale",
                                           "pre")}
            y, fin = recurrence(u, u * q["wa"] + q["ba"], u * q["wb"] + q["bb"], q["lam"],
                                p["h0"][k], cu)
            res, u = norm(y, res, q["post"], u * q["wz"], q["scale"], q["pre"])
            total = total + (fin * cot[2][k]).sum()
        return total + (res * cot[0]).sum() + (u * cot[1]).sum()

    mine = {n: v.to(dev).requires_grad_() for n, v in leaves.items()}
    cud = torch.tensor(ends, dtype=torch.int32, device=dev)
    loss(mine, _Recurrence.apply, _Norm.apply, cud, [c.to(dev) for c in cot]).backward()
    wide = {n: v.double().requires_grad_() for n, v in leaves.items()}
    loss(wide, _recurrence64, _norm64, ends, [c.double() for c in cot]).backward()
    for n in leaves:
        want = wide[n].grad
        off = (mine[n].grad.cpu().double() - want).abs().max()
        assert off <= 1e-3 * want.abs().max(), f"{n}: {off} of {want.abs().max()}"
