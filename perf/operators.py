"""The gated linear recurrence and the norms between two blocks, as cases that
can be timed and checked: the plain form of each operator (elementary torch
operations in fp32, rounded once), the framework's call, and the same in 64
bits.

Families (the "op" of a case):

  scan    prefill: h_t = alpha_t h_{t-1} + sqrt(1 - alpha_t^2) sigmoid(b_t) x_t
          with alpha_t = exp(-c softplus(lam) sigmoid(a_t)), per channel, over
          ragged sequences that go on from a state; outputs and final states
  update  decode: the same step for one token of every sequence of a batch (or
          a few drafted tokens of each, a state kept for every one of them), on
          a pool of states
  train   scan, then its backward pass: gradients of x, a, b, lam and the
          initial states
  norm    the step from one block to the next: RMSNorm of the block's output,
          its SiLU gate and residual scale, the residual sum, and the RMSNorm
          that the next block reads
  ntrain  norm, then its backward pass

The gates' two projections come as one wide row, as one product leaves them,
and a and b are views of it.
"""
import math
import random

import torch

own = False

DEV = "cuda"
C = 8.0
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # Prefill of a full batch: 8 ragged prompts.
        {"name": "scan_prefill", "op": "scan", "tokens": 16384, "seqs": 8, "dim": 4096,
         "dtype": "bf16"},
        # One long prompt on a rank's share of the channels: few columns, many steps.
        {"name": "scan_long", "op": "scan", "tokens": 32768, "seqs": 1, "dim": 1024,
         "dtype": "bf16"},
        # A small ragged batch of an odd width in full precision.
        {"name": "scan_odd", "op": "scan", "tokens": 5003, "seqs": 3, "dim": 1125,
         "dtype": "f32"},
        # A single user's token: the smallest call, all latency.
        {"name": "update_1", "op": "update", "batch": 1, "tokens": 1, "dim": 4096,
         "dtype": "bf16"},
        # A full decode batch.
        {"name": "update_256", "op": "update", "batch": 256, "tokens": 1, "dim": 4096,
         "dtype": "bf16"},
        # Speculative decoding: 3 draft tokens and the last accepted one.
        {"name": "verify_64", "op": "update", "batch": 64, "tokens": 4, "dim": 2048,
         "dtype": "f16"},
        # A training step of a few packed documents.
        {"name": "scan_train", "op": "train", "tokens": 8192, "seqs": 4, "dim": 4096,
         "dtype": "bf16"},
        # Training in full precision, one document, a rank's share of the channels.
        {"name": "scan_train_f32", "op": "train", "tokens": 4099, "seqs": 1, "dim": 640,
         "dtype": "f32"},
        # Between two blocks of a full prefill batch.
        {"name": "norm_prefill", "op": "norm", "rows": 16384, "hidden": 4096, "dtype": "bf16",
         "residual": "bf16", "parts": "post+gate+scale+pre"},
        # The same for a single user's token.
        {"name": "norm_1", "op": "norm", "rows": 1, "hidden": 4096, "dtype": "bf16",
         "residual": "bf16", "parts": "post+gate+scale+pre"},
        # A training step with the residual stream in full precision.
        {"name": "norm_train", "op": "ntrain", "rows": 8192, "hidden": 4096, "dtype": "bf16",
         "residual": "f32", "parts": "post+gate+scale+pre"},
        # A small one whose rows are no whole vectors, without the gate.
        {"name": "norm_train_odd", "op": "ntrain", "rows": 1001, "hidden": 2500, "dtype": "f16",
         "residual": "f16", "parts": "post+scale+pre"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _dim(rng, lo, hi):
    """A width: mostly whole 16-byte vectors, some even ones, some odd ones."""
    step = rng.choice([64, 8, 8, 2, 1])
    return step * _log(rng, max(1, lo // step), hi // step)


PARTS = ["post+gate+scale+pre", "post+gate+pre", "post+scale+pre", "gate+scale+pre", "post+pre",
         "scale+pre", "pre", "post+gate+scale"]


def draw(rng):
    op = rng.choice(["scan", "scan", "update", "update", "train", "train", "norm", "ntrain"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "update":
        return {"op": op, "batch": _log(rng, 1, 512), "tokens": rng.choice([1, 1, 2, 3, 4, 5]),
                "dim": _dim(rng, 128, 8192), "dtype": dtype}
    if op in ("scan", "train"):
        dim = _dim(rng, 128, 8192)
        most = (1 << 26 if op == "scan" else 1 << 25) // (dim * (2 if dtype == "f32" else 1))
        tokens = _log(rng, 1, min(32768, most))
        return {"op": op, "tokens": tokens, "seqs": min(tokens, _log(rng, 1, 64)), "dim": dim,
                "dtype": dtype}
    hidden = _dim(rng, 128, 8192)
    most = (1 << 26 if op == "norm" else 1 << 25) // (hidden * (2 if dtype == "f32" else 1))
    return {"op": op, "rows": _log(rng, 1, min(16384, most)), "hidden": hidden, "dtype": dtype,
            "residual": rng.choice([dtype, "f32"]), "parts": rng.choice(PARTS)}


def _lengths(case):
    """Ragged sequence lengths that sum to the case's tokens (a property of
    the case, not of the seed)."""
    n, total = case["seqs"], case["tokens"]
    rng = random.Random(1000003 * n + total)
    w = [rng.uniform(0.25, 1.75) for _ in range(n)]
    lens = [1 + int((total - n) * x / sum(w)) for x in w]
    lens[lens.index(max(lens))] += total - sum(lens)
    return lens


def _bounds(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def n(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        x = torch.randn(*shape, generator=self.g, device=DEV, dtype=torch.float32)
        return x.mul_(std).add_(mean).to(dtype)

    def slots(self, n, lines):
        return torch.randperm(lines, generator=self.g, device=DEV)[:n].to(torch.int32)


def _lam(r, dim):
    """The usual initialisation: at an open gate a channel keeps between 0.9
    and 0.999 of its state over a token."""
    keep = 0.9 + 0.099 * torch.rand(dim, generator=r.g, device=DEV, dtype=torch.float64)
    return torch.log(torch.expm1(-torch.log(keep) / C)).float()


def prepare(case, seed):
    r, op, dt = _Rand(seed), case["op"], DTYPES[case["dtype"]]
    s = {"op": op}
    if op in ("scan", "train"):
        t, d, lens = case["tokens"], case["dim"], _lengths(case)
        ab = r.n(1, t, 2 * d, dtype=dt)
        s.update(x=r.n(1, t, d, dtype=dt), a=ab[..., :d], b=ab[..., d:], lam=_lam(r, d),
                 h0=r.n(len(lens), d),
                 cu=torch.tensor(_bounds(lens), dtype=torch.int32, device=DEV))
        if op == "train":
            s.update(dy=r.n(1, t, d, dtype=dt), dfinal=r.n(len(lens), d))
        return s
    if op == "update":
        n, t, d = case["batch"], case["tokens"], case["dim"]
        ab = r.n(n, t, 2 * d, dtype=dt)
        s.update(x=r.n(n, t, d, dtype=dt), a=ab[..., :d], b=ab[..., d:], lam=_lam(r, d),
                 pool=r.n(n * t, d), slots=r.slots(n * t, n * t), accepted=None)
        if t > 1:
            s["slots"] = s["slots"].view(n, t)
            s["accepted"] = torch.randint(1, t + 1, (n,), generator=r.g, device=DEV,
                                          dtype=torch.int32)
        return s
    m, d, parts = case["rows"], case["hidden"], case["parts"].split("+")
    rt = DTYPES[case["residual"]]
    s.update(x=r.n(m, d, dtype=dt), res=r.n(m, d, std=2.0, dtype=rt),
             post=r.n(d, std=0.1, mean=1.0, dtype=dt) if "post" in parts else None,
             gate=r.n(m, d, dtype=dt) if "gate" in parts else None,
             scale=r.n(d, std=0.1, mean=0.5, dtype=dt) if "scale" in parts else None,
             pre=r.n(d, std=0.1, mean=1.0, dtype=dt) if "pre" in parts else None)
    if op == "ntrain":
        s.update(dh=r.n(m, d, dtype=rt), dy=r.n(m, d, dtype=dt) if "pre" in parts else None)
    return s


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------
def _gates(a, b, x, lam):
    """r, i, log decay, alpha, s = sqrt(1 - alpha^2) and the input i x."""
    r, i = torch.sigmoid(a), torch.sigmoid(b)
    ell = -C * torch.log1p(torch.exp(lam)) * r
    return r, i, ell, torch.exp(ell), torch.sqrt(-torch.expm1(2 * ell)), i * x


def _doubling(alpha, add):
    """Inclusive scan of h -> alpha h + add along dim 0 from h = 0: spans of 1,
    2, 4, ... tokens are joined until they reach the start."""
    span = 1
    while span < add.size(0):
        add = torch.cat([add[:span], add[span:] + alpha[span:] * add[:-span]])
        alpha = torch.cat([alpha[:span], alpha[span:] * alpha[:-span]])
        span *= 2
    return add


def _states(alpha, add, h0, cu):
    """h_t and h_{t-1} of every token; a sequence starts from its h0."""
    first, last = cu[:-1].long(), cu[1:].long() - 1
    cut, inp = alpha.clone(), add.clone()
    cut[first] = 0
    inp[first] += alpha[first] * h0
    h = _doubling(cut, inp)
    before = torch.cat([h[:1], h[:-1]])
    before[first] = h0
    return h, before, h[last]


def _scan(s):
    x, a, b = s["x"][0].float(), s["a"][0].float(), s["b"][0].float()
    r, i, ell, alpha, g, u = _gates(a, b, x, s["lam"])
    h, _, final = _states(alpha, g * u, s["h0"], s["cu"])
    return {"y": h.to(s["x"].dtype)[None], "final": final}


def _train(s):
    dt, first, last = s["x"].dtype, s["cu"][:-1].long(), s["cu"][1:].long() - 1
    x, a, b = s["x"][0].float(), s["a"][0].float(), s["b"][0].float()
    r, i, ell, alpha, g, u = _gates(a, b, x, s["lam"])
    h, before, final = _states(alpha, g * u, s["h0"], s["cu"])
    # G_t = dy_t + alpha_{t+1} G_{t+1}, the last token's with the final state's gradient.
    dy = s["dy"][0].to(torch.float32, copy=True)
    dy[last] += s["dfinal"]
    nxt = torch.cat([alpha[1:], alpha[:1]])
    nxt[last] = 0
    big = _doubling(nxt.flip(0), dy.flip(0)).flip(0)
    dell = big * alpha * before - big * u * alpha * alpha / g
    dlam = -C * torch.sigmoid(s["lam"]) * (dell * r).sum(0)
    da = dell * ell * (1 - r)
    db = big * g * u * (1 - i)
    return {"y": h.to(dt)[None], "final": final, "dx": (big * g * i).to(dt)[None],
            "da": da.to(dt)[None], "db": db.to(dt)[None], "dlam": dlam,
            "dh0": alpha[first] * big[first]}


def _update(s):
    n, t, _ = s["x"].shape
    slots = s["slots"].view(n, t).long()
    at = torch.zeros(n, dtype=torch.long, device=DEV) if t == 1 else s["accepted"].long() - 1
    h = s["pool"][slots.gather(1, at[:, None])[:, 0]]
    r, i, ell, alpha, g, u = _gates(s["a"].float(), s["b"].float(), s["x"].float(), s["lam"])
    add = g * u
    y = torch.empty_like(s["x"])
    for k in range(t):
        h = alpha[:, k] * h + add[:, k]
        y[:, k] = h
        s["pool"][slots[:, k]] = h
    return {"y": y, "pool": s["pool"]}


def _norm_parts(s):
    x, res = s["x"].float(), s["res"].float()
    r1 = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x if s["post"] is None else x * r1 * s["post"].float()
    z = None if s["gate"] is None else s["gate"].float()
    v = n if z is None else n * z * torch.sigmoid(z)
    h = res + (v if s["scale"] is None else s["scale"].float() * v)
    r2 = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    return x, r1, n, z, v, h, r2


def _norm_out(s, h, r2):
    out = {"h": h.to(s["res"].dtype)}
    if s["pre"] is not None:
        out["y"] = (h * r2 * s["pre"].float()).to(s["x"].dtype)
    return out


def _norm(s):
    x, r1, n, z, v, h, r2 = _norm_parts(s)
    return _norm_out(s, h, r2)


def _ntrain(s):
    dt = s["x"].dtype
    x, r1, n, z, v, h, r2 = _norm_parts(s)
    out = _norm_out(s, h, r2)
    d = s["dh"].float()
    if s["pre"] is not None:
        dy, hh = s["dy"].float(), h * r2
        out["dpre"] = (dy * hh).sum(0).to(dt)
        wd = s["pre"].float() * dy
        d = d + r2 * (wd - hh * (wd * hh).mean(-1, keepdim=True))
    out["dres"] = d.to(s["res"].dtype)
    if s["scale"] is not None:
        out["dscale"] = (d * v).sum(0).to(dt)
        d = s["scale"].float() * d
    if z is not None:
        sg = torch.sigmoid(z)
        out["dgate"] = (d * n * sg * (1 + z * (1 - sg))).to(dt)
        d = d * z * sg
    if s["post"] is not None:
        xh = x * r1
        out["dpost"] = (d * xh).sum(0).to(dt)
        wd = s["post"].float() * d
        d = r1 * (wd - xh * (wd * xh).mean(-1, keepdim=True))
    out["dx"] = d.to(dt)
    return out


# --------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------
def _named(**parts):
    return {key: val for key, val in parts.items() if val is not None}


def _own_scan(s):
    from torch_npu_ops_amd import _xk_torch as xt
    y, final, _ = xt.npu_gated_linear_recurrence(s["x"], s["a"], s["b"], s["lam"], C, s["h0"],
                                                 True, s["cu"])
    return {"y": y, "final": final}


def _own_train(s):
    from torch_npu_ops_amd import _xk_torch as xt
    y, final, states = xt.npu_gated_linear_recurrence(s["x"], s["a"], s["b"], s["lam"], C,
                                                      s["h0"], True, s["cu"], True)
    dx, da, db, dlam, dh0 = xt.npu_gated_linear_recurrence_bwd(
        s["dy"], s["x"], s["a"], s["b"], s["lam"], states, C, s["h0"], s["dfinal"], s["cu"])
    return {"y": y, "final": final, "dx": dx, "da": da, "db": db, "dlam": dlam, "dh0": dh0}


def _own_update(s):
    from torch_npu_ops_amd import _xk_torch as xt
    y = xt.npu_gated_linear_recurrence_update(s["x"], s["a"], s["b"], s["lam"], s["pool"], C,
                                              s["slots"], s["accepted"])
    return {"y": y, "pool": s["pool"]}


def _own_norm(s):
    from torch_npu_ops_amd import _xk_torch as xt
    h, y, _, _ = xt.npu_gated_residual_rms_norm(s["x"], s["res"], s["post"], s["gate"],
                                                s["scale"], s["pre"], EPS)
    return _named(h=h, y=y)


def _own_ntrain(s):
    from torch_npu_ops_amd import _xk_torch as xt
    h, y, r1, r2 = xt.npu_gated_residual_rms_norm(s["x"], s["res"], s["post"], s["gate"],
                                                  s["scale"], s["pre"], EPS)
    dx, dres, dgate, dpost, dscale, dpre = xt.npu_gated_residual_rms_norm_bwd(
        s["dh"], s["dy"], s["x"], s["res"], r1, r2, s["post"], s["gate"], s["scale"], s["pre"])
    return _named(h=h, y=y, dx=dx, dres=dres, dgate=dgate, dpost=dpost, dscale=dscale, dpre=dpre)


def run(state):
    op = state["op"]
    if own:
        if op == "scan":
            return _own_scan(state)
        if op == "train":
            return _own_train(state)
        if op == "update":
            return _own_update(state)
        return _own_norm(state) if op == "norm" else _own_ntrain(state)
    if op == "scan":
        return _scan(state)
    if op == "train":
        return _train(state)
    if op == "update":
        return _update(state)
    return _norm(state) if op == "norm" else _ntrain(state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    op, e = case["op"], 4 if case["dtype"] == "f32" else 2
    if op in ("scan", "train"):
        t, d, n = case["tokens"], case["dim"], case["seqs"]
        if op == "scan":
            return {"bytes": 4 * e * t * d + 8 * n * d + 4 * d, "flops": 20 * t * d}
        return {"bytes": 8 * e * t * d + 16 * n * d + 8 * d, "flops": 65 * t * d}
    if op == "update":
        n, t, d = case["batch"], case["tokens"], case["dim"]
        return {"bytes": 4 * e * n * t * d + 4 * n * (t + 1) * d + 4 * d + 4 * n * (t + 1),
                "flops": 20 * n * t * d}
    m, d, parts = case["rows"], case["hidden"], case["parts"].split("+")
    r = 4 if case["residual"] == "f32" else 2
    gate, pre = "gate" in parts, "pre" in parts
    vectors = e * d * (len(parts) - gate)
    if op == "norm":
        return {"bytes": m * d * (e * (1 + gate + pre) + 2 * r) + vectors, "flops": 15 * m * d}
    return {"bytes": m * d * (e * (2 + 2 * gate + 2 * pre) + 4 * r) + 2 * vectors,
            "flops": 45 * m * d}


# --------------------------------------------------------------------------
# the same in 64 bits, token by token
# --------------------------------------------------------------------------
def _gates64(a, b, lam):
    """alpha, sqrt(1 - alpha^2) and the two sigmoids."""
    r, i = 1 / (1 + torch.exp(-a)), 1 / (1 + torch.exp(-b))
    keep = torch.exp(-C * torch.nn.functional.softplus(lam) * r)
    return keep, torch.sqrt((1 - keep) * (1 + keep)), r, i


def _by_length(lens):
    """Sequences from the longest to the shortest, and their first tokens."""
    at = _bounds(lens)
    order = sorted(range(len(lens)), key=lambda i: -lens[i])
    return order, torch.tensor([at[i] for i in order], device=DEV)


def _exact_scan(s, lens):
    x, a, b = s["x"][0].double(), s["a"][0].double(), s["b"][0].double()
    keep, g, r, i = _gates64(a, b, s["lam"].double())
    order, first = _by_length(lens)
    h = s["h0"].double()[order]
    y, before = torch.empty_like(x), torch.empty_like(x)
    for k in range(max(lens)):
        live = sum(1 for j in order if lens[j] > k)
        tok = first[:live] + k
        before[tok] = h[:live]
        h[:live] = keep[tok] * h[:live] + g[tok] * i[tok] * x[tok]
        y[tok] = h[:live]
    final = torch.empty_like(h)
    final[order] = h
    return x, keep, g, r, i, y, before, final


def _exact_train(s, lens):
    x, keep, g, r, i, y, before, final = _exact_scan(s, lens)
    order, first = _by_length(lens)
    dy, carry = s["dy"][0].double(), s["dfinal"].double()[order]
    big = torch.empty_like(x)
    for k in range(max(lens) - 1, -1, -1):
        live = sum(1 for j in order if lens[j] > k)
        tok = first[:live] + k
        big[tok] = dy[tok] + carry[:live]
        carry[:live] = keep[tok] * big[tok]
    dh0 = torch.empty_like(carry)
    dh0[order] = carry
    # d alpha through h_{t-1} and through g = sqrt(1 - alpha^2); alpha = exp(ell).
    dell = keep * big * (before - i * x * keep / g)
    rate = C * torch.nn.functional.softplus(s["lam"].double())
    return {"y": y[None], "final": final, "dx": (big * g * i)[None],
            "da": (-dell * rate * r * (1 - r))[None], "db": (big * g * x * i * (1 - i))[None],
            "dlam": -(dell * r).sum(0) * C * torch.sigmoid(s["lam"].double()), "dh0": dh0}


def _exact_update(s):
    n, t, _ = s["x"].shape
    slots, pool = s["slots"].view(n, t).long(), s["pool"].double()
    keep, g, r, i = _gates64(s["a"].double(), s["b"].double(), s["lam"].double())
    start = pool[slots[:, 0]]
    if t > 1:
        start = pool[slots[torch.arange(n, device=DEV), s["accepted"].long() - 1]]
    y = torch.empty_like(keep)
    for k in range(t):
        start = keep[:, k] * start + g[:, k] * i[:, k] * s["x"][:, k].double()
        y[:, k] = start
        pool[slots[:, k]] = start
    return {"y": y, "pool": pool}


def _exact_norm(s, backward):
    leaf = {key: val.double().requires_grad_(backward) for key, val in s.items()
            if torch.is_tensor(val) and key not in ("dh", "dy")}

    def rms(v):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)

    v = leaf["x"]
    if "post" in leaf:
        v = rms(v) * leaf["post"]
    if "gate" in leaf:
        v = v * leaf["gate"] / (1 + torch.exp(-leaf["gate"]))
    if "scale" in leaf:
        v = v * leaf["scale"]
    h = leaf["res"] + v
    out = {"h": h}
    loss = (h * s["dh"].double()).sum() if backward else None
    if "pre" in leaf:
        out["y"] = rms(h) * leaf["pre"]
        if backward:
            loss = loss + (out["y"] * s["dy"].double()).sum()
    if backward:
        names = list(leaf)
        out.update({"d" + key: grad for key, grad in
                    zip(names, torch.autograd.grad(loss, [leaf[k] for k in names]))})
    return {key: val.detach() for key, val in out.items()}


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "scan":
        out = _exact_scan(s, _lengths(case))
        return {"y": out[5][None], "final": out[7]}
    if op == "train":
        return _exact_train(s, _lengths(case))
    if op == "update":
        return _exact_update(s)
    return _exact_norm(s, op == "ntrain")
