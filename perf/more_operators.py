"""Rotary positions, the paged key-value cache and the attention of new tokens
over it, as cases that can be timed and checked: the plain form of each
operator (elementary torch operations in fp32, the angles in 64 bits, rounded
once), the framework's call, and the same in 64 bits.

Families (the "op" of a case):

  rotary  q and k turned by their positions: pairs (i, i + r/2) or (2i, 2i + 1)
          of the first r elements of a head, the frequencies and the length of
          the turned vectors scaled where the context is longer than trained
  rtrain  the same, and its backward pass: gradients of q and k
  append  q and k turned, k and v written to their slots of a paged cache (in
          the tokens' type, or in 8 bits with a scale for each head)
  attend  one new token of every sequence, or a few drafted ones, over the
          sequence's pages: softmax(scale q k) v with the new tokens at the
          sequence's end, over all positions or a window

q, k and v come as one wide row, as one product leaves them.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0


def listed():
    return [
        # Training or a prefill without a cache: a full batch, the whole head turned.
        {"name": "rotary_prefill", "op": "rotary", "tokens": 16384, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "pairs": "half", "factor": 1, "dtype": "bf16"},
        # A training step at a long context: a quarter of a wide head turned, frequencies
        # scaled 32 times, in full precision.
        {"name": "rotary_train_long", "op": "rtrain", "tokens": 4096, "q_heads": 16, "kv_heads": 2,
         "dim": 256, "rot": 64, "pairs": "half", "factor": 32, "dtype": "f32"},
        # A small one with neighbours as pairs and heads that are no power of two.
        {"name": "rotary_train_odd", "op": "rtrain", "tokens": 1001, "q_heads": 5, "kv_heads": 1,
         "dim": 80, "rot": 80, "pairs": "next", "factor": 1, "dtype": "f16"},
        # Prefill: 6 ragged prompts enter the cache.
        {"name": "append_prefill", "op": "append", "tokens": 8192, "seqs": 6, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "pairs": "half", "factor": 1, "page": 128,
         "dtype": "bf16", "cache": "same"},
        # A single user's token: the smallest call, all latency.
        {"name": "append_1", "op": "append", "tokens": 1, "seqs": 1, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "pairs": "half", "factor": 1, "page": 128, "dtype": "bf16",
         "cache": "same"},
        # A full decode batch: wide heads, a quarter of them turned, an 8-bit cache.
        {"name": "append_256_fp8", "op": "append", "tokens": 256, "seqs": 256, "q_heads": 16,
         "kv_heads": 2, "dim": 256, "rot": 64, "pairs": "half", "factor": 1, "page": 128,
         "dtype": "bf16", "cache": "fp8"},
        # A single user's token at a short context: latency.
        {"name": "attend_1", "op": "attend", "seqs": 1, "tokens": 1, "context": 900,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "window": 0, "dtype": "bf16",
         "cache": "same", "lse": False},
        # A single user's token at a long context, with what joins it to other parts.
        {"name": "attend_long", "op": "attend", "seqs": 1, "tokens": 1, "context": 131072,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "window": 0, "dtype": "bf16",
         "cache": "same", "lse": True},
        # A full decode batch of ragged contexts.
        {"name": "attend_64", "op": "attend", "seqs": 64, "tokens": 1, "context": 4096,
         "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "dtype": "bf16",
         "cache": "same", "lse": False},
        # A larger one of wide heads on an 8-bit cache.
        {"name": "attend_128_fp8", "op": "attend", "seqs": 128, "tokens": 1, "context": 2500,
         "q_heads": 16, "kv_heads": 2, "dim": 256, "page": 128, "window": 0, "dtype": "bf16",
         "cache": "fp8", "lse": False},
        # Speculative decoding (3 drafts and the last accepted token) in a layer with a window.
        {"name": "attend_verify", "op": "attend", "seqs": 48, "tokens": 4, "context": 6000,
         "q_heads": 32, "kv_heads": 4, "dim": 64, "page": 32, "window": 2048, "dtype": "f16",
         "cache": "same", "lse": False},
        # A small ragged batch in full precision, heads and pages that are no powers of two.
        {"name": "attend_f32", "op": "attend", "seqs": 7, "tokens": 1, "context": 1777,
         "q_heads": 15, "kv_heads": 5, "dim": 80, "page": 24, "window": 0, "dtype": "f32",
         "cache": "same", "lse": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 8, rng.randint(1, 10)])
    group = rng.choice([1, 2, 4, 4, 8, rng.randint(1, 16)])
    return min(64, kv * group) // kv * kv, kv


def draw(rng):
    op = rng.choice(["rotary", "rtrain", "append", "append", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    wide = 2 if dtype == "f32" else 1
    q_heads, kv_heads = _heads(rng)
    if op == "attend":
        dim = rng.choice([64, 128, 128, 256, 8 * rng.randint(4, 32)])
        seqs = _log(rng, 1, 256)
        most = (1 << 28) // (wide * seqs * kv_heads * dim)
        context = _log(rng, 1, max(1, min(131072, most)))
        return {"op": op, "seqs": seqs, "tokens": rng.choice([1, 1, 1, 2, 3, 4, 6]),
                "context": context, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([16, 32, 64, 128, 128, rng.randint(1, 100)]),
                "window": rng.choice([0, 0, 0, _log(rng, 1, 8192)]), "dtype": dtype,
                "cache": rng.choice(["same", "same", "fp8"]) if dtype != "f32" else "same",
                "lse": rng.random() < 0.3}
    if rng.random() < 0.8:
        dim = rng.choice([64, 128, 128, 256, 8 * rng.randint(4, 32)])
        rot = rng.choice([dim, dim, dim // 2, dim // 4])
    else:
        dim = rng.randint(20, 256)
        rot = dim
    rot -= rot % 2
    row = (q_heads + 2 * kv_heads) * dim
    most = (1 << 26) // ((2 if op == "rtrain" else 1) * wide * row)
    tokens = _log(rng, 1, min(16384, most))
    case = {"op": op, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "rot": rot, "pairs": rng.choice(["half", "half", "next"]),
            "factor": rng.choice([1, 1, 4, 32]), "dtype": dtype}
    if op == "append":
        fp8 = dtype != "f32" and rng.random() < 0.3
        case.update(seqs=tokens if rng.random() < 0.4 and tokens <= 512 else _log(rng, 1, min(64, tokens)),
                    page=rng.choice([16, 32, 128, 128, rng.randint(1, 100)]),
                    cache="fp8" if fp8 else "same")
    return case


def _lengths(case):
    """Ragged lengths (a property of the case, not of the seed): shares of the
    tokens that sum to them, or contexts spread around the case's."""
    n = case["seqs"]
    if case["op"] == "attend":
        rng = random.Random(1000003 * n + case["context"])
        if n == 1:
            return [max(case["tokens"], case["context"])]
        return [max(case["tokens"], int(case["context"] * rng.uniform(0.25, 1.75)))
                for _ in range(n)]
    total = case["tokens"]
    rng = random.Random(1000003 * n + total)
    w = [rng.uniform(0.25, 1.75) for _ in range(n)]
    lens = [1 + int((total - n) * x / sum(w)) for x in w]
    lens[lens.index(max(lens))] += total - sum(lens)
    return lens


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def n(self, *shape, std=1.0, dtype=torch.float32):
        x = torch.randn(*shape, generator=self.g, device=DEV, dtype=torch.float32)
        return x.mul_(std).to(dtype)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)


def _frequencies(rot, factor):
    """1e6^(-2i / rot) in turns of 2 pi a token; with a factor, frequencies
    that turn less than once in the trained context are divided by it, those
    that turn more than 32 times are kept, those between are blended, and the
    turned vectors are a little longer (1 + ln(factor) / 10)."""
    f = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if factor == 1:
        return f.float().to(DEV), 1.0
    turns = 32768 * f / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return (f * keep + f / factor * (1 - keep)).float().to(DEV), 1 + 0.1 * math.log(factor)


def _qkv(r, case, dtype):
    t, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
    row = r.n(t, (hq + 2 * hkv) * d, dtype=dtype)
    parts = row.split([hq * d, hkv * d, hkv * d], dim=1)
    return [p.unflatten(1, (h, d)) for p, h in zip(parts, (hq, hkv, hkv))]


def _kv_scales(r, heads):
    """What a calibration leaves: the largest value of a head over 448."""
    return [(0.8 + 0.4 * torch.rand(heads, generator=r.g, device=DEV)) * 6.0 / FP8_MAX
            for _ in range(2)]


def prepare(case, seed):
    r, op, dt = _Rand(seed), case["op"], DTYPES[case["dtype"]]
    s = {"op": op}
    if op == "attend":
        n, t, hkv, d, page = (case[k] for k in ("seqs", "tokens", "kv_heads", "dim", "page"))
        lens = _lengths(case)
        count = [-(-length // page) for length in lens]
        width, pages = max(count), sum(count)
        # Every sequence's pages lie anywhere in the pool.
        own_pages = torch.zeros(n, width, dtype=torch.int32, device=DEV)
        used = torch.arange(width, device=DEV)[None] < torch.tensor(count, device=DEV)[:, None]
        own_pages[used] = r.perm(pages).to(torch.int32)
        s.update(q=r.n(n, t, case["q_heads"], d, std=1.5, dtype=dt), table=own_pages,
                 lens=torch.tensor(lens, dtype=torch.int32, device=DEV), longest=max(lens),
                 window=case["window"], lse=case["lse"], ks=None, vs=None)
        if case["cache"] == "fp8":
            s["ks"], s["vs"] = _kv_scales(r, hkv)
        for name in ("kc", "vc"):
            pool = torch.empty(pages, page, hkv, d, device=DEV,
                               dtype=FP8 if case["cache"] == "fp8" else dt)
            step = max(1, (1 << 27) // (page * hkv * d))
            for at in range(0, pages, step):
                part = pool[at:at + step]
                x = r.n(*part.shape)
                if case["cache"] == "fp8":
                    scale = s["ks" if name == "kc" else "vs"][:, None]
                    x = (x / scale).clamp(-FP8_MAX, FP8_MAX)
                part.copy_(x)
            s[name] = pool
        return s
    t = case["tokens"]
    s["q"], s["k"], s["v"] = _qkv(r, case, dt)
    s["freq"], s["long"] = _frequencies(case["rot"], case["factor"])
    s["next"] = case["pairs"] == "next"
    reach = 32768 * case["factor"]
    if op != "append":
        start = torch.randint(0, reach, (1,), generator=r.g, device=DEV)
        s["pos"] = (start + torch.arange(t, device=DEV)) % reach
        if op == "rtrain":
            s.update(dq=r.n(*s["q"].shape, dtype=dt), dk=r.n(*s["k"].shape, dtype=dt))
        return s
    page, lens = case["page"], _lengths(case)
    host = random.Random(seed)
    begin = [host.randrange(reach) for _ in lens]
    count = [-(-(page - 1 + length) // page) for length in lens]  # wherever it begins in a page
    pages = sum(count)
    perm = r.perm(pages)
    reps = torch.tensor(lens, device=DEV)
    b = torch.tensor(begin, device=DEV).repeat_interleave(reps)
    first = torch.tensor([sum(lens[:i]) for i in range(len(lens))], device=DEV)
    base = torch.tensor([sum(count[:i]) for i in range(len(lens))], device=DEV)
    local = torch.arange(t, device=DEV) - first.repeat_interleave(reps)
    at = b % page + local
    s["pos"] = b + local
    s["slots"] = perm[base.repeat_interleave(reps) + at // page] * page + at % page
    hkv, d = case["kv_heads"], case["dim"]
    s["ks"], s["vs"] = _kv_scales(r, hkv) if case["cache"] == "fp8" else (None, None)
    for name in ("kc", "vc"):
        s[name] = torch.zeros(pages, page, hkv, d, device=DEV,
                              dtype=FP8 if case["cache"] == "fp8" else dt)
    return s


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------
def _cos_sin(s):
    angle = s["pos"].double()[:, None] * s["freq"].double()
    return ((torch.cos(angle) * s["long"]).float()[:, None],
            (torch.sin(angle) * s["long"]).float()[:, None])


def _turn(x, cos, sin, neighbours):
    """The first 2 * cos.size(-1) elements of x's heads turned, in fp32."""
    half = cos.size(-1)
    x = x.float()
    if neighbours:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        a, b = x[..., :half], x[..., half:2 * half]
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if neighbours else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _rotary(s):
    cos, sin = _cos_sin(s)
    dt = s["q"].dtype
    return {"q": _turn(s["q"], cos, sin, s["next"]).to(dt),
            "k": _turn(s["k"], cos, sin, s["next"]).to(dt)}


def _rtrain(s):
    cos, sin = _cos_sin(s)
    dt = s["q"].dtype
    return {"q": _turn(s["q"], cos, sin, s["next"]).to(dt),
            "k": _turn(s["k"], cos, sin, s["next"]).to(dt),
            "dq": _turn(s["dq"], cos, -sin, s["next"]).to(dt),
            "dk": _turn(s["dk"], cos, -sin, s["next"]).to(dt)}


def _stored(x, scale, dtype):
    if scale is None:
        return x.to(dtype)
    return (x / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(dtype)


def _append(s):
    cos, sin = _cos_sin(s)
    k = _stored(_turn(s["k"], cos, sin, s["next"]), s["ks"], s["kc"].dtype)
    v = _stored(s["v"].float(), s["vs"], s["vc"].dtype)
    for pool, rows in ((s["kc"], k), (s["vc"], v)):
        if pool.dtype == FP8:  # no indexed copy of 8-bit floats: their bytes
            pool, rows = pool.view(torch.uint8), rows.view(torch.uint8)
        pool.flatten(0, 1)[s["slots"]] = rows
    return _cached(s, _turn(s["q"], cos, sin, s["next"]).to(s["q"].dtype))


def _cached(s, q):
    """Both caches whole; what is held in 8 bits as the numbers it stands for
    in a wider type (before the head's scale)."""
    if s["ks"] is None:
        return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}
    return {"q": q, "k_cache": s["kc"].to(q.dtype), "v_cache": s["vc"].to(q.dtype)}


def _attend(s):
    q, table, page = s["q"], s["table"], s["kc"].size(1)
    n, t, hq, d = q.shape
    hkv, longest = s["kc"].size(2), s["longest"]
    table = table[:, :-(-longest // page)].long()
    k = s["kc"][table].float().flatten(1, 2)[:, :longest].permute(0, 2, 3, 1).contiguous()
    v = s["vc"][table].float().flatten(1, 2)[:, :longest].permute(0, 2, 1, 3).contiguous()
    qq = q.float().view(n, t, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d)
    if s["ks"] is not None:
        qq = qq * s["ks"][:, None, None]
    score = torch.matmul(qq, k) / math.sqrt(d)
    at = torch.arange(longest, device=DEV)
    last = s["lens"][:, None] - t + torch.arange(t, device=DEV)  # a token's own position
    seen = at <= last[..., None]
    if s["window"]:
        seen &= at > last[..., None] - s["window"]
    seen = seen[:, None, :, None].expand(n, hkv, t, hq // hkv, longest).reshape(score.shape)
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / total
    if s["vs"] is not None:
        o = o * s["vs"][:, None, None]
    o = o.view(n, hkv, t, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(q.shape)
    if not s["lse"]:
        return {"o": o.to(q.dtype)}
    lse = (top + torch.log(total)).view(n, hkv, t, hq // hkv).permute(0, 2, 1, 3)
    return {"o": o.to(q.dtype), "lse": lse.reshape(n, t, hq)}


# --------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------
def _own_rotary(s):
    from torch_npu_ops_amd import _xk_torch as xt
    q, k = xt.npu_rotary_embedding(s["q"], s["k"], s["pos"], s["freq"], s["next"], s["long"])
    return {"q": q, "k": k}


def _own_rtrain(s):
    from torch_npu_ops_amd import _xk_torch as xt
    q, k = xt.npu_rotary_embedding(s["q"], s["k"], s["pos"], s["freq"], s["next"], s["long"])
    dq, dk = xt.npu_rotary_embedding_bwd(s["dq"], s["dk"], s["pos"], s["freq"], s["next"],
                                         s["long"])
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _own_append(s):
    from torch_npu_ops_amd import _xk_torch as xt
    q = xt.npu_rotary_cache_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"],
                                   s["pos"], s["freq"], s["next"], s["long"], s["ks"], s["vs"])
    return _cached(s, q)


def _own_attend(s):
    from torch_npu_ops_amd import _xk_torch as xt
    o, lse = xt.npu_paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], None,
                                    s["window"], s["ks"], s["vs"], s["lse"])
    return {"o": o, "lse": lse} if s["lse"] else {"o": o}


def run(state):
    op = state["op"]
    if own:
        if op == "rotary":
            return _own_rotary(state)
        if op == "rtrain":
            return _own_rtrain(state)
        return _own_append(state) if op == "append" else _own_attend(state)
    if op == "rotary":
        return _rotary(state)
    if op == "rtrain":
        return _rtrain(state)
    return _append(state) if op == "append" else _attend(state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    t, hq, hkv, d = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        c = 1 if case["cache"] == "fp8" else e
        lens, n = _lengths(case), case["seqs"]
        w = case["window"] or 1 << 40
        read = sum(min(length, w + t - 1) for length in lens)  # positions that some token sees
        seen = sum(min(length - t + 1 + j, w) for length in lens for j in range(t))
        pages = sum(-(-length // case["page"]) for length in lens)
        out = 2 * e * n * t * hq * d + (4 * n * t * hq if case["lse"] else 0)
        return {"bytes": 2 * c * read * hkv * d + out + 4 * pages + 4 * n,
                "flops": 4 * seen * hq * d}
    turned = t * (hq + hkv)
    flops = turned * (3 * case["rot"])
    if case["op"] == "append":
        c = 1 if case["cache"] == "fp8" else e
        return {"bytes": t * d * (2 * e * hq + 2 * (e + c) * hkv) + 16 * t, "flops": flops}
    passes = 2 if case["op"] == "rtrain" else 1
    return {"bytes": passes * (2 * e * turned * d + 8 * t), "flops": passes * flops}


# --------------------------------------------------------------------------
# the same in 64 bits
# --------------------------------------------------------------------------
def _exact_turn(x, s, back=False):
    """As a product with a complex number of length s["long"] for each pair."""
    r = 2 * s["freq"].numel()
    angle = torch.outer(s["pos"].double(), s["freq"].double())
    by = torch.polar(torch.full_like(angle, s["long"]), -angle if back else angle)[:, None]
    x = x.double().clone()
    if s["next"]:
        z = torch.view_as_complex(x[..., :r].unflatten(-1, (r // 2, 2)).contiguous()) * by
        x[..., :r] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * by
        x[..., :r // 2], x[..., r // 2:r] = z.real, z.imag
    return x


def _exact_append(s):
    out = {"q": _exact_turn(s["q"], s)}
    for name, pool, rows, scale in (("k_cache", s["kc"], _exact_turn(s["k"], s), s["ks"]),
                                    ("v_cache", s["vc"], s["v"].double(), s["vs"])):
        whole = pool.double().flatten(0, 1)
        if scale is not None:  # 4 significant bits, steps of 2^-9 at the least
            rows = (rows / scale.double()[:, None]).clamp(-FP8_MAX, FP8_MAX)
            step = torch.exp2(torch.frexp(rows)[1].double() - 4).clamp_min(2.0 ** -9)
            rows = torch.round(rows / step) * step
        whole[s["slots"]] = rows
        out[name] = whole.view(pool.shape)
    return out


def _exact_attend(s):
    q, page = s["q"].double(), s["kc"].size(1)
    n, t, hq, d = q.shape
    group = hq // s["kc"].size(2)
    o, lse = torch.empty_like(q), torch.empty(n, t, hq, dtype=torch.float64, device=DEV)
    for i, length in enumerate(s["lens"].tolist()):
        pages = s["table"][i, :-(-length // page)].long()
        k = s["kc"][pages].flatten(0, 1)[:length].double()
        v = s["vc"][pages].flatten(0, 1)[:length].double()
        if s["ks"] is not None:
            k, v = k * s["ks"].double()[:, None], v * s["vs"].double()[:, None]
        for j in range(t):
            end = length - t + 1 + j
            begin = max(0, end - s["window"]) if s["window"] else 0
            for h in range(hq):
                score = (k[begin:end, h // group] @ q[i, j, h]) / math.sqrt(d)
                lse[i, j, h] = torch.logsumexp(score, 0)
                o[i, j, h] = torch.softmax(score, 0) @ v[begin:end, h // group]
    return {"o": o, "lse": lse} if s["lse"] else {"o": o}


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "attend":
        return _exact_attend(s)
    if op == "append":
        return _exact_append(s)
    out = {"q": _exact_turn(s["q"], s), "k": _exact_turn(s["k"], s)}
    if op == "rtrain":
        out.update(dq=_exact_turn(s["dq"], s, True), dk=_exact_turn(s["dk"], s, True))
    return out
