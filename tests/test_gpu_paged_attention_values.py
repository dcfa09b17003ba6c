"""GPU checks of what the attention over a paged cache gives where its
arithmetic shows.  Bounds are derived from the formulas (u = 2^-24)."""
import pytest
import torch

from oracle import paged_attention as opa
from rounding_tol import assert_within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FP8 = torch.float8_e4m3fn
TYPES = [(BF16, BF16), (F16, F16), (F32, F32), (BF16, FP8), (F16, FP8)]
U = 2.0 ** -24


def _api(name):
    from torch_npu_ops_amd import _xk_torch, ops
    return {"cpp": _xk_torch, "py": ops}[name]


def _parts(x, dtype):
    """x (float64) as three values of dtype, each cut off what the ones before leave."""
    out = []
    for _ in range(3):
        step = torch.exp2(torch.frexp(x)[1].double() - (7 if dtype == BF16 else 10))
        out.append((torch.trunc(x / step) * step).to(dtype))
        x = x - out[-1].double()
    return out


def cancelling(dtype, cache, seed=0):
    """Two positions with scores 0 and s, values -a and b: in the element whose
    a / b is exp(s), up to 2^-13 of it, o = (b exp(s) - a) / (1 + exp(s)) shows
    the weight's last bits.  Rows of 64 heads, each with an element of its own;
    a < b from 8 to 15, so that a / b has all bits and 8 bits hold a and b."""
    pairs = [(a, b) for a in range(8, 16) for b in range(a + 1, 16)]
    g = torch.Generator().manual_seed(seed)
    B, hq, D = 16, 64, 64
    pair = torch.tensor([pairs[d % len(pairs)] for d in range(D)], dtype=torch.float64)
    own = torch.arange(hq)
    near = 1 + (torch.rand(B, hq, generator=g, dtype=torch.float64) - 0.5) * 2.0 ** -12
    s = torch.log(pair[own, 0] / pair[own, 1] * near)
    q = torch.zeros(B, 1, hq, D, dtype=dtype)
    for i, x in enumerate(_parts(s, dtype)):
        q[:, 0, :, i] = x
    kc, vc = torch.zeros(B, 16, 1, D), torch.zeros(B, 16, 1, D)
    kc[:, 1, 0, :3] = 1
    vc[:, 0, 0], vc[:, 1, 0] = -pair[:, 0].float(), pair[:, 1].float()
    table = torch.arange(B, dtype=torch.int32)[:, None]
    return q, kc.to(cache), vc.to(cache), table, [2] * B


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_weights_keep_their_digits(dev, dtype, cache):
    """|score| <= 1 in powers of two, off by 2 u from its sum of three, u from
    the scale's rounding, u from the product with it: 4 u, 3 u of the weight;
    its exponential 2 u; its parts in fp16 2^-21, in bf16 u; products and sums
    6 u, the division 2 u."""
    rel = (2.0 ** -21 if dtype == F16 else U if dtype == BF16 else 0.0) + 13 * U
    q, kc, vc, table, lens = cancelling(dtype, cache)
    want = opa.attention(q, kc, vc, table, lens, 1.0)["o"]
    size = opa.attention(q, kc, vc.float().abs().to(cache), table, lens, 1.0)["o"]
    n = torch.tensor(lens, dtype=torch.int32)
    for api in ("cpp", "py"):
        o, _ = _api(api).npu_paged_attention(*(t.to(dev) for t in (q, kc, vc, table, n)), 1.0)
        assert_within(o, want, size * rel, "o")


def _pool(seed, lens, page, hkv, D, dtype):
    g = torch.Generator().manual_seed(seed)
    count = [-(-n // page) for n in lens]
    order = torch.randperm(sum(count), generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max(count), dtype=torch.int32)
    at = 0
    for b, c in enumerate(count):
        table[b, :c] = order[at:at + c]
        at += c
    kc, vc = (torch.randn(at, page, hkv, D, generator=g).to(dtype) for _ in range(2))
    return kc, vc, table


# Element -> signs at positions from the sequence's end: in the last tile, which
# no draft or some see, in tiles that all see, in the first, outside a window.
INFINITIES = {3: {1: 1}, 5: {2: -1}, 7: {1: 1, 3: -1}, 11: {40: 1}, 13: {70: -1, 90: -1},
              17: {2: 1, 80: 1}, 19: {41: 1, 75: -1}, 23: {300: 1}, 31: {299: -1}}


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,G,page", [(64, 4, 16), (64, 12, 10), (128, 2, 32), (128, 8, 32),
                                      (256, 1, 16), (256, 10, 24)])
@pytest.mark.parametrize("T,window", [(1, 0), (1, 75), (4, 0), (4, 76)])
def test_infinite_values_that_a_row_sees(dev, dtype, D, G, page, T, window):
    """They make its element infinite, NaN where both signs meet; weights whose
    last bits are zeros (equal scores) and any others; no other row or element."""
    lens, hkv = [300, 131, 93], 2
    for std in (0.0, 1.0):
        kc, vc, table = _pool(D + T, lens, page, hkv, D, dtype)
        g = torch.Generator().manual_seed(7)
        q = (torch.randn(3, T, hkv * G, D, generator=g) * std).to(dtype)
        want = opa.attention(q, kc, vc, table, lens, None, window)
        plus, minus = (torch.zeros(3, T, D, dtype=torch.bool) for _ in range(2))
        for b, n in enumerate(lens):
            for e, places in INFINITIES.items():
                for back, sign in places.items():
                    j = n - back
                    if j < 0:
                        continue
                    vc[table[b, j // page], j % page, :, e] = sign * float("inf")
                    for t in range(T):
                        at = n - T + t
                        if j <= at and not (window and j <= at - window):
                            (plus if sign > 0 else minus)[b, t, e] = True
        n = torch.tensor(lens, dtype=torch.int32)
        for api in ("cpp", "py"):
            o, lse = _api(api).npu_paged_attention(*(x.to(dev) for x in (q, kc, vc, table, n)), None,
                                                   window, output_lse=True)
            o = o.cpu()
            wide = lambda m: m[:, :, None].expand(o.shape)  # noqa: E731
            assert torch.equal(o.isnan(), wide(plus & minus))
            assert torch.equal(o == float("inf"), wide(plus & ~minus))
            assert torch.equal(o == -float("inf"), wide(minus & ~plus))
            fine = o.isfinite()
            assert_within(o[fine], want["o"][fine], want["o_err"][fine], "the others")
            assert_within(lse, want["lse"], want["lse_err"], "lse")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,G", [(1, 4), (3, 8)])
def test_a_scale_that_is_nan(dev, dtype, T, G):
    """Every row of its head that sees something is NaN, with a scale of values
    but the lse; the other heads, and rows that see nothing, are as ever."""
    lens, page, hkv, D = [300, 2, 33], 16, 3, 64
    kc, vc, table = _pool(1, lens, page, hkv, D, FP8)
    q = torch.randn(3, T, hkv * G, D, generator=torch.Generator().manual_seed(2)).to(dtype)
    ks, vs = torch.tensor([0.5, float("nan"), 2.0]), torch.tensor([1.0, 0.5, 2.0])
    want = opa.attention(q, kc, vc, table, lens, None, 0, ks.nan_to_num(1.0), vs)
    n = torch.tensor(lens, dtype=torch.int32)
    for api in ("cpp", "py"):
        o, lse = _api(api).npu_paged_attention(
            *(x.to(dev) for x in (q, kc, vc, table, n)), None, 0, ks.to(dev), vs.to(dev), True)
        o, lse = o.cpu(), lse.cpu()
        there = want["lse"].isfinite()
        bad = there.clone()
        bad[:, :, :G], bad[:, :, 2 * G:] = False, False
        assert bad.any() and (T == 1 or not there.all())
        assert o[bad].isnan().all() and lse[bad].isnan().all()
        assert_within(o[~bad], want["o"][~bad], want["o_err"][~bad], "o")
        assert_within(lse[~bad], want["lse"][~bad], want["lse_err"][~bad], "lse")
        o, lse = (x.cpu() for x in _api(api).npu_paged_attention(
            *(x.to(dev) for x in (q, kc, vc, table, n)), None, 0, ks.nan_to_num(1.0).to(dev),
            (vs * (ks / ks)).to(dev), True))
        assert o[bad].isnan().all()
        assert_within(o[~bad], want["o"][~bad], want["o_err"][~bad], "o")
        assert_within(lse, want["lse"], want["lse_err"], "lse")


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("T,G", [(1, 4), (3, 8)])
def test_a_scale_of_zero(dev, dtype, cache, T, G):
    """The mean of the values seen, however large the scores would be; NaN
    where a query or a key that a row sees is not finite (0 * inf)."""
    lens, page, hkv, D = [300, 2, 33], 16, 2, 64
    kc, vc, table = _pool(3, lens, page, hkv, D, cache)
    q = torch.randn(3, T, hkv * G, D, generator=torch.Generator().manual_seed(4)).to(dtype)
    if cache != FP8:  # products beyond fp32 in bf16 and fp32
        kc, q = kc * (1e4 if dtype == F16 else 9e18), q * (1e4 if dtype == F16 else 9e18)
    ks = torch.tensor([0.0, -0.0]) if cache == FP8 else None
    scale = 1.0 if cache == FP8 else 0.0
    want = opa.attention(q, torch.zeros_like(kc), vc, table, lens, 0.0)
    n = torch.tensor(lens, dtype=torch.int32)
    on = lambda x: None if x is None else x.to(dev)  # noqa: E731
    for api in ("cpp", "py"):
        args = [kc, vc, table, n, scale, 0, ks, None, True]
        call = lambda q, *a: _api(api).npu_paged_attention(  # noqa: E731
            q.to(dev), *(on(x) if torch.is_tensor(x) else x for x in a))
        o, lse = call(q, *args)
        assert_within(o, want["o"], want["o_err"], "o")
        assert_within(lse, want["lse"], want["lse_err"], "lse")
        bad = q.clone()
        bad[0, 0, 1, 5], bad[1, T - 1, 2, 7] = float("inf"), float("nan")
        o, lse = (x.cpu() for x in call(bad, *args))
        hit = torch.zeros(o.shape[:3], dtype=torch.bool)
        hit[0, 0, 1] = hit[1, T - 1, 2] = True
        assert o[hit].isnan().all() and lse[hit].isnan().all()
        assert_within(o[~hit], want["o"][~hit], want["o_err"][~hit], "the other rows")
        keys = kc.clone()
        keys[table[2, (33 - 2) // page], (33 - 2) % page, 1, 9] = float("nan" if cache == FP8 else "-inf")
        o, lse = (x.cpu() for x in call(q, keys, *args[1:]))
        hit = torch.zeros(o.shape[:3], dtype=torch.bool)
        hit[2, max(0, T - 2):, G:] = True
        assert o[hit].isnan().all() and lse[hit].isnan().all()
        assert_within(o[~hit], want["o"][~hit], want["o_err"][~hit], "rows that do not see the key")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,G", [(1, 4), (3, 8)])
def test_scores_that_are_not_finite(dev, dtype, T, G):
    """NaN and inf make a row NaN; a score of -inf has no weight, and a row of
    such alone is 0 with an lse of -inf.  Rows before them are as ever."""
    lens, page, hkv, D = [300, 90, 40], 16, 2, 64
    kc, vc, table = _pool(5, lens, page, hkv, D, dtype)
    q = torch.randn(3, T, hkv * G, D, generator=torch.Generator().manual_seed(6)).to(dtype)
    q[..., 3] = q[..., 3].abs() + 0.5
    n = torch.tensor(lens, dtype=torch.int32)

    def call(api, keys):
        o, lse = _api(api).npu_paged_attention(*(x.to(dev) for x in (q, keys, vc, table, n)),
                                               output_lse=True)
        return o.cpu(), lse.cpu()

    def put(keys, b, j, head, x):
        keys[table[b, j // page], j % page, head, 3] = x
    inf = float("inf")
    for api in ("cpp", "py"):
        for bad in (float("nan"), inf):
            for j in (lens[0] - 1, 7):  # one that the last token sees, one that all do
                keys = kc.clone()
                put(keys, 0, j, 1, bad)
                want = opa.attention(q, kc, vc, table, lens)
                o, lse = call(api, keys)
                hit = torch.zeros(lse.shape, dtype=torch.bool)
                hit[0, T - 1 if j > 7 else 0:, G:] = True
                assert o[hit].isnan().all() and lse[hit].isnan().all()
                assert_within(o[~hit], want["o"][~hit], want["o_err"][~hit], "o")
                assert_within(lse[~hit], want["lse"][~hit], want["lse_err"][~hit], "lse")
        # without weight: as if the page were not there
        keys, without = kc.clone(), table.clone()
        for j in range(32, 48):
            put(keys, 1, j, slice(None), -inf)
        without[1, 2] = -1
        for j in range(lens[2]):
            put(keys, 2, j, slice(None), -inf)
        without[2] = -1
        want = opa.attention(q, kc, vc, without, lens)
        o, lse = call(api, keys)
        assert (o[2] == 0).all() and (lse[2] == -inf).all()
        assert_within(o, want["o"], want["o_err"], "o")
        assert_within(lse, want["lse"], want["lse_err"], "lse")
