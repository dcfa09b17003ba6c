"""GPU checks of rotary positions and the write into the paged cache against
oracle/rotary.py in float64.  Tolerances: the oracle's bound of the arithmetic
plus half a step of the output's type (rounding_tol.py)."""
import pytest
import torch

from oracle import rotary
from rounding_tol import assert_within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FP8 = torch.float8_e4m3fn


def _api(name):
    from torch_npu_ops_amd import _xk_torch, ops
    return {"cpp": _xk_torch, "py": ops}[name]


def _freq(rot, base=1e4):
    return (base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float()


def _qkv(seed, T, hq, hkv, D, dtype):
    g = torch.Generator().manual_seed(seed)
    row = torch.randn(T, (hq + 2 * hkv) * D, generator=g).to(dtype)
    return [p.unflatten(1, (h, D)) for p, h in
            zip(row.split([hq * D, hkv * D, hkv * D], 1), (hq, hkv, hkv))]


def _same_view(x, dev):
    """x on the device with x's strides."""
    base = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=dev)
    return base.copy_(x.to(dev))


# head length, turned part: whole and odd vectors, single units, no vectors
SHAPES = [(128, 128), (256, 64), (64, 32), (80, 80), (16, 16), (8, 4), (100, 50), (37, 36), (2, 2),
          (512, 512), (192, 64)]


@pytest.mark.parametrize("D,rot", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rotary_and_its_gradients(dev, D, rot, interleaved, dtype):
    if rot % 2:
        pytest.skip("pairs")
    api = _api("cpp" if interleaved else "py")
    for T, hq, hk in ((1, 3, 1), (29, 5, 2)):
        print(f"rotary T={T} heads={hq}/{hk} D={D} rot={rot}", flush=True)
        q, k, _ = _qkv(T, T, hq, hk, D, dtype)
        pos = torch.randint(0, 1 << 20, (T,), generator=torch.Generator().manual_seed(D))
        f = _freq(rot)
        args = (pos.to(dev), f.to(dev), interleaved, 1.125)
        for fn, back in ((api.npu_rotary_embedding, False), (api.npu_rotary_embedding_bwd, True)):
            got = fn(q.to(dev), k.to(dev), *args)
            for x, y, name in zip((q, k), got, "qk"):
                want, err = rotary.turn(x, pos, f, interleaved, 1.125, back)
                assert y.is_contiguous() and y.dtype == dtype
                assert_within(y, want, err, f"{name} back={back}")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_gradient_is_that_of_differences(dev, dtype):
    """<dy, R(x + e) - R(x - e)> / 2 = <R'dy, e>: the map is linear, so that
    differences of any size say it; sums in 64 bits of the kernel's outputs."""
    api = _api("cpp")
    T, H, D = 5, 2, 64
    g = torch.Generator().manual_seed(0)
    x, e, dy = (torch.randn(T, H, D, generator=g).to(dtype) for _ in range(3))
    pos, f = torch.arange(T) * 1000, _freq(D)
    args = (pos.to(dev), f.to(dev), False, 1.0)
    turn = lambda v: api.npu_rotary_embedding(v.to(dev), None, *args)[0].cpu().double()  # noqa: E731
    up, down = (x + e), (x - e)
    lhs = (dy.double() * (turn(up) - turn(down))).sum() / 2
    back = api.npu_rotary_embedding_bwd(dy.to(dev), None, *args)[0].cpu().double()
    rhs = (back * (up.double() - down.double())).sum() / 2
    # each output of up to 8 is off by half a step: sums of |dy| and |up - down| times that
    room = torch.finfo(dtype).eps / 2 * 8 * (dy.double().abs().sum()
                                             + (up.double() - down.double()).abs().sum() / 2)
    assert (lhs - rhs).abs() <= room


@pytest.mark.parametrize("ptype", [torch.int32, torch.int64])
def test_far_and_negative_positions(dev, ptype):
    pos = torch.tensor([0, 1, -1, 131071, 10 ** 7, (1 << 29) - 1, -(1 << 29)], dtype=ptype)
    f = torch.cat([_freq(62), torch.tensor([1.0])])
    x = torch.randn(7, 2, 64, generator=torch.Generator().manual_seed(1))
    for api in ("cpp", "py"):
        y, none = _api(api).npu_rotary_embedding(x.to(dev), None, pos.to(dev), f.to(dev))
        assert none is None
        want, err = rotary.turn(x, pos, f)
        assert_within(y, want, err, "far")


def test_views_broadcast_and_leading_dims(dev):
    f = _freq(64).to(dev)
    g = torch.Generator().manual_seed(2)
    base = torch.randn(3, 4, 6, 64, generator=g).bfloat16()
    pos = torch.randint(0, 5000, (3, 4), generator=g)
    for x in (base, base.transpose(0, 1).contiguous().transpose(0, 1), base[:, :1].expand(3, 4, 6, 64),
              base[..., :1, :].expand(3, 4, 6, 64), base.transpose(1, 2).contiguous().transpose(1, 2)):
        for api in ("cpp", "py"):
            y, k = _api(api).npu_rotary_embedding(_same_view(x, dev) if 0 not in x.stride() else
                                                  x.to(dev), x.to(dev)[..., :2, :], pos.to(dev), f)
            want, err = rotary.turn(x, pos, f.cpu())
            assert_within(y, want, err, "view")
            assert_within(k, want[..., :2, :], err[..., :2, :], "view k")
    # element offset 1: no aligned vectors; a head dimension that is not dense
    wide = torch.randn(5, 2, 67, generator=g).bfloat16()
    for x in (wide[..., 1:65], torch.randn(5, 2, 64, 2, generator=g).bfloat16()[..., 0]):
        p5 = torch.arange(5)
        want, err = rotary.turn(x, p5, f.cpu())
        for api in ("cpp", "py"):
            y, _ = _api(api).npu_rotary_embedding(_same_view(x, dev), None, p5.to(dev), f)
            assert_within(y, want, err, "unaligned")


def test_in_place_and_empty_calls(dev):
    from torch_npu_ops_amd import _lib
    lib = _lib.lib()
    for D, dtype, dt in ((128, BF16, _lib.XK_BF16), (37, F32, _lib.XK_F32)):
        for inter in (0, 1):
            x = torch.randn(700, 3, D, generator=torch.Generator().manual_seed(3)).to(dtype)
            pos, f = torch.arange(700) * 3, _freq(36)
            d, p, fd = x.to(dev), pos.to(dev), f.to(dev)
            st = lib.xk_rotary_embedding(
                d.data_ptr(), 3 * D, D, d.data_ptr(), 3 * D, D, 3, None, 0, 0, None, 0, 0, 0,
                p.data_ptr(), _lib.XK_I64, fd.data_ptr(), 36, inter, 1.0, 0, 700, D, dt,
                torch.cuda.current_stream().cuda_stream)
            assert st == 0
            want, err = rotary.turn(x, pos, f, bool(inter))
            assert_within(d, want, err, "in place")
    for api in ("cpp", "py"):
        q, k = _api(api).npu_rotary_embedding(torch.zeros(0, 4, 64, device=dev),
                                              torch.zeros(0, 2, 64, device=dev),
                                              torch.zeros(0, dtype=torch.int64, device=dev),
                                              _freq(64).to(dev))
        assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)


def test_nan_and_inf_stay_in_their_pair(dev):
    x = torch.zeros(1, 1, 16)
    x[0, 0, 3], x[0, 0, 14] = float("nan"), float("inf")
    y, _ = _api("cpp").npu_rotary_embedding(x.to(dev), None, torch.ones(1, dtype=torch.int64).to(dev),
                                            _freq(8).to(dev))
    y = y.cpu()[0, 0]
    assert y[[3, 7]].isnan().all() and y[14] == float("inf")
    assert y[[0, 1, 2, 4, 5, 6, 8, 9, 10, 11, 12, 13, 15]].eq(0).all()


# --------------------------------------------------------------------------
# the paged cache
# --------------------------------------------------------------------------
def _check_append(dev, api, q, k, v, kc, vc, slots, pos, f, interleaved=False, scale=1.0, ks=None,
                  vs=None):
    """kc, vc: CPU caches (with their strides); slots may lie outside."""
    dk, dv = _same_view(kc, dev), _same_view(vc, dev)
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = api.npu_rotary_cache_append(on(q), on(k), on(v), dk, dv, on(slots), on(pos), on(f),
                                      interleaved, scale, on(ks), on(vs))
    turn = (lambda x: rotary.turn(x, pos, f, interleaved, scale)) if pos is not None else \
        (lambda x: (x.double(), torch.zeros(x.shape, dtype=torch.float64)))  # noqa: E731
    if q is None:
        assert got is None
    else:
        assert_within(got, *turn(q), "q")
    flat = lambda x: x.reshape(-1, *x.shape[-2:])  # noqa: E731
    yk, ek = turn(k)
    want, err = rotary.append(kc, flat(yk), flat(ek), slots.reshape(-1), ks)
    assert_within(dk, want, err, "k_cache")
    want, err = rotary.append(vc, flat(v.double()), torch.zeros_like(flat(v.double())),
                              slots.reshape(-1), vs)
    assert_within(dv, want, err, "v_cache")
    return dk, dv


def _slots(seed, T, places, dtype=torch.int64):
    return torch.randperm(places, generator=torch.Generator().manual_seed(seed))[:T].to(dtype)


@pytest.mark.parametrize("D,rot,page", [(128, 128, 16), (256, 64, 128), (80, 80, 24), (44, 44, 7),
                                        (37, 36, 1), (64, 16, 3)])
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, FP8),
                                         (F16, FP8)])
def test_append(dev, D, rot, page, dtype, cache):
    api = _api("py" if page == 16 else "cpp")
    for T, hq, hkv in ((1, 4, 1), (37, 6, 2)):
        print(f"append T={T} D={D} rot={rot} page={page} {dtype} {cache}", flush=True)
        q, k, v = _qkv(T + D, T, hq, hkv, D, dtype)
        pages = -(-2 * T // page) + 1
        g = torch.Generator().manual_seed(5)
        kc = torch.randn(pages, page, hkv, D, generator=g).to(cache)
        vc = torch.randn(pages, page, hkv, D, generator=g).to(cache)
        slots = _slots(T, T, pages * page, torch.int32 if page == 7 else torch.int64)
        if T > 3:  # padding, and slots outside the cache
            slots[0], slots[1], slots[2] = -1, pages * page, -pages
        pos = torch.randint(0, 100000, (T,), generator=g)
        ks, vs = (torch.rand(2, hkv, generator=g) * 0.02 + 0.01).unbind(0) if cache == FP8 else (None, None)
        _check_append(dev, api, q, k, v, kc, vc, slots, pos, _freq(rot), page == 24, 1.0, ks, vs)


def test_append_layouts_without_q_and_without_positions(dev):
    D, page, pages, T = 64, 16, 5, 23
    q, k, v = _qkv(9, T, 4, 2, D, BF16)
    slots = _slots(1, T, pages * page)
    pos, f = torch.arange(T), _freq(D)
    g = torch.Generator().manual_seed(1)
    heads_first = torch.randn(pages, 2, page, D, generator=g).bfloat16().transpose(1, 2)
    both = torch.randn(pages, 2, page, 2, D, generator=g).bfloat16()  # k and v in one pool
    for api in ("cpp", "py"):
        _check_append(dev, _api(api), q, k, v, heads_first, heads_first.clone(), slots, pos, f)
        _check_append(dev, _api(api), q, k, v, both[:, 0], both[:, 1], slots, pos, f)
        _check_append(dev, _api(api), None, k, v, heads_first, heads_first, slots, pos, f)
        _check_append(dev, _api(api), q, k, v, heads_first, heads_first, slots, None, None)
        # [B, T, heads, D] tokens, and padding alone
        _check_append(dev, _api(api), q[:22].unflatten(0, (2, 11)), k[:22].unflatten(0, (2, 11)),
                      v[:22].unflatten(0, (2, 11)), heads_first, heads_first,
                      slots[:22].view(2, 11), pos[:22].view(2, 11), f)
        _check_append(dev, _api(api), q, k, v, heads_first, heads_first,
                      torch.full((T,), -1), pos, f)


def test_append_8_bit_borders(dev):
    """Every finite e4m3 value, the values halfway between two (to the even
    one), beyond the largest, NaN; a scale of 1 keeps them exact."""
    every = torch.arange(256, dtype=torch.uint8).view(FP8).float()
    pos = every[(every >= 0) & every.isfinite()].unique()
    mid = (pos[1:] + pos[:-1]) / 2
    x = torch.cat([pos, mid, torch.tensor([449.0, 1000.0, float("inf")])])
    x = torch.cat([x, -x, torch.tensor([float("nan")])])
    x = torch.nn.functional.pad(x, (0, -x.numel() % 64)).half()
    v = x.view(-1, 1, 64)
    T = v.size(0)
    kc, vc = torch.zeros(1, T, 1, 64, dtype=FP8, device=dev), torch.zeros(1, T, 1, 64, dtype=FP8,
                                                                         device=dev)
    _api("cpp").npu_rotary_cache_append(None, v.to(dev), v.to(dev), kc, vc, torch.arange(T).to(dev))
    want = v.float().clamp(-448, 448).to(FP8).float()
    for c in (kc, vc):
        got = c.cpu().float().view(T, 1, 64)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~want.isnan()], want[~want.isnan()])


def test_append_beyond_32_bit_offsets(dev):
    """Pages past 2^32 bytes of the cache."""
    D, hkv, page = 128, 8, 128
    pages = (1 << 32) // (page * hkv * D * 2) + 3
    kc = torch.zeros(pages, page, hkv, D, dtype=BF16, device=dev)
    vc = torch.zeros(pages, page, hkv, D, dtype=BF16, device=dev)
    q, k, v = _qkv(3, 3, 8, hkv, D, BF16)
    slots = torch.tensor([pages * page - 1, (pages - 2) * page + 5, 7])
    pos, f = torch.arange(3) + 5, _freq(D)
    _api("cpp").npu_rotary_cache_append(q.to(dev), k.to(dev), v.to(dev), kc, vc, slots.to(dev),
                                        pos.to(dev), f.to(dev))
    want, err = rotary.turn(k, pos, f)
    assert_within(kc.view(-1, hkv, D)[slots.to(dev)], want, err, "k")
    assert torch.equal(vc.view(-1, hkv, D)[slots.to(dev)].cpu(), v)
    assert int((vc != 0).any(-1).any(-1).sum()) == 3


def test_many_tokens(dev):
    """A prefill's size: one wave a token, several rounds of units."""
    T, hq, hkv, D = 5000, 24, 3, 128
    q, k, v = _qkv(11, T, hq, hkv, D, F16)
    pages, page = 45, 128
    kc = torch.zeros(pages, page, hkv, D, dtype=F16)
    _check_append(dev, _api("cpp"), q, k, v, kc, kc.clone(), _slots(2, T, pages * page),
                  torch.arange(T) + 30000, _freq(D))


def test_more_blocks_than_a_dimension_holds(dev):
    """2^26 tokens and some: more blocks of four than 2^32 threads are."""
    T, D = (1 << 26) + 5, 2
    f = torch.ones(1)
    x = torch.zeros(T, 1, D, dtype=BF16, device=dev)
    x[:, 0, 0] = 1.0
    pos = torch.zeros(T, dtype=torch.int32, device=dev)
    at = torch.tensor([0, 3, (1 << 25) + 1, (1 << 26) - 1, 1 << 26, T - 1])
    turns = torch.arange(1, 7)
    pos[at.to(dev)] = turns.to(dev, torch.int32)
    y, none = _api("cpp").npu_rotary_embedding(x, None, pos, f.to(dev))
    assert none is None
    want, err = rotary.turn(x[at.to(dev)].cpu(), turns, f)
    assert_within(y[at.to(dev)], want, err, "chosen tokens")
    y[at.to(dev)] = x[at.to(dev)]
    assert torch.equal(y, x)  # the others' angle is 0
