"""GPU checks of the attention over a paged cache against
oracle/paged_attention.py in float64.  Tolerances: the oracle's bound of the
arithmetic plus half a step of the output's type (rounding_tol.py)."""
import math

import pytest
import torch

from oracle import paged_attention as opa
from oracle import rotary
from rounding_tol import assert_within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FP8 = torch.float8_e4m3fn
TYPES = [(BF16, BF16), (F16, F16), (F32, F32), (BF16, FP8), (F16, FP8)]


def _api(name):
    from torch_npu_ops_amd import _xk_torch, ops
    return {"cpp": _xk_torch, "py": ops}[name]


def _pool(seed, lens, page, hkv, D, cache, fill=math.nan, spare=2, std=1.0):
    """Caches whose sequences' pages lie anywhere, `fill` in every place that
    no sequence has, and the table (its unused entries name no page)."""
    g = torch.Generator().manual_seed(seed)
    count = [-(-max(n, 0) // page) for n in lens]
    pages = sum(count) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    width = max(max(count), 1)
    table = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)
    kc, vc = (torch.full((pages, page, hkv, D), fill).to(cache) for _ in range(2))
    at = 0
    for b, n in enumerate(lens):
        table[b, :count[b]] = order[at:at + count[b]]
        for j in range(count[b]):
            m = min(page, n - j * page)
            for c in (kc, vc):
                c[order[at + j], :m] = (torch.randn(m, hkv, D, generator=g) * std).to(cache)
        at += count[b]
    return kc, vc, table


def _query(seed, B, T, hq, D, dtype, std=1.5):
    return (torch.randn(B, T, hq, D, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def _check(dev, api, q, kc, vc, table, lens, scale=None, window=0, ks=None, vs=None, what=""):
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    lens_t = torch.tensor(lens, dtype=torch.int32)
    o, lse = api.npu_paged_attention(on(q), on(kc), on(vc), on(table), on(lens_t), scale, window,
                                     on(ks), on(vs), True)
    want = opa.attention(q, kc, vc, table, lens, scale, window, ks, vs)
    assert o.dtype == q.dtype
    assert_within(o, want["o"], want["o_err"], "o " + what)
    assert_within(lse, want["lse"], want["lse_err"], "lse " + what)
    again, none = api.npu_paged_attention(on(q), on(kc), on(vc), on(table), on(lens_t), scale,
                                          window, on(ks), on(vs))
    assert none is None and torch.equal(o, again)  # no order of atomics: the same bits
    return o, lse


def _scales(seed, hkv, cache):
    if cache != FP8:
        return None, None
    return (torch.rand(2, hkv, generator=torch.Generator().manual_seed(seed)) + 0.25).unbind(0)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("D,hq,hkv", [(8, 3, 1), (64, 8, 2), (80, 15, 5), (128, 4, 4),
                                      (128, 32, 2), (136, 6, 2), (200, 5, 5), (256, 16, 2)])
def test_decode(dev, dtype, cache, D, hq, hkv):
    """One token a sequence: lengths 0, 1, around tiles and pages, and more
    than one part; pages that end inside a tile."""
    for page in (16, 24):
        lens = [0, 1, 15, 16, 33, 100, 700, 31]
        print(f"decode D={D} heads={hq}/{hkv} page={page}", flush=True)
        kc, vc, table = _pool(D + page, lens, page, hkv, D, cache)
        _check(dev, _api("cpp" if page == 16 else "py"), _query(1, len(lens), 1, hq, D, dtype), kc,
               vc, table, lens, None, 0, *_scales(2, hkv, cache))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("page", [1, 5, 32, 100, 128])
@pytest.mark.parametrize("T,G", [(4, 1), (3, 5), (5, 8), (2, 16)])
def test_drafts_and_windows(dev, dtype, cache, page, T, G):
    hkv, D = 2, 64 if page != 32 else 128
    lens = [0, 1, T - 1, T, T + 1, 40, 300, 517]
    kc, vc, table = _pool(page, lens, page, hkv, D, cache)
    q = _query(T, len(lens), T, hkv * G, D, dtype)
    for window in (0, 1, 33, 250):
        print(f"drafts T={T} G={G} page={page} window={window}", flush=True)
        _check(dev, _api("py" if window else "cpp"), q, kc, vc, table, lens, 0.2, window,
               *_scales(3, hkv, cache), what=f"window {window}")


def test_wide_heads_with_many_rows(dev):
    lens = [70, 5, 333]
    for dtype, cache in TYPES:
        kc, vc, table = _pool(4, lens, 16, 2, 256, cache)
        _check(dev, _api("cpp"), _query(5, 3, 6, 16, 256, dtype), kc, vc, table, lens, None, 0,
               *_scales(6, 2, cache))


@pytest.mark.parametrize("B", [63, 64, 65, 150])
def test_many_sequences(dev, B):
    """The plan's search over sequences, ragged and with empty ones."""
    g = torch.Generator().manual_seed(B)
    lens = (torch.rand(B, generator=g) ** 4 * 900).int().tolist()
    lens[3], lens[B - 1] = 0, 2500
    kc, vc, table = _pool(B, lens, 16, 1, 64, BF16)
    _check(dev, _api("cpp"), _query(B, B, 1, 4, 64, BF16), kc, vc, table, lens)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_long_context(dev, dtype, cache):
    """Many parts of one sequence, one of another."""
    lens = [20001, 31]
    kc, vc, table = _pool(7, lens, 64, 1, 128, cache)
    _check(dev, _api("cpp"), _query(8, 2, 1, 8, 128, dtype), kc, vc, table, lens, None, 0,
           *_scales(9, 1, cache))
    _check(dev, _api("py"), _query(8, 2, 2, 8, 128, dtype)[:1], kc, vc, table[:1], lens[:1], None,
           15000, *_scales(9, 1, cache))


def test_far_apart_scores(dev):
    """Scores of hundreds: one position holds all the weight; and equal scores."""
    lens = [900, 17]
    for dtype in (BF16, F16, F32):
        kc, vc, table = _pool(10, lens, 16, 2, 64, dtype)
        _check(dev, _api("cpp"), _query(11, 2, 1, 4, 64, dtype, std=40.0), kc, vc, table, lens)
        _check(dev, _api("cpp"), torch.zeros(2, 1, 4, 64, dtype=dtype), kc, vc, table, lens)
        _check(dev, _api("cpp"), _query(11, 2, 1, 4, 64, dtype), kc, vc, table, lens, 0.0)
        _check(dev, _api("cpp"), _query(11, 2, 1, 4, 64, dtype), kc, vc, table, lens, -0.5)


def test_small_weights_keep_their_digits(dev):
    """fp16: one position outweighs each of 4,000 others by 2^20, which
    together still count; a weight alone would be far below fp16's normals."""
    n, D = 4001, 64
    kc, vc, table = _pool(12, [n], 16, 1, D, F16, fill=0.0)
    for j in range(n):
        kc[table[0, j // 16], j % 16] = 0
        vc[table[0, j // 16], j % 16] = 64.0 if j else 0.0
    kc[table[0, 0], 0, 0, 0] = 20 * math.log(2.0)
    q = torch.zeros(1, 1, 1, D, dtype=F16)
    q[..., 0] = 1.0
    _check(dev, _api("cpp"), q, kc, vc, table, [n], 1.0)


# --------------------------------------------------------------------------
# what masked places hold
# --------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, "most"])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_places_that_nobody_sees(dev, bad, dtype, cache):
    """Places past the end, before the window and in pages that are not there."""
    if cache == FP8 and bad in (math.inf, -math.inf):
        bad = math.nan  # e4m3 has no infinities
    fill = bad if bad != "most" else -torch.finfo(cache).max
    lens = [45, 3, 130]
    for T, window in ((1, 0), (1, 20), (3, 20), (3, 0)):
        kc, vc, table = _pool(13, lens, 16, 2, 64, cache, fill=fill)
        if window:  # old places hold anything, and old pages are gone
            for b, n in enumerate(lens):
                for j in range(max(0, n - T - window + 1)):
                    for c in (kc, vc):
                        c[table[b, j // 16], j % 16] = torch.full((2, 64), fill).to(cache)
            table[2, 0], table[2, 1] = -1, 1 << 29
        q = _query(14, 3, T, 4, 64, dtype)
        got, _ = _check(dev, _api("cpp"), q, kc, vc, table, lens, None, window,
                        *_scales(15, 2, cache))
        assert got.isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_drafts_do_not_see_later_drafts(dev, dtype, bad):
    """A draft's key or value that is not finite has no part in the tokens
    before it, in every token after it."""
    lens, T = [50, 64, 7], 4
    for which in (0, 1):
        for window in (0, 30):
            kc, vc, table = _pool(16, lens, 16, 2, 64, dtype)
            clean = _pool(16, lens, 16, 2, 64, dtype)
            for b, n in enumerate(lens):
                (kc, vc)[which][table[b, (n - 2) // 16], (n - 2) % 16, :, 5] = bad
            q = _query(17, 3, T, 8, 64, dtype).abs()
            want = opa.attention(q, *clean, lens, None, window)
            for api in ("cpp", "py"):
                o, _ = _api(api).npu_paged_attention(
                    q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                    torch.tensor(lens, dtype=torch.int32).to(dev), None, window)
                assert_within(o[:, :2], want["o"][:, :2], want["o_err"][:, :2], "before")
                bad_ones = o[:, 2:].cpu()[..., 5] if which else o[:, 2:].cpu()
                assert (bad_ones.isnan() if math.isnan(bad) or not which else ~bad_ones.isfinite()).all()
                if which:
                    rest = [i for i in range(64) if i != 5]
                    assert o[:, 2:].cpu()[..., rest].isfinite().all()


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_later_drafts_with_many_rows(dev, dtype, cache, D):
    """The same with rows for more than one tile, in every head length, and
    with places that nobody sees filled likewise."""
    lens, T, bad = [50, 64, 7, 200], 4, math.nan
    ks, vs = _scales(90, 2, cache)
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    for which in (0, 1):
        for window in (0, 30):
            kc, vc, table = _pool(91, lens, 16, 2, D, cache, fill=bad)
            clean = _pool(91, lens, 16, 2, D, cache, fill=0.0)
            for b, n in enumerate(lens):
                place = (kc, vc)[which][table[b, (n - 2) // 16], (n - 2) % 16]
                x = place.float()
                x[:, 5] = bad
                place.copy_(x.to(cache))
            q = _query(92, 4, T, 20, D, dtype)
            want = opa.attention(q, *clean, lens, None, window, ks, vs)
            o, _ = _api("cpp").npu_paged_attention(
                on(q), on(kc), on(vc), on(table), torch.tensor(lens, dtype=torch.int32).to(dev), None,
                window, on(ks), on(vs))
            assert_within(o[:, :2], want["o"][:, :2], want["o_err"][:, :2], f"before {which} {window}")
            after = o[:, 2:].cpu()
            assert (after[..., 5] if which else after).isnan().all()
            if which:
                rest = [i for i in range(D) if i != 5]
                assert_within(after[..., rest], want["o"][:, 2:][..., rest],
                              want["o_err"][:, 2:][..., rest], f"after {window}")


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_either_side_of_the_choice_of_row_tiles(dev, dtype, cache, D):
    """Batches with little and with much to read, whose rows of tokens and
    heads fill one tile and a half."""
    for lens in ([300, 0, 40], [5000, 3000, 25000, 1]):
        kc, vc, table = _pool(93, lens, 64, 1, D, cache)
        for window in (0, 2000):
            _check(dev, _api("cpp"), _query(94, len(lens), 3, 8, D, dtype), kc, vc, table, lens, None,
                   window, *_scales(95, 1, cache))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("D,hkv", [(8, 8), (8, 12), (16, 6), (32, 7), (64, 2), (64, 10)])
def test_heads_that_share_cache_lines(dev, dtype, cache, D, hkv):
    """Rows of 8 to 256 bytes, numbers of heads with and without common factors."""
    lens = [1500, 0, 33, 700]
    kc, vc, table = _pool(98, lens, 16, hkv, D, cache)
    for T in (1, 9):
        _check(dev, _api("cpp"), _query(99, 4, T, 2 * hkv, D, dtype), kc, vc, table, lens, None, 0,
               *_scales(100, hkv, cache))


def test_windows_beyond_every_length(dev):
    lens = [700, 3]
    kc, vc, table = _pool(96, lens, 16, 2, 64, BF16)
    q = _query(97, 2, 5, 8, 64, BF16)
    for api in ("cpp", "py"):
        args = [t.to(dev) for t in (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))]
        want = _api(api).npu_paged_attention(*args)[0]
        for window in (700, 1 << 28, (1 << 31) - 1, 1 << 31, (1 << 63) - 1):
            assert torch.equal(_api(api).npu_paged_attention(*args, None, window)[0], want)


def test_pages_that_are_not_there(dev):
    """Entries outside the cache count as masked, in the middle too."""
    lens = [100, 40, 64]
    for page in (16, 10, 32):
        kc, vc, table = _pool(18, lens, page, 2, 64, BF16)
        table[0, 1], table[0, 2], table[1, :] = -1, kc.size(0), -5
        _, lse = _check(dev, _api("cpp"), _query(19, 3, 2, 4, 64, BF16), kc, vc, table, lens)
        assert (lse[1] == -math.inf).all()


def test_lengths_beyond_the_table_and_empty_pools(dev):
    lens = [1000, -7, 33]
    kc, vc, table = _pool(20, [48, 48, 48], 16, 2, 64, BF16)
    _check(dev, _api("cpp"), _query(21, 3, 1, 4, 64, BF16), kc, vc, table, lens)
    for api in ("cpp", "py"):
        for k, t in ((kc[:0], table), (kc, table[:, :0])):
            o, lse = _api(api).npu_paged_attention(
                _query(21, 3, 2, 4, 64, BF16).to(dev), k.to(dev), k.to(dev), t.to(dev),
                torch.tensor(lens, dtype=torch.int32).to(dev), output_lse=True)
            assert (o == 0).all() and (lse == -math.inf).all()
        for B, T in ((0, 1), (3, 0)):
            o, lse = _api(api).npu_paged_attention(
                torch.zeros(B, T, 4, 64, dtype=BF16, device=dev), kc.to(dev), vc.to(dev),
                table[:B].to(dev), torch.zeros(B, dtype=torch.int32, device=dev), output_lse=True)
            assert o.shape == (B, T, 4, 64) and lse.shape == (B, T, 4)


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("page", [48, 64, 96, 256])
@pytest.mark.parametrize("D", [64, 128])
def test_runs_of_pages(dev, dtype, cache, page, D):
    """Pages that hold whole tiles, halves or quarters of them: a table entry
    serves 64, 32 or 16 positions."""
    lens = [0, 1, page, page + 1, 3 * page - 1, 1100, 63]
    kc, vc, table = _pool(60 + page, lens, page, 2, D, cache)
    for T in (1, 6):
        print(f"runs page={page} D={D} T={T}", flush=True)
        _check(dev, _api("cpp"), _query(61, len(lens), T, 8, D, dtype), kc, vc, table, lens, None,
               0 if T == 1 else 200, *_scales(62, 2, cache))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_many_new_tokens(dev, dtype, cache):
    """Row groups of a head, each with positions of its own."""
    lens = [70, 71, 300, 12]
    kc, vc, table = _pool(63, lens, 16, 2, 64, cache)
    for window in (0, 50):
        _check(dev, _api("cpp"), _query(64, 4, 70, 8, 64, dtype), kc, vc, table, lens, None, window,
               *_scales(65, 2, cache))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_many_short_sequences(dev, dtype, cache):
    """Shares that hold many sequences whole, of a tile or none each."""
    g = torch.Generator().manual_seed(66)
    lens = torch.randint(0, 40, (700,), generator=g).tolist()
    kc, vc, table = _pool(67, lens, 16, 8, 64, cache)
    _check(dev, _api("cpp"), _query(68, 700, 1, 16, 64, dtype), kc, vc, table, lens, None, 0,
           *_scales(69, 8, cache))


@pytest.mark.parametrize("D", [64, 256])
def test_many_pieces(dev, D):
    """More pieces of a sequence than the lanes that join them take at once."""
    lens = [30001]
    kc, vc, table = _pool(70, lens, 16, 1, D, BF16)
    for T in (1, 3):
        _check(dev, _api("cpp"), _query(71, 1, T, 4, D, BF16), kc, vc, table, lens)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_one_share_needs_no_workspace(dev, dtype, cache):
    lens = [20, 7]
    kc, vc, table = _pool(72, lens, 16, 2, 64, cache)
    for api in ("cpp", "py"):
        _check(dev, _api(api), _query(73, 2, 1, 8, 64, dtype), kc, vc, table, lens, None, 0,
               *_scales(74, 2, cache))


# --------------------------------------------------------------------------
# layouts
# --------------------------------------------------------------------------
def test_layouts_and_views(dev):
    lens = [77, 300]
    for dtype, cache in TYPES:
        kc, vc, table = _pool(22, lens, 16, 2, 64, cache, fill=0.0)
        ks, vs = _scales(23, 2, cache)
        q = _query(24, 2, 3, 8, 64, dtype)
        want = opa.attention(q, kc, vc, table, lens, None, 0, ks, vs)
        on = lambda t: None if t is None else t.to(dev)  # noqa: E731
        n = torch.tensor(lens, dtype=torch.int32).to(dev)
        as_bytes = lambda c: c.to(dev).view(torch.uint8) if cache == FP8 else c.to(dev)  # noqa: E731
        typed = lambda c: c.view(FP8) if cache == FP8 else c  # noqa: E731
        heads_first = [typed(as_bytes(c).transpose(1, 2).contiguous().transpose(1, 2)) for c in (kc, vc)]
        both = typed(torch.stack([as_bytes(kc), as_bytes(vc)], 1))
        wide = torch.zeros(2, 3, 8, 128, dtype=dtype, device=dev)
        wide[..., 64:] = q.to(dev)
        odd = torch.zeros(2 * 3 * 8 * 64 + 1, dtype=dtype, device=dev)[1:].view(2, 3, 8, 64)
        odd.copy_(q)
        queries = [q.to(dev), wide[..., 64:], odd, q.to(dev).transpose(1, 2).contiguous().transpose(1, 2)]
        tables = [table.to(dev), table.to(dev).repeat(1, 2)[:, :table.size(1)],
                  table.to(dev).t().contiguous().t()]
        for api in ("cpp", "py"):
            for k, v in (heads_first, (both[:, 0], both[:, 1])):
                for i in range(4):
                    o, _ = _api(api).npu_paged_attention(queries[i], k, v, tables[i % 3], n, None, 0,
                                                         on(ks), on(vs))
                    assert_within(o, want["o"], want["o_err"], f"layout {i}")
            o, lse = _api(api).npu_paged_attention(queries[0][:, 0], k, v, tables[0], n, None, 0,
                                                   on(ks), on(vs), True)
            assert o.shape == (2, 8, 64) and lse.shape == (2, 8)


def test_shared_pages(dev):
    """Sequences with a common prefix share its pages."""
    kc, vc, table = _pool(25, [64, 70, 90], 16, 2, 64, BF16)
    table[1, :4], table[2, :4] = table[0, :4], table[0, :4]
    _check(dev, _api("cpp"), _query(26, 3, 1, 8, 64, BF16), kc, vc, table, [64, 70, 90])


def test_beyond_32_bit_offsets(dev):
    """Pages past 2^32 bytes of the cache."""
    D, hkv, page = 128, 8, 128
    pages = (1 << 32) // (page * hkv * D * 2) + 4
    small = _pool(27, [300], page, hkv, D, BF16, fill=0.0, spare=0)
    far = torch.tensor([[pages - 1, 2, pages - 3]], dtype=torch.int32)
    pools = []
    for c in small[:2]:
        pool = torch.zeros(pages, page, hkv, D, dtype=BF16, device=dev)
        pool[far[0].long().to(dev)] = c[small[2][0].long()].to(dev)
        pools.append(pool)
    q = _query(28, 1, 1, 16, D, BF16)
    want = opa.attention(q, *small, [300])
    o, _ = _api("cpp").npu_paged_attention(q.to(dev), *pools, far.to(dev),
                                           torch.tensor([300], dtype=torch.int32).to(dev))
    assert_within(o, want["o"], want["o_err"], "far pages")


# --------------------------------------------------------------------------
# as it is used
# --------------------------------------------------------------------------
def _layer(api, x, kc, vc, table, slots, pos, f, lens, hq, hkv, D, window=0, ks=None, vs=None):
    """A layer's step between its projections: [B, T, row] -> [B, T, Hq, D]."""
    q, k, v = (p.unflatten(-1, (-1, D)) for p in x.split([hq * D, hkv * D, hkv * D], -1))
    q = api.npu_rotary_cache_append(q, k, v, kc, vc, slots, pos, f, False, 1.0, ks, vs)
    return api.npu_paged_attention(q, kc, vc, table, lens, None, window, ks, vs)[0]


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_prefill_then_decode_with_drafts(dev, dtype, cache):
    """Prompts enter the cache, then steps of 1 and 3 tokens follow, the
    rejected drafts' places written again; against attention over all tokens
    in 64 bits from the rounded cache."""
    hq, hkv, D, page = 8, 2, 64, 16
    prompts, f = [37, 5], (1e4 ** (-torch.arange(0, D, 2) / D)).float()
    g = torch.Generator().manual_seed(30)
    row = (hq + 2 * hkv) * D
    ks, vs = _scales(31, hkv, cache)
    on = lambda t: None if t is None else t.to(dev)  # noqa: E731
    pages = 12
    table = torch.randperm(pages, generator=g).to(torch.int32).view(2, 6)
    kc, vc = (torch.zeros(pages, page, hkv, D).to(cache).to(dev) for _ in range(2))

    def slots_of(b, at):
        return table[b, at // page].long() * page + at % page

    for b, n in enumerate(prompts):
        x = torch.randn(n, row, generator=g).to(dtype)
        _, k, v = (p.unflatten(-1, (-1, D)) for p in x.split([hq * D, hkv * D, hkv * D], -1))
        at = torch.arange(n)
        _api("cpp").npu_rotary_cache_append(None, on(k), on(v), kc, vc, on(slots_of(b, at)), on(at),
                                            on(f), False, 1.0, on(ks), on(vs))
    lens = list(prompts)
    for T, kept in ((1, 1), (3, 2), (3, 1), (1, 1)):
        x = torch.randn(2, T, row, generator=g).to(dtype)
        pos = torch.stack([torch.arange(n, n + T) for n in lens])
        slots = torch.stack([slots_of(b, pos[b]) for b in range(2)])
        now = torch.tensor([n + T for n in lens], dtype=torch.int32)
        o = _layer(_api("cpp"), on(x), kc, vc, on(table), on(slots), on(pos), on(f), on(now), hq, hkv,
                   D, 0, on(ks), on(vs))
        q = x.split([hq * D, hkv * D, hkv * D], -1)[0].unflatten(-1, (-1, D))
        turned, err = rotary.turn(q, pos, f)
        got_q = _api("cpp").npu_rotary_embedding(on(q), None, on(pos), on(f))[0]
        assert_within(got_q, turned, err, "q")
        want = opa.attention(got_q.cpu(), kc.cpu(), vc.cpu(), table, now.tolist(), None, 0, ks, vs)
        assert_within(o, want["o"], want["o_err"], f"step of {T}")
        lens = [n + kept for n in lens]


def test_captured_step(dev):
    """A decode step captured once and replayed as the sequences grow: the
    lengths, slots and positions are read from the same buffers; eager steps
    and synchronizations between the replays."""
    hq, hkv, D, page, B = 8, 2, 128, 16, 3
    f = (1e4 ** (-torch.arange(0, D, 2) / D)).float().to(dev)
    g = torch.Generator().manual_seed(32)
    row = (hq + 2 * hkv) * D
    table = torch.randperm(60, generator=g).to(torch.int32).view(3, 20).to(dev)
    caches = [torch.randn(60, page, hkv, D, generator=g).bfloat16().to(dev) for _ in range(2)]
    lens = torch.tensor([250, 3, 120], dtype=torch.int32, device=dev)
    x = torch.zeros(B, 1, row, dtype=BF16, device=dev)
    api = _api("cpp")

    def step(kc, vc):
        pos = (lens - 1)[:, None]
        slots = table.gather(1, (pos // page).long()).long() * page + pos % page
        return _layer(api, x, kc, vc, table, slots, pos, f, lens, hq, hkv, D)

    other = [c.clone() for c in caches]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*other)
    torch.cuda.current_stream().wait_stream(side)
    for c, o in zip(caches, other):
        o.copy_(c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*caches)
    for i in range(4):
        x.copy_(torch.randn(B, 1, row, generator=g).bfloat16())
        lens += 1
        torch.cuda.synchronize()
        want = step(*other)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert all(torch.equal(c, o) for c, o in zip(caches, other)), i


def test_two_streams_at_once(dev):
    """Calls that overlap have a workspace each (the C++ API's come from the
    allocator, by stream)."""
    api = _api("cpp")
    cases = []
    for i, lens in enumerate(([9000, 20], [100, 8000])):
        kc, vc, table = _pool(40 + i, lens, 16, 2, 128, BF16)
        q = _query(50 + i, 2, 1, 16, 128, BF16)
        n = torch.tensor(lens, dtype=torch.int32)
        cases.append([t.to(dev) for t in (q, kc, vc, table, n)])
    alone = [api.npu_paged_attention(*c)[0] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(api.npu_paged_attention(*cases[i])[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(alone[i], o) for o in got[i])


def test_two_graphs_and_eager_calls(dev):
    """Two captured calls replayed at once on two streams, eager ones between."""
    api = _api("cpp")
    calls, graphs, outs = [], [], []
    for i, lens in enumerate(([5000, 20], [100, 3000])):
        kc, vc, table = _pool(80 + i, lens, 16, 2, 128, BF16)
        q = _query(82 + i, 2, 1, 16, 128, BF16)
        calls.append([t.to(dev) for t in (q, kc, vc, table, torch.tensor(lens, dtype=torch.int32))])
    alone = [api.npu_paged_attention(*c)[0] for c in calls]
    torch.cuda.synchronize()
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(api.npu_paged_attention(*c)[0])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in calls]
    for i in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [api.npu_paged_attention(*c)[0] for c in calls]
        torch.cuda.synchronize()
        for a, o, e in zip(alone, outs, eager):
            assert torch.equal(a, o) and torch.equal(a, e), i
