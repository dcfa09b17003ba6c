"""GPU checks of the gated linear recurrence (forward, decode step, backward)
against oracle/recurrence.py in float64.  Tolerances: the oracle's bound of
the fp32 arithmetic plus half a step of the output's type (rounding_tol.py).
"""
import pytest
import torch

from oracle import recurrence as orc
from rounding_tol import assert_within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
C = 8.0


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _lam(g, D):
    # softplus(lam) from 1e-4 (long memory) to 1 (a few tokens)
    return torch.log(torch.expm1(10.0 ** (-4 * torch.rand(D, generator=g)))).float()


def _inputs(seed, total, D, n, dtype):
    g = _gen(seed)
    x, a, b, dy = (torch.randn(1, total, D, generator=g).clamp_(-8, 8).to(dtype)
                   for _ in range(4))
    h0, df = (torch.randn(n, D, generator=g) for _ in range(2))
    return x, a, b, dy, _lam(g, D), h0, df


def _cu(lens, first=0):
    at = [first]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _live(cu, total):
    m = torch.zeros(total, dtype=torch.bool)
    for t0, t1 in orc.runs(cu, total):
        m[t0:t1] = True
    return m


def _both():
    from torch_npu_ops_amd import _xk_torch, ops
    return {"cpp": _xk_torch, "py": ops}


def _check(dev, api, lens, D, dtype, seed=0, c=C, states=True, h0=True, cu_dtype=torch.int32,
           behind=0, first=0):
    cu = _cu(lens, first)
    total = cu[-1] + behind
    x, a, b, dy, lam, start, df = _inputs(seed, total, D, len(lens), dtype)
    start = start if h0 else None
    d = [t.to(dev) for t in (x, a, b, lam)]
    cud = torch.tensor(cu, dtype=cu_dtype, device=dev)
    sd = start.to(dev) if h0 else None
    y, fin, st = api.npu_gated_linear_recurrence(*d, c, sd, True, cud, True)
    ref = orc.forward(x[0], a[0], b[0], lam, c, start, cu)
    m = _live(cu, total)
    assert_within(y[0].cpu()[m], ref["h"][m], ref["h_err"][m], "y")
    assert_within(fin, ref["final"], ref["final_err"], "final state")
    assert st.shape == (-(-total // 16), D)
    starts = {t0 for t0, t1 in orc.runs(cu, total) if t1 > t0}
    rows = [w for w in range(st.size(0)) if m[16 * w] and 16 * w not in starts]
    if rows:
        tok = [16 * w for w in rows]
        assert_within(st[rows], ref["before"][tok], ref["before_err"][tok], "states")
    plain = api.npu_gated_linear_recurrence(*d, c, sd, False, cud)
    assert torch.equal(plain[0][0][m], y[0][m]) and plain[1] is None and plain[2] is None
    got = api.npu_gated_linear_recurrence_bwd(dy.to(dev), *d, st, c, sd, df.to(dev), cud)
    want = orc.backward(dy[0], x[0], a[0], b[0], lam, c, start, df, cu)
    for name, t in zip(("dx", "da", "db"), got):
        assert_within(t[0].cpu()[m], want[name][m], want[name + "_err"][m], name)
    assert_within(got[3], want["dlam"], want["dlam_err"], "dlam")
    assert_within(got[4], want["dh0"], want["dh0_err"], "dh0")


LENS = [[1], [2, 1, 3], [15], [16], [17], [64, 65], [130], [257, 1, 127], [600]]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_lengths(dev, lens, dtype):
    print(f"lens={lens} {dtype}", flush=True)
    _check(dev, _both()["cpp"], lens, 130, dtype, seed=sum(lens))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", [1, 2, 3, 63, 64, 65, 127, 128, 129, 255, 520])
def test_widths(dev, D, dtype):
    print(f"D={D} {dtype}", flush=True)
    _check(dev, _both()["cpp"], [70, 3, 33], D, dtype, seed=D)


@pytest.mark.parametrize("which", ["cpp", "py"])
@pytest.mark.parametrize("kw", [dict(h0=False), dict(c=0.5), dict(c=0.0),
                                dict(cu_dtype=torch.int64), dict(behind=37), dict(first=21),
                                dict(first=200, behind=150)], ids=str)
def test_options(dev, which, kw):
    print(f"{which} {kw}", flush=True)
    _check(dev, _both()[which], [40, 0, 100, 1, 0], 96, BF16, seed=5, **kw)


@pytest.mark.parametrize("lens", [[0], [0, 0, 5], [3, 0, 0, 0, 140, 0], [0] * 90 + [9] + [0] * 80],
                         ids=lambda v: f"{len(v)}seqs")
def test_empty_sequences_keep_their_state(dev, lens):
    _check(dev, _both()["cpp"], lens, 66, BF16, seed=len(lens), behind=0 if sum(lens) else 4)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 300])
def test_many_short_sequences(dev, n):
    lens = [1 + (7 * k) % 5 for k in range(n)]
    _check(dev, _both()["cpp"], lens, 40, BF16, seed=n)


def test_no_tokens_at_all(dev):
    for api in _both().values():
        x = torch.empty(1, 0, 8, device=dev)
        lam, h0 = torch.zeros(8, device=dev), torch.randn(2, 8, device=dev)
        cu = torch.zeros(3, dtype=torch.int32, device=dev)
        y, fin, st = api.npu_gated_linear_recurrence(x, x, x, lam, 8.0, h0, True, cu, True)
        assert y.shape == x.shape and st.shape == (0, 8) and torch.equal(fin, h0)
        out = api.npu_gated_linear_recurrence_bwd(x, x, x, x, lam, st, 8.0, h0, h0, cu)
        assert torch.equal(out[4], h0) and (out[3] == 0).all()


@pytest.mark.parametrize("B,T", [(1, 1), (3, 50), (5, 16), (2, 131)])
def test_batch_rows_without_cu_seqlens(dev, B, T):
    x, a, b, dy, lam, h0, df = _inputs(B * T, B * T, 72, B, BF16)
    view = [t.view(B, T, 72).to(dev) for t in (x, a, b)]
    cu = list(range(0, B * T + 1, T))
    for api in _both().values():
        y, fin, st = api.npu_gated_linear_recurrence(*view, lam.to(dev), C, h0.to(dev), True, None,
                                                     True)
        ref = orc.forward(x[0], a[0], b[0], lam, C, h0, cu)
        assert_within(y.view(B * T, 72), ref["h"], ref["h_err"], "y")
        assert_within(fin, ref["final"], ref["final_err"], "final")
        got = api.npu_gated_linear_recurrence_bwd(dy.view(B, T, 72).to(dev), *view, lam.to(dev),
                                                  st, C, h0.to(dev))
        want = orc.backward(dy[0], x[0], a[0], b[0], lam, C, h0, None, cu)
        assert_within(got[1].view(B * T, 72), want["da"], want["da_err"], "da")
        assert_within(got[4], want["dh0"], want["dh0_err"], "dh0")


def _view_forms(dev, t, form):
    """t [1, T, D] in another memory layout."""
    T, D = t.shape[1:]
    if form == "slice":
        wide = torch.randn(1, T, 2 * D + 3, device=dev).to(t.dtype)
        wide[..., 1:1 + D] = t
        return wide[..., 1:1 + D]
    if form == "every_other":
        wide = torch.randn(1, 2 * T, D, device=dev).to(t.dtype)
        wide[:, ::2] = t
        return wide[:, ::2]
    if form == "channel_major":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    assert form == "expanded"  # one channel's value for all
    return t[..., :1].expand(-1, -1, D)


@pytest.mark.parametrize("form", ["slice", "every_other", "channel_major", "expanded"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views_equal_contiguous_copies(dev, form, dtype):
    x, a, b, dy, lam, h0, df = _inputs(9, 90, 75, 2, dtype)
    x, a, b, dy = (_view_forms(dev, t.to(dev), form) for t in (x, a, b, dy))
    lam, h0, df = lam.to(dev), h0.to(dev), df.to(dev)
    cu = torch.tensor([0, 33, 90], dtype=torch.int32, device=dev)
    for api in _both().values():
        one = api.npu_gated_linear_recurrence(x, a, b, lam, C, h0, True, cu, True)
        grad = api.npu_gated_linear_recurrence_bwd(dy, x, a, b, lam, one[2], C, h0, df, cu)
        xc, ac, bc, dyc = (t.contiguous() for t in (x, a, b, dy))
        two = api.npu_gated_linear_recurrence(xc, ac, bc, lam, C, h0, True, cu, True)
        same = api.npu_gated_linear_recurrence_bwd(dyc, xc, ac, bc, lam, two[2], C, h0, df, cu)
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
        assert all(torch.equal(p, q) for p, q in zip(grad, same))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nothing_leaks_from_a_sequence_or_from_rows_outside(dev, bad):
    # The rows before, between and behind, and all of one sequence, hold `bad`.
    from torch_npu_ops_amd import _xk_torch as xt
    total, D = 420, 70
    cu = [10, 150, 280, 400]
    x, a, b, dy, lam, h0, df = _inputs(11, total, D, 3, BF16)
    want = orc.forward(x[0], a[0], b[0], lam, C, h0, cu)
    grads = orc.backward(dy[0], x[0], a[0], b[0], lam, C, h0, df, cu)
    spoiled = torch.ones(total, dtype=torch.bool)
    spoiled[10:150] = False
    spoiled[280:400] = False
    for t in (x, a, b, dy):
        t[0, spoiled] = bad
    h0[1], df[1] = bad, bad
    d = [t.to(dev) for t in (x, a, b, lam)]
    cud = torch.tensor(cu, dtype=torch.int32, device=dev)
    y, fin, st = xt.npu_gated_linear_recurrence(*d, C, h0.to(dev), True, cud, True)
    got = xt.npu_gated_linear_recurrence_bwd(dy.to(dev), *d, st, C, h0.to(dev), df.to(dev), cud)
    m = ~spoiled
    assert_within(y[0].cpu()[m], want["h"][m], want["h_err"][m], "y")
    assert_within(fin[[0, 2]], want["final"][[0, 2]], want["final_err"][[0, 2]], "final")
    for name, t in zip(("dx", "da", "db"), got):
        assert_within(t[0].cpu()[m], grads[name][m], grads[name + "_err"][m], name)
    assert_within(got[4][[0, 2]], grads["dh0"][[0, 2]], grads["dh0_err"][[0, 2]], "dh0")


def test_a_value_that_is_not_finite_stays_in_its_sequence_from_its_token_on(dev):
    from torch_npu_ops_amd import _xk_torch as xt
    x, a, b, _, lam, _, _ = _inputs(12, 300, 8, 1, F32)
    x[0, 100, 3] = float("nan")
    y, fin, _ = xt.npu_gated_linear_recurrence(x.to(dev), a.to(dev), b.to(dev), lam.to(dev), C,
                                               None, True)
    bad = y[0].isnan().cpu()
    assert bad[100:, 3].all() and int(bad.sum()) == 200 and fin[0, 3].isnan()


@pytest.mark.parametrize("a_value,lam_value", [(-1e4, 0.0), (-float("inf"), 0.0), (90.0, -60.0),
                                               (0.0, -100.0), (1e4, 80.0), (-200.0, 30.0)])
def test_gates_at_their_ends(dev, a_value, lam_value):
    # The state is kept or forgotten whole; no gradient is NaN.
    from torch_npu_ops_amd import _xk_torch as xt
    T, D = 40, 6
    x, _, b, dy, _, h0, df = _inputs(13, T, D, 1, F32)
    a, lam = torch.full((1, T, D), a_value), torch.full((D,), lam_value)
    d = [t.to(dev) for t in (x, a, b, lam)]
    y, fin, st = xt.npu_gated_linear_recurrence(*d, C, h0.to(dev), True, None, True)
    ref = orc.forward(x[0], a[0], b[0], lam, C, h0, [0, T])
    torch.testing.assert_close(y[0].cpu().double(), ref["h"], rtol=1e-5, atol=1e-5)
    got = xt.npu_gated_linear_recurrence_bwd(dy.to(dev), *d, st, C, h0.to(dev), df.to(dev))
    want = orc.backward(dy[0], x[0], a[0], b[0], lam, C, h0, df, [0, T])
    for name, t in zip(("dx", "da", "db"), got):
        torch.testing.assert_close(t[0].cpu().double(), want[name], rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(got[4].cpu().double(), want["dh0"], rtol=1e-4, atol=1e-5)
    assert got[3].isfinite().all()


def test_gradients_against_differences(dev):
    # fp32, central differences of the device's own forward pass in a loss of
    # 400 terms: each is off by its rounding (2^-24 of |h| <= 8, 1e-6 of a
    # difference 2e-2 wide) and by the cubic term (step^2 / 6 of a third
    # derivative of order 1): 2e-3 covers both.
    from torch_npu_ops_amd import _xk_torch as xt
    T, D = 40, 10
    x, a, b, dy, lam, h0, df = (t.to(dev) for t in _inputs(14, T, D, 2, F32))
    cu = torch.tensor([0, 23, 40], dtype=torch.int32, device=dev)

    def loss(*args):
        y, fin, _ = xt.npu_gated_linear_recurrence(*args[:4], C, args[4], True, cu)
        return (y.double() * dy).sum() + (fin.double() * df).sum()
    args = [x, a, b, lam, h0]
    st = xt.npu_gated_linear_recurrence(x, a, b, lam, C, h0, False, cu, True)[2]
    dx, da, db, dlam, dh0 = xt.npu_gated_linear_recurrence_bwd(dy, x, a, b, lam, st, C, h0, df, cu)
    g = _gen(15)
    for k, grad in enumerate((dx, da, db, dlam, dh0)):
        way = torch.randn(args[k].shape, generator=g).to(dev)
        way /= way.norm()
        step = 1e-2
        ends = [loss(*[t + s * step * way if j == k else t for j, t in enumerate(args)])
                for s in (1, -1)]
        got = float((grad.double() * way).sum())
        assert got == pytest.approx(float(ends[0] - ends[1]) / (2 * step), rel=2e-3, abs=2e-3)


def test_the_same_call_gives_the_same_bits(dev):
    from torch_npu_ops_amd import _xk_torch as xt
    x, a, b, dy, lam, h0, df = (t.to(dev) for t in _inputs(16, 6000, 300, 3, BF16))
    cu = torch.tensor([0, 2500, 2600, 6000], dtype=torch.int32, device=dev)
    first = None
    for _ in range(6):
        y, fin, st = xt.npu_gated_linear_recurrence(x, a, b, lam, C, h0, True, cu, True)
        out = [y, fin] + list(xt.npu_gated_linear_recurrence_bwd(dy, x, a, b, lam, st, C, h0, df,
                                                                 cu))
        first = first or out
        assert all(torch.equal(p, q) for p, q in zip(first, out))


def test_two_streams_at_once_and_off_the_default_stream(dev):
    from torch_npu_ops_amd import _xk_torch as xt
    sets = [tuple(t.to(dev) for t in _inputs(20 + k, 5000, 256, 1, BF16)) for k in range(2)]
    cu = torch.tensor([0, 5000], dtype=torch.int32, device=dev)

    def both(s):
        x, a, b, dy, lam, h0, df = s
        y, fin, st = xt.npu_gated_linear_recurrence(x, a, b, lam, C, h0, True, cu, True)
        return [y, fin, *xt.npu_gated_linear_recurrence_bwd(dy, x, a, b, lam, st, C, h0, df, cu)]
    want = [both(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[], []]
    for _ in range(4):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[k].append(both(sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for out in outs[k]:
            assert all(torch.equal(p, q) for p, q in zip(want[k], out))


def test_captured_and_replayed(dev):
    from torch_npu_ops_amd import _xk_torch as xt
    x, a, b, dy, lam, h0, df = (t.to(dev) for t in _inputs(30, 3000, 200, 2, BF16))
    cu = torch.tensor([0, 1111, 3000], dtype=torch.int32, device=dev)

    def both():
        y, fin, st = xt.npu_gated_linear_recurrence(x, a, b, lam, C, h0, True, cu, True)
        return [y, fin, *xt.npu_gated_linear_recurrence_bwd(dy, x, a, b, lam, st, C, h0, df, cu)]
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(4):
        x.copy_(torch.randn(x.shape, generator=_gen(40 + k)).to(x.dtype))
        if k == 2:  # other lengths, the same graph
            cu.copy_(torch.tensor([0, 2000, 2900], dtype=torch.int32))
        want = both()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        end = int(cu[-1])
        for p, q in zip(want[:1] + want[2:5], out[:1] + out[2:5]):
            assert torch.equal(p[:, :end], q[:, :end])
        assert torch.equal(want[1], out[1]) and torch.equal(want[5], out[5])
        assert torch.equal(want[6], out[6])


def test_rows_outside_are_left_and_buffers_may_be_shared(dev):
    """The C-ABI: y over x, the final state over the initial one."""
    from torch_npu_ops_amd import _lib
    x, a, b, _, lam, h0, _ = (t.to(dev) for t in _inputs(50, 400, 66, 3, BF16))
    cu = torch.tensor([5, 130, 130, 390], dtype=torch.int32, device=dev)
    ref = orc.forward(x[0].cpu(), a[0].cpu(), b[0].cpu(), lam.cpu(), C, h0.cpu(), cu.tolist())
    before = x.clone()
    lib = _lib.lib()
    size = lib.xk_gated_linear_recurrence_workspace_bytes(400, 66)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device=dev)
    st = lib.xk_gated_linear_recurrence(
        x.data_ptr(), 66, a.data_ptr(), 66, b.data_ptr(), 66, _lib.XK_BF16, lam.data_ptr(), C,
        x.data_ptr(), 66, h0.data_ptr(), h0.data_ptr(), None, cu.data_ptr(), _lib.XK_I32, 3, 400,
        66, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    assert st == _lib.XK_OK
    m = _live(cu.tolist(), 400)
    assert_within(x[0].cpu()[m], ref["h"][m], ref["h_err"][m], "y")
    assert_within(h0, ref["final"], ref["final_err"], "final")
    assert torch.equal(x[0].cpu()[~m], before[0].cpu()[~m])


def test_offsets_beyond_32_bits(dev):
    # 50,000 tokens of pitch 46,000: the last row starts at element 2.3e9.
    from torch_npu_ops_amd import _xk_torch as xt
    T, D, pitch = 50000, 4, 46000
    x, a, b, dy, lam, h0, _ = _inputs(60, T, D, 1, BF16)
    wide = torch.empty(1, T, pitch, dtype=BF16, device=dev)
    wide[..., -D:] = x.to(dev)
    xv = wide[..., -D:]
    d = [t.to(dev) for t in (a, b, lam)]
    y, fin, st = xt.npu_gated_linear_recurrence(xv, *d, C, h0.to(dev), True, None, True)
    two = xt.npu_gated_linear_recurrence(x.to(dev), *d, C, h0.to(dev), True, None, True)
    assert torch.equal(y, two[0]) and torch.equal(fin, two[1])
    got = xt.npu_gated_linear_recurrence_bwd(dy.to(dev), xv, *d, st, C, h0.to(dev))
    want = xt.npu_gated_linear_recurrence_bwd(dy.to(dev), x.to(dev), *d, st, C, h0.to(dev))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    ref = orc.forward(x[0, :2000], a[0, :2000], b[0, :2000], lam, C, h0, [0, 2000])
    assert_within(y[0, :2000], ref["h"], ref["h_err"], "y")


# ---------------------------------------------------------------------------
# decode step
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [1, 5, 64, 130, 516, 1024])
@pytest.mark.parametrize("n", [1, 7])
def test_update_one_token(dev, n, D, dtype):
    x, a, b, _, lam, _, _ = _inputs(n + D, n, D, n, dtype)
    pool = torch.randn(n + 3, D, generator=_gen(1))
    slots = torch.randperm(n + 3, generator=_gen(2))[:n].tolist()
    slots[-1] = -1 if n > 1 else slots[-1]
    want, err, new, new_err = orc.update(x[0], a[0], b[0], lam, C, pool, slots, None,
                                         list(range(n + 1)))
    for api in _both().values():
        pd = pool.to(dev)
        y = api.npu_gated_linear_recurrence_update(
            x[0].to(dev), a[0].to(dev), b[0].to(dev), lam.to(dev), pd, C,
            torch.tensor(slots, dtype=torch.int32, device=dev))
        assert y.shape == (n, D)
        assert_within(y, want, err, "y")
        assert_within(pd, new, new_err, "pool")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,cols", [(1, 1), (4, 4), (3, 5), (5, 2)])
def test_update_drafted_tokens(dev, T, cols, dtype):
    n, D = 6, 200
    x, a, b, _, lam, _, _ = _inputs(T, n * T, D, n, dtype)
    lines = n * cols + 2
    pool = torch.randn(lines, D, generator=_gen(3))
    table = torch.randperm(lines, generator=_gen(4))[:n * cols].view(n, cols)
    table[2, 0] = -1
    table[3, -1] = lines + 7
    accepted = torch.tensor([1, cols, 1, cols, cols + 9, 0], dtype=torch.int32)
    want, err, new, new_err = orc.update(x[0], a[0], b[0], lam, C, pool, table.tolist(),
                                         accepted.tolist(), list(range(0, n * T + 1, T)))
    cu = torch.arange(0, n * T + 1, T, dtype=torch.int32, device=dev)
    for api in _both().values():
        for ragged in (False, True):
            pd = pool.to(dev)
            shape = (1, n * T, D) if ragged else (n, T, D)
            y = api.npu_gated_linear_recurrence_update(
                *[t.view(shape).to(dev) for t in (x, a, b)], lam.to(dev), pd, C,
                table.to(torch.int32).to(dev), accepted.to(dev), cu if ragged else None)
            assert_within(y.reshape(n * T, D), want, err, "y")
            assert_within(pd, new, new_err, "pool")


def test_update_ragged_with_empty_sequences_and_rows_behind(dev):
    from torch_npu_ops_amd import _xk_torch as xt
    cu, D, total = [0, 2, 2, 5, 6], 34, 9
    x, a, b, _, lam, _, _ = _inputs(70, total, D, 4, BF16)
    pool = torch.randn(4, D, generator=_gen(5))
    want, err, new, new_err = orc.update(x[0], a[0], b[0], lam, C, pool, None, None, cu)
    pd = pool.to(dev)
    y = xt.npu_gated_linear_recurrence_update(
        x.to(dev), a.to(dev), b.to(dev), lam.to(dev), pd, C,
        cu_seqlens=torch.tensor(cu, dtype=torch.int64, device=dev))
    assert_within(y[0, :6], want[:6], err[:6], "y")
    assert_within(pd, new, new_err, "pool")
    assert torch.equal(pd[1].cpu(), pool[1])  # the empty sequence's slot


def test_update_strided_views_and_pool(dev):
    from torch_npu_ops_amd import _xk_torch as xt
    n, D = 5, 100
    x, a, b, _, lam, _, _ = _inputs(71, n, D, n, BF16)
    pool = torch.randn(n, D, generator=_gen(6))
    want, err, new, new_err = orc.update(x[0], a[0], b[0], lam, C, pool, None, None,
                                         list(range(n + 1)))
    ab = torch.cat([a[0], b[0]], -1).to(dev)
    wide = torch.zeros(n, D + 28, device=dev)
    wide[:, 3:3 + D] = pool.to(dev)
    y = xt.npu_gated_linear_recurrence_update(x[0].to(dev), ab[:, :D], ab[:, D:], lam.to(dev),
                                              wide[:, 3:3 + D])
    assert_within(y, want, err, "y")
    assert_within(wide[:, 3:3 + D], new, new_err, "pool")
    assert (wide[:, :3] == 0).all() and (wide[:, 3 + D:] == 0).all()


def test_update_many_sequences(dev):
    from torch_npu_ops_amd import _xk_torch as xt
    n, D = 70001, 6
    x, a, b, _, lam, _, _ = _inputs(72, n, D, 1, F32)
    pool = torch.randn(n, D, generator=_gen(7))
    pd = pool.to(dev)
    y = xt.npu_gated_linear_recurrence_update(x[0].to(dev), a[0].to(dev), b[0].to(dev),
                                              lam.to(dev), pd)
    r, i, ell, alpha, s = orc.gates(a[0], b[0], lam, C)
    want = alpha * pool.double() + s * i * x[0].double()
    torch.testing.assert_close(y.cpu().double(), want, rtol=3e-6, atol=3e-6)
    torch.testing.assert_close(pd.cpu().double(), want, rtol=3e-6, atol=3e-6)


def test_update_replayed_from_a_graph(dev):
    from torch_npu_ops_amd import _xk_torch as xt
    n, D = 9, 256
    x, a, b, _, lam, _, _ = (t.to(dev) for t in _inputs(73, n, D, n, BF16))
    pool = torch.randn(n, D, generator=_gen(8)).to(dev)
    eager, graphed = pool.clone(), pool.clone()
    slots = torch.arange(n, dtype=torch.int32, device=dev).flip(0).contiguous()
    args = (x[0], a[0], b[0], lam)
    xt.npu_gated_linear_recurrence_update(*args, pool.clone(), C, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = xt.npu_gated_linear_recurrence_update(*args, graphed, C, slots)
    graphed.copy_(pool)
    for k in range(4):
        want = xt.npu_gated_linear_recurrence_update(*args, eager, C, slots)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(graphed, eager)


def test_prefill_then_decode_equals_one_prefill(dev):
    from torch_npu_ops_amd import _xk_torch as xt
    T, more, D = 200, 5, 128
    x, a, b, _, lam, h0, _ = _inputs(80, T + more, D, 1, F32)
    d = [t.to(dev) for t in (x, a, b)]
    _, state, _ = xt.npu_gated_linear_recurrence(*[t[:, :T] for t in d], lam.to(dev), C,
                                                 h0.to(dev), True)
    ys = []
    for k in range(T, T + more):
        ys.append(xt.npu_gated_linear_recurrence_update(*[t[:, k] for t in d], lam.to(dev),
                                                        state, C))
    ref = orc.forward(x[0], a[0], b[0], lam, C, h0, [0, T + more])
    assert_within(torch.cat(ys), ref["h"][T:], ref["h_err"][T:], "y")
    assert_within(state, ref["final"], ref["final_err"], "state")


@pytest.mark.parametrize("T, D, dtype", [(2112, 8256, F32), (4112, 4100, BF16), (4099, 640, F32),
                                         (3000, 2047, F16), (2700, 1, BF16)], ids=str)
def test_many_tiles_of_either_length(dev, T, D, dtype):
    # More windows than the rule's limit for long tiles, and fewer.
    print(f"T={T} D={D} {dtype}", flush=True)
    _check(dev, _both()["cpp"], [T // 3, 0, 1, T - T // 3 - 1], D, dtype, seed=T)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("where", ["x", "a", "b", "h0"])
def test_a_value_that_is_not_finite_stays_in_its_channel_and_sequence(dev, where, value):
    from torch_npu_ops_amd import _xk_torch as xt
    T, D = 700, 131
    x, a, b, dy, lam, h0, df = _inputs(23, T, D, 2, BF16)
    cu = torch.tensor([0, 400, 700], dtype=torch.int32, device=dev)
    t = {"x": x, "a": a, "b": b, "h0": h0}

    def run():
        d = {k: v.to(dev) for k, v in t.items()}
        out = xt.npu_gated_linear_recurrence(d["x"], d["a"], d["b"], lam.to(dev), C, d["h0"], True, cu)
        return out[0][0].float().cpu()
    clean = run()
    if where == "h0":
        t["h0"][0, 64] = value
    else:
        t[where][0, 17, 64] = value
    got = run()
    kept = torch.ones_like(clean, dtype=torch.bool)
    kept[17 if where != "h0" else 0:400, 64] = False
    assert torch.equal(got[kept], clean[kept])
    if value != value:  # NaN reaches every later token of the sequence
        assert got[17:400, 64].isnan().all() and got[400:].isfinite().all()


@pytest.mark.parametrize("default", [BF16, torch.float64], ids=str)
def test_another_default_dtype(dev, default):
    print(f"default dtype {default}", flush=True)
    torch.set_default_dtype(default)
    try:
        x, a, b, dy, lam, h0, df = _inputs(90, 200, 72, 2, BF16)
        both = {}
        for name, api in _both().items():
            d = [t.to(dev) for t in (x, a, b, lam.float())]
            cu = torch.tensor([0, 70, 200], dtype=torch.int32, device=dev)
            y, fin, st = api.npu_gated_linear_recurrence(*d, C, None, True, cu, True)
            both[name] = [y, fin, st[1:4], *api.npu_gated_linear_recurrence_bwd(
                dy.to(dev), *d, st, C, None, None, cu)]
        assert all(torch.equal(p, q) and p.dtype == q.dtype
                   for p, q in zip(both["cpp"], both["py"]))
    finally:
        torch.set_default_dtype(torch.float32)


# ---------------------------------------------------------------------------
# values that are not finite
# ---------------------------------------------------------------------------
def _spoiled(dev, where, value, at, lens, lam=None):
    """The forward and backward call on clean inputs and on inputs with one
    value changed (channel 64; token `at`, for states the first sequence), and
    the oracle's results for the changed ones, by name."""
    from torch_npu_ops_amd import _xk_torch as xt
    cu, D = _cu(lens), 131
    x, a, b, dy, usual, h0, df = _inputs(23, cu[-1], D, len(lens), BF16)
    lam = usual if lam is None else torch.full((D,), lam)
    t = {"x": x, "a": a, "b": b, "dy": dy, "h0": h0, "df": df}
    cud = torch.tensor(cu, dtype=torch.int32, device=dev)

    def run():
        d = {k: v.to(dev) for k, v in t.items()}
        args = d["x"], d["a"], d["b"], lam.to(dev)
        y, fin, st = xt.npu_gated_linear_recurrence(*args, C, d["h0"], True, cud, True)
        out = xt.npu_gated_linear_recurrence_bwd(d["dy"], *args, st, C, d["h0"], d["df"], cud)
        names = ("y", "final", "dx", "da", "db", "dlam", "dh0")
        return {k: (v[0] if v.dim() == 3 else v).cpu() for k, v in zip(names, (y, fin, *out))}
    clean = run()
    if where in ("h0", "df"):
        t[where][0, 64] = value
    else:
        t[where][0, at, 64] = value
    fwd = orc.forward(x[0], a[0], b[0], lam, C, h0, cu)
    want = {"y": fwd["h"], "final": fwd["final"]}
    want.update(orc.backward(dy[0], x[0], a[0], b[0], lam, C, h0, df, cu))
    return clean, run(), want


def _same_but_for_what_is_not_finite(clean, got, want):
    """Elements that the formulas make NaN or infinite are that, all others
    have the clean call's bits."""
    for name, t in got.items():
        w = want[name]
        assert torch.equal(t.isnan(), w.isnan()), name
        inf = w.isinf()
        assert torch.equal(t[inf].double(), w[inf]), name
        kept = w.isfinite()
        assert torch.equal(t[kept], clean[name][kept]), name


@pytest.mark.parametrize("at", [0, 17, 31, 395, 399])
@pytest.mark.parametrize("where", ["x", "a", "b", "dy", "h0", "df"])
def test_a_nan_reaches_all_that_depends_on_it(dev, where, at):
    # Inside a window and at its ends, in the sequence's first and last window.
    clean, got, want = _spoiled(dev, where, float("nan"), at, [400, 300])
    if where == "b":  # dlam and da alone depend on what comes before a token
        assert want["dx"][at, 64].isnan() and want["dx"][at + 1:, 64].isfinite().all()
    assert want["dlam"][64].isnan()
    _same_but_for_what_is_not_finite(clean, got, want)


@pytest.mark.parametrize("value", [float("inf"), float("-inf")])
@pytest.mark.parametrize("where", ["x", "dy", "h0", "df"])
@pytest.mark.parametrize("lam", [-6.0, -0.5, 3.0])
@pytest.mark.parametrize("lens", [[9, 3], [400, 300]], ids=str)
def test_an_infinite_value_leaves_no_finite_one_that_depends_on_it(dev, lens, lam, where, value):
    # alpha near 1, around 0.15 and around 10^-5 (whose product over a window is 0).
    clean, got, want = _spoiled(dev, where, value, 5, lens, lam)
    if where in ("x", "h0"):
        assert want["y"][5:lens[0], 64].isinf().all()
    for name, t in got.items():
        kept = want[name].isfinite()
        assert torch.equal(t.isfinite(), kept), name
        assert torch.equal(t[kept], clean[name][kept]), name


@pytest.mark.parametrize("lam", [-6.0, -0.5, 3.0])
def test_update_of_an_infinite_state(dev, lam):
    from torch_npu_ops_amd import _xk_torch as xt
    x, a, b, _, _, pool, _ = _inputs(93, 4, 70, 4, BF16)
    args = [t[0].to(dev) for t in (x, a, b)] + [torch.full((70,), lam, device=dev)]
    clean = pool.to(dev)
    xt.npu_gated_linear_recurrence_update(*args, clean)
    pool[1, 3], pool[2, 5] = float("inf"), float("-inf")
    args[0][0, 7] = float("-inf")
    state = pool.to(dev)
    y = xt.npu_gated_linear_recurrence_update(*args, state)
    kept = torch.ones(4, 70, dtype=torch.bool, device=dev)
    kept[1, 3] = kept[2, 5] = kept[0, 7] = False
    assert torch.equal(state.isfinite(), kept) and torch.equal(y.isfinite(), kept)
    assert torch.equal(state[kept], clean[kept])


@pytest.mark.parametrize("a_value,b_value", [(-75.0, 0.5), (-85.0, 0.5), (0.5, -75.0), (0.5, -85.0),
                                             (-70.0, -10.0)])
def test_gradients_of_nearly_closed_gates(dev, a_value, b_value):
    # A sigmoid at v carries |v| + 2 u from its argument, 0.22 |v| u from the
    # constant log2 e and 4 u from the exponential, the sum and the reciprocal:
    # 1.3 |v| + 8 of them.  A gradient holds either gate at most twice.
    # Where l is no normal number, s^2 = 2 |l| is below 2^-125 and formed from
    # what is left of l's digits: s, at most 2^-62.5, is off by 2^-62 at most, and
    # so is l / s, which is s / 2 there.  dx = G i s, db = G i s x (1 - i) and
    # da = G (h l - i x l / s) (with alpha and 1 - r both 1) are off by that much
    # times what stands beside s; h l is below 2^-120.
    from torch_npu_ops_amd import _xk_torch as xt
    T, D = 40, 70
    x, _, _, dy, lam, h0, df = _inputs(94, T, D, 1, F32)
    a, b = torch.full((1, T, D), a_value), torch.full((1, T, D), b_value)
    d = [t.to(dev) for t in (x, a, b, lam)]
    st = xt.npu_gated_linear_recurrence(*d, C, h0.to(dev), False, None, True)[2]
    got = xt.npu_gated_linear_recurrence_bwd(dy.to(dev), *d, st, C, h0.to(dev), df.to(dev))
    want = orc.backward(dy[0], x[0], a[0], b[0], lam, C, h0, df, [0, T])
    more = 2 * (1.3 * (abs(a_value) + abs(b_value)) + 16) * orc.U
    _, i, ell, _, s = orc.gates(a[0], b[0], lam, C)
    tiny = (ell.abs() < 2.0 ** -126) * 2.0 ** -62 * (want["dx"] / s).abs()  # 2^-62 |G| i
    beside = {"dx": 1.0, "db": x[0].double().abs(), "da": x[0].double().abs() + 1.0}
    for name, t in zip(("dx", "da", "db", "dlam", "dh0"), got):
        t = t[0] if t.dim() == 3 else t
        room = want[name + "_err"] + more * want[name].abs()
        if name in beside:
            room = room + tiny * beside[name]
        if name == "dlam":
            room = room + (2 * more * want["da"].abs() + 2 * tiny * beside["da"]).sum(0)
        assert (want[name] != 0).all() and want[name].isfinite().all()
        assert_within(t, want[name], room, name)


def _strong(D):
    # With a = 0 a token keeps 10^-3 to 10^-9 of the state (and 0.8 to 0.9 for
    # every fourth channel, on the other side of the series).
    keep = 10.0 ** -torch.linspace(3, 9, D, dtype=torch.float64)
    keep[::4] = torch.linspace(0.8, 0.9, len(keep[::4]), dtype=torch.float64)
    return torch.log(torch.expm1(-torch.log(keep) / (C * 0.5))).float()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("first", [0, 13, 125, 1021])
def test_a_strong_decay_keeps_its_digits(dev, first, dtype):
    # Small inputs beside states of order 1: what is left of the state is seen.
    # Sequences start 3 tokens before a window's, a tile's or a group's end.
    lens, D = [3, 1, 2, 5, 40, 300], 70
    cu = _cu(lens, first)
    total = cu[-1] + 9
    x, a, b, dy, _, h0, df = _inputs(91, total, D, len(lens), F32)
    x, a, b, dy = ((t * f).to(dtype) for t, f in ((x, 1e-12), (a, 0), (b, 1), (dy, 1e-12)))
    lam = _strong(D)
    d = [t.to(dev) for t in (x, a, b, lam)]
    cud, m = torch.tensor(cu, dtype=torch.int32, device=dev), _live(cu, total)
    want = orc.forward(x[0], a[0], b[0], lam, C, h0, cu)
    grads = orc.backward(dy[0], x[0], a[0], b[0], lam, C, h0, df, cu)
    for api in _both().values():
        y, fin, st = api.npu_gated_linear_recurrence(*d, C, h0.to(dev), True, cud, True)
        assert_within(y[0].cpu()[m], want["h"][m], want["h_err"][m], "y")
        assert_within(fin, want["final"], want["final_err"], "final state")
        got = api.npu_gated_linear_recurrence_bwd(dy.to(dev), *d, st, C, h0.to(dev), df.to(dev),
                                                  cud)
        for name, t in zip(("dx", "da", "db"), got):
            assert_within(t[0].cpu()[m], grads[name][m], grads[name + "_err"][m], name)
        assert_within(got[3], grads["dlam"], grads["dlam_err"], "dlam")
        assert_within(got[4], grads["dh0"], grads["dh0_err"], "dh0")


@pytest.mark.parametrize("n", [3, 9000])
def test_update_under_a_strong_decay(dev, n):
    # Both numbers of channels a lane.
    from torch_npu_ops_amd import _xk_torch as xt
    D = 70
    x, a, b, _, _, pool, _ = _inputs(92, n, D, n, F32)
    x, a, lam = x * 1e-12, a * 0, _strong(D)
    r, i, ell, alpha, s = orc.gates(a[0], b[0], lam, C)
    add = s * i * x[0].double()
    want = alpha * pool.double() + add
    err = alpha * pool.abs() * orc.keep(ell) + add.abs() * orc.EPS + 2 * orc.U * want.abs()
    state = pool.to(dev)
    y = xt.npu_gated_linear_recurrence_update(x[0].to(dev), a[0].to(dev), b[0].to(dev),
                                              lam.to(dev), state)
    assert_within(y, want, err, "y")
    assert_within(state, want, err, "pool")


@pytest.mark.parametrize("which", ["cpp", "py"])
def test_rows_further_apart_than_a_tiles_offsets_reach(dev, which):
    # The last token of a batch of long prompts, and rows of 2^25 elements' pitch.
    api = _both()[which]
    B, D, pitch = 3, 72, (1 << 25) + 8
    x, a, b, dy, lam, h0, df = (t.to(dev) for t in _inputs(95, B, D, B, BF16))
    wide = torch.empty((B - 1) * pitch + D, dtype=BF16, device=dev)
    far = wide.as_strided((B, 1, D), (pitch, D, 1))
    far.copy_(x[0][:, None])
    pools = h0.clone(), h0.clone()
    cut = [t[0][:, None] for t in (x, a, b)]
    one = api.npu_gated_linear_recurrence_update(far, *cut[1:], lam, pools[0])
    two = api.npu_gated_linear_recurrence_update(*cut, lam, pools[1])
    assert torch.equal(one, two) and torch.equal(*pools)
    row = wide.as_strided((1, B, D), (D, pitch, 1))  # a sequence of B tokens
    y, fin, st = api.npu_gated_linear_recurrence(row, a, b, lam, C, h0[:1], True, None, True)
    same = api.npu_gated_linear_recurrence(x, a, b, lam, C, h0[:1], True, None, True)
    assert torch.equal(y, same[0]) and torch.equal(fin, same[1])
    far.copy_(dy[0][:, None])
    got = api.npu_gated_linear_recurrence_bwd(row, x, a, b, lam, st, C, h0[:1])
    want = api.npu_gated_linear_recurrence_bwd(dy, x, a, b, lam, st, C, h0[:1])
    assert all(torch.equal(p, q) for p, q in zip(got, want))
