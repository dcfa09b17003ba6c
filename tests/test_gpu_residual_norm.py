"""GPU checks of the block-to-block norm (RMSNorm, gate, residual scale,
residual sum, RMSNorm) and its gradients against oracle/residual_norm.py in
float64.  Tolerances: the oracle's bound of the fp32 arithmetic plus half a
step of the output's type (rounding_tol.py)."""
import itertools

import pytest
import torch

from oracle import residual_norm as orn
from rounding_tol import assert_within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-6
WEIGHTS = ("post", "scale", "pre")


def _both():
    from torch_npu_ops_amd import _xk_torch, ops
    return {"cpp": _xk_torch, "py": ops}


def _inputs(seed, M, N, dtype, rdtype=None, wdtype=None, parts=("post", "gate", "scale", "pre")):
    g = torch.Generator().manual_seed(seed)
    rdtype, wdtype = rdtype or dtype, wdtype or dtype

    def r(*s, dt, std=1.0, mean=0.0):
        return (torch.randn(*s, generator=g).clamp_(-8, 8) * std + mean).to(dt)
    p = {"x": r(M, N, dt=dtype), "res": r(M, N, dt=rdtype, std=2.0),
         "post": r(N, dt=wdtype, std=0.1, mean=1.0), "gate": r(M, N, dt=dtype),
         "scale": r(N, dt=wdtype, std=0.1, mean=0.5),
         "pre": r(N, dt=wdtype, std=0.1, mean=1.0), "dh": r(M, N, dt=rdtype),
         "dy": r(M, N, dt=dtype)}
    for k in ("post", "gate", "scale", "pre"):
        if k not in parts:
            p[k] = None
    if p["pre"] is None:
        p["dy"] = None
    return p


def _dev(p, dev):
    return {k: None if v is None else v.to(dev) for k, v in p.items()}


def _args(p):
    return [p[k] for k in ("x", "res", "post", "gate", "scale", "pre")]


def _run(api, d, offset=False):
    h, y, r1, r2 = api.npu_gated_residual_rms_norm(*_args(d), EPS, offset)
    grads = api.npu_gated_residual_rms_norm_bwd(d["dh"], d["dy"], d["x"], d["res"], r1, r2,
                                                d["post"], d["gate"], d["scale"], d["pre"],
                                                offset)
    return h, y, r1, r2, dict(zip(("dx", "dres", "dgate", "dpost", "dscale", "dpre"), grads))


def _check(api, p, dev, offset=False):
    d = _dev(p, dev)
    h, y, r1, r2, grads = _run(api, d, offset)
    o = orn.forward(*_args(p), EPS, offset)
    assert h.dtype == p["res"].dtype
    assert_within(h, o["h"], o["h_err"], "h")
    if p["pre"] is None:
        assert y is None and r2 is None
    else:
        assert_within(y, o["y"], o["y_err"], "y")
        assert_within(r2, o["r2"][:, 0], (o["r2"] * (o["r2_rel"] + 4 * orn.U))[:, 0], "rstd_pre")
    if p["post"] is None:
        assert r1 is None
    else:
        assert_within(r1, o["r1"][:, 0], o["r1"][:, 0] * (orn.SUM + 4 * orn.U), "rstd_post")
    want = orn.backward(p["dh"], p["dy"], *_args(p), EPS, offset)
    for k, t in grads.items():
        if k not in want:
            assert t is None, k
            continue
        assert t.dtype == p[k[1:]].dtype
        assert_within(t, want[k], want[k + "_err"], k)


@pytest.mark.parametrize("parts", [c for n in range(5) for c in
                                   itertools.combinations(("post", "gate", "scale", "pre"), n)],
                         ids="+".join)
@pytest.mark.parametrize("which", ["cpp", "py"])
def test_parts(dev, which, parts):
    print(which, parts, flush=True)
    _check(_both()[which], _inputs(len(parts), 9, 264, BF16, parts=parts), dev)


TYPES = [(BF16, BF16, BF16), (BF16, F32, BF16), (BF16, BF16, F32), (BF16, F32, F32),
         (F16, F16, F16), (F16, F32, F32), (F32, F32, F32)]


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("N", [1, 3, 8, 100, 515, 1024, 2050, 4096])
def test_widths_and_types(dev, N, types):
    print(N, types, flush=True)
    _check(_both()["cpp"], _inputs(N, 5, N, *types), dev)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N", [5000, 8192, 8200, 16384, 20001, 33000])
def test_wide_rows(dev, N, dtype):
    print(N, dtype, flush=True)
    _check(_both()["cpp"], _inputs(N, 3, N, dtype), dev)


@pytest.mark.parametrize("M", [1, 2, 255, 513, 2051])
@pytest.mark.parametrize("N", [96, 1200])
def test_rows(dev, M, N):
    print(M, N, flush=True)
    _check(_both()["cpp"], _inputs(M, M, N, BF16), dev)


def test_many_rows(dev):
    _check(_both()["cpp"], _inputs(1, 9000, 72, F16, F32), dev)


@pytest.mark.parametrize("which", ["cpp", "py"])
def test_unit_offset(dev, which):
    _check(_both()[which], _inputs(2, 7, 320, BF16), dev, offset=True)


@pytest.mark.parametrize("which", ["cpp", "py"])
def test_missing_gradients(dev, which):
    api = _both()[which]
    p = _inputs(3, 11, 200, BF16)
    d = _dev(p, dev)
    _, _, r1, r2 = api.npu_gated_residual_rms_norm(*_args(d), EPS)
    for dh, dy in (("dh", None), (None, "dy")):
        got = api.npu_gated_residual_rms_norm_bwd(
            d[dh] if dh else None, d[dy] if dy else None, d["x"], d["res"], r1, r2, d["post"],
            d["gate"], d["scale"], d["pre"])
        want = orn.backward(p[dh] if dh else None, p[dy] if dy else None, *_args(p), EPS)
        for k, t in zip(("dx", "dres", "dgate", "dpost", "dscale", "dpre"), got):
            assert_within(t, want[k], want[k + "_err"], k)
        if dy is None:
            assert (got[5] == 0).all()


def test_wide_rows_with_missing_parts(dev):
    api = _both()["cpp"]
    for parts in ((), ("post",), ("gate", "pre"), ("scale",)):
        _check(api, _inputs(4, 2, 33001, BF16, parts=parts), dev)
    p = _inputs(5, 3, 33001, BF16)
    d = _dev(p, dev)
    _, _, r1, r2 = api.npu_gated_residual_rms_norm(*_args(d), EPS)
    got = api.npu_gated_residual_rms_norm_bwd(d["dh"], None, d["x"], d["res"], r1, r2, d["post"],
                                              d["gate"], d["scale"], d["pre"])
    want = orn.backward(p["dh"], None, *_args(p), EPS)
    for k, t in zip(("dx", "dres", "dgate", "dpost", "dscale", "dpre"), got):
        assert_within(t, want[k], want[k + "_err"], k)


def test_no_rows(dev):
    for api in _both().values():
        d = _dev(_inputs(6, 0, 40, BF16), dev)
        h, y, r1, r2, grads = _run(api, d)
        assert h.shape == (0, 40) and y.shape == (0, 40) and r1.shape == (0,)
        assert all((grads[k] == 0).all() for k in ("dpost", "dscale", "dpre"))


def test_leading_dims(dev):
    p = _inputs(7, 24, 48, BF16)
    d = _dev(p, dev)
    want = _run(_both()["cpp"], d)
    cube = {k: v.view(2, 3, 4, 48) if v is not None and v.dim() == 2 else v for k, v in d.items()}
    for api in _both().values():
        h, y, r1, r2, grads = _run(api, cube)
        assert h.shape == (2, 3, 4, 48) and r1.shape == (2, 3, 4)
        assert torch.equal(h.view(24, 48), want[0]) and torch.equal(y.view(24, 48), want[1])
        assert torch.equal(grads["dx"].view(24, 48), want[4]["dx"])
    one = {k: v[0] if v is not None and v.dim() == 2 else v for k, v in d.items()}
    h, y, *_ = _run(_both()["cpp"], one)
    assert h.shape == (48,) and torch.equal(h, want[0][0])


@pytest.mark.parametrize("form", ["slice", "odd_start", "every_other", "column_major", "expanded"])
@pytest.mark.parametrize("N", [64, 515])
def test_views_equal_contiguous_copies(dev, form, N):
    M = 10

    def view(t):
        if t is None or t.dim() == 1:
            return t
        if form in ("slice", "odd_start"):
            at = 8 if form == "slice" else 1
            wide = torch.randn(M, N + 29, device=dev).to(t.dtype)
            wide[:, at:at + N] = t
            return wide[:, at:at + N]
        if form == "every_other":
            wide = torch.randn(2 * M, N, device=dev).to(t.dtype)
            wide[::2] = t
            return wide[::2]
        if form == "column_major":
            return t.t().contiguous().t()
        return t[:1].expand(M, N)
    d = {k: view(v) for k, v in _dev(_inputs(8, M, N, BF16, F32), dev).items()}
    flat = {k: None if v is None else v.contiguous() for k, v in d.items()}
    for api in _both().values():
        one, two = _run(api, d), _run(api, flat)
        assert all(torch.equal(p, q) for p, q in zip(one[:4], two[:4]))
        assert all(torch.equal(one[4][k], two[4][k]) for k in one[4])


@pytest.mark.parametrize("N", [200, 4096, 33000])
def test_a_row_that_is_not_finite_stays_alone(dev, N):
    api = _both()["cpp"]
    d = _dev(_inputs(9, 6, N, BF16), dev)
    want = _run(api, d)
    for k, bad in (("x", float("nan")), ("res", float("inf")), ("gate", -float("inf"))):
        spoiled = {q: None if v is None else v.clone() for q, v in d.items()}
        spoiled[k][2, 5] = bad
        h, y, _, _, grads = _run(api, spoiled)
        keep = [0, 1, 3, 4, 5]
        assert torch.equal(h[keep], want[0][keep]) and torch.equal(y[keep], want[1][keep])
        for g in ("dx", "dres", "dgate"):
            assert torch.equal(grads[g][keep], want[4][g][keep])


def test_outputs_over_inputs(dev):
    """The C-ABI: h over residual, y over x or gate, at every kind of width."""
    from torch_npu_ops_amd import _lib
    lib = _lib.lib()
    for N in (130, 3000, 9000, 33000):
        d = _dev(_inputs(10, 4, N, BF16), dev)
        h, y, _, _, _ = _run(_both()["cpp"], d)
        for over in ("x", "gate"):
            c = {k: v.clone() for k, v in d.items()}
            st = lib.xk_gated_residual_rms_norm(
                c["x"].data_ptr(), N, c["res"].data_ptr(), N, c["gate"].data_ptr(), N,
                c["post"].data_ptr(), c["scale"].data_ptr(), c["pre"].data_ptr(),
                c["res"].data_ptr(), N, c[over].data_ptr(), N, None, None, 4, N, EPS, 0,
                _lib.XK_BF16, _lib.XK_BF16, _lib.XK_BF16,
                torch.cuda.current_stream().cuda_stream)
            assert st == _lib.XK_OK
            assert torch.equal(c["res"], h) and torch.equal(c[over], y)


def test_rows_beyond_32_bits(dev):
    # Rows one pitch of 2^30 elements apart: the last starts at element 2^31.
    p = _inputs(11, 3, 96, BF16)
    d = _dev(p, dev)
    want = _run(_both()["cpp"], d)
    wide = torch.empty(2 * (1 << 30) + 96, dtype=BF16, device=dev)
    view = wide.as_strided((3, 96), (1 << 30, 1))
    view.copy_(d["x"])
    got = _run(_both()["cpp"], {**d, "x": view})
    assert all(torch.equal(a, b) for a, b in zip(got[:4], want[:4]))
    assert all(torch.equal(got[4][k], want[4][k]) for k in want[4])


def test_gradients_against_differences(dev):
    # fp32 on the device; a directional difference of a sum of 600 products is
    # off by its rounding (600 * 2^-24 * 10 / 2e-2 = 2e-2 at the very worst,
    # in practice its root) and the cubic term: 5e-3 of values of order 10.
    api = _both()["cpp"]
    d = _dev(_inputs(12, 6, 100, F32), dev)
    _, _, _, _, grads = _run(api, d)

    def loss(q):
        h, y, _, _ = api.npu_gated_residual_rms_norm(*_args(q), EPS)
        return float((h.double() * d["dh"]).sum() + (y.double() * d["dy"]).sum())
    g = torch.Generator().manual_seed(13)
    for k in ("x", "res", "post", "gate", "scale", "pre"):
        way = torch.randn(d[k].shape, generator=g).to(dev)
        way /= way.norm()
        ends = [loss({**d, k: d[k] + s * 1e-2 * way}) for s in (1, -1)]
        got = float((grads["d" + k].double() * way).sum())
        assert got == pytest.approx((ends[0] - ends[1]) / 2e-2, rel=5e-3, abs=5e-3)


def test_same_bits_two_streams_and_graph(dev):
    api = _both()["cpp"]
    sets = [_dev(_inputs(20 + k, 3000, 1000, BF16), dev) for k in range(2)]
    want = [_run(api, d) for d in sets]
    torch.cuda.synchronize()

    def same(a, b):
        return (all(torch.equal(p, q) for p, q in zip(a[:4], b[:4]))
                and all(torch.equal(a[4][k], b[4][k]) for k in a[4]))
    outs = [[], []]
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[k].append(_run(api, sets[k]))
    torch.cuda.synchronize()
    assert all(same(out, want[k]) for k in range(2) for out in outs[k])
    graph = torch.cuda.CUDAGraph()
    d = sets[0]
    with torch.cuda.graph(graph):
        out = _run(api, d)
    for k in range(4):
        d["x"].copy_(torch.randn(3000, 1000, generator=torch.Generator().manual_seed(k)))
        eager = _run(api, d)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, eager)


@pytest.mark.parametrize("N", [7, 1025, 1027, 1031, 2051, 4101, 8195])
def test_output_over_residual_where_a_row_ends_inside_a_vector(dev, N):
    # The last lane reads elements that another wave writes; without the first
    # norm no barrier stands between.  Around the rows everything stays.
    from torch_npu_ops_amd import _lib
    M, pitch = 37, N + 5
    p = _inputs(N, M, N, BF16, parts=("scale", "pre"))
    d = _dev(p, dev)
    h, y, _, _ = _both()["cpp"].npu_gated_residual_rms_norm(*_args(d), EPS)
    buf = torch.full((M, pitch), 3.0, dtype=BF16, device=dev)
    out = buf.clone()
    buf[:, :N] = d["res"]
    st = _lib.lib().xk_gated_residual_rms_norm(
        d["x"].data_ptr(), N, buf.data_ptr(), pitch, None, 0, None, d["scale"].data_ptr(),
        d["pre"].data_ptr(), buf.data_ptr(), pitch, out.data_ptr(), pitch, None, None, M, N, EPS, 0,
        _lib.XK_BF16, _lib.XK_BF16, _lib.XK_BF16, torch.cuda.current_stream().cuda_stream)
    assert st == _lib.XK_OK
    assert torch.equal(buf[:, :N], h) and torch.equal(out[:, :N], y)
    assert (buf[:, N:] == 3.0).all() and (out[:, N:] == 3.0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N", [1, 3, 5, 9, 15, 17, 519, 1023, 1029, 2057])
def test_every_remainder_of_a_vector(dev, N, dtype):
    p = _inputs(N, 11, N, dtype, rdtype=F32)
    _check(_both()["cpp"], p, dev)


@pytest.mark.parametrize("dtype, rdtype", [(BF16, BF16), (BF16, F32), (F32, F32)], ids=str)
@pytest.mark.parametrize("vectors", [257, 384, 385, 513, 700, 768, 769, 1000, 1025, 1500, 1537])
def test_teams_of_every_size(dev, vectors, dtype, rdtype):
    N = vectors * (16 // dtype.itemsize)
    for n in (N, N - 3):
        _check(_both()["cpp"], _inputs(vectors, 5, n, dtype, rdtype=rdtype), dev)
