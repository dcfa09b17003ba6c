"""CPU checks of the gated linear recurrence and the block-to-block norm: the
calls that are refused, by the C-ABI, the C++ API and its Python mirror,
before anything touches a GPU."""
import ctypes

import pytest
import torch

from torch_npu_ops_amd import _lib


@pytest.fixture(params=["cpp", "py"])
def api(request):
    from torch_npu_ops_amd import _xk_torch, ops
    return _xk_torch if request.param == "cpp" else ops


REFUSED = (RuntimeError, ValueError)
PTR = 1 << 20  # aligned, never read: the calls are refused first


def _glr(**change):
    v = dict(x=PTR, sx=64, a=PTR, sa=64, b=PTR, sb=64, dt=_lib.XK_BF16, lam=PTR, c=8.0, y=PTR,
             sy=64, h0=None, fin=None, states=None, cu=PTR, cdt=_lib.XK_I32, N=2, total=10, D=64,
             ws=None, size=0, stream=None)
    v.update(change)
    return _lib.lib().xk_gated_linear_recurrence(*v.values())


@pytest.mark.parametrize("change", [
    dict(N=-1), dict(total=-1), dict(D=0), dict(c=-1.0), dict(c=float("nan")), dict(x=None),
    dict(a=None), dict(b=None), dict(y=None), dict(lam=None), dict(sx=63), dict(sa=63),
    dict(sb=0), dict(sy=63), dict(cdt=_lib.XK_F32), dict(cu=None, N=3)], ids=str)
def test_recurrence_refuses(change):
    assert _glr(**change) == _lib.XK_ERR_INVALID


def test_recurrence_refuses_types_and_small_workspaces():
    assert _glr(dt=_lib.XK_I32) == _lib.XK_ERR_UNSUPPORTED
    assert _glr(N=0, cu=None, x=None) == _lib.XK_OK
    need = _lib.lib().xk_gated_linear_recurrence_workspace_bytes(100000, 64)
    if need > 0:
        assert _glr(total=100000) == _lib.XK_ERR_WORKSPACE
        assert _glr(total=100000, ws=PTR, size=need - 1) == _lib.XK_ERR_WORKSPACE
        assert _glr(total=100000, ws=PTR + 8, size=need) == _lib.XK_ERR_WORKSPACE


def _update(**change):
    v = dict(x=PTR, sx=64, a=PTR, sa=64, b=PTR, sb=64, dt=_lib.XK_BF16, lam=PTR, c=8.0, y=PTR,
             sy=64, state=PTR, ss=64, slots=4, idx=PTR, cols=0, acc=None, cu=None,
             cdt=_lib.XK_I32, N=2, T=1, total=2, D=64, stream=None)
    v.update(change)
    return _lib.lib().xk_gated_linear_recurrence_update(*v.values())


@pytest.mark.parametrize("change", [
    dict(N=-1), dict(D=0), dict(c=-0.5), dict(slots=-1), dict(cols=-1), dict(x=None),
    dict(lam=None), dict(state=None), dict(ss=63), dict(sx=1), dict(T=0), dict(T=2),
    dict(cols=2, idx=None), dict(cu=PTR, cdt=_lib.XK_F16)], ids=str)
def test_update_refuses(change):
    assert _update(**change) == _lib.XK_ERR_INVALID


def test_update_refuses_types_and_takes_no_work():
    assert _update(dt=_lib.XK_I64) == _lib.XK_ERR_UNSUPPORTED
    assert _update(N=0) == _lib.XK_OK


def _bwd(**change):
    v = dict(dy=PTR, sdy=64, x=PTR, sx=64, a=PTR, sa=64, b=PTR, sb=64, dt=_lib.XK_BF16, lam=PTR,
             c=8.0, states=PTR, h0=None, df=None, dx=PTR, sdx=64, da=PTR, sda=64, db=PTR, sdb=64,
             dlam=PTR, dh0=PTR, cu=PTR, cdt=_lib.XK_I32, N=2, total=10, D=64, ws=PTR,
             size=1 << 30, stream=None)
    v.update(change)
    return _lib.lib().xk_gated_linear_recurrence_bwd(*v.values())


@pytest.mark.parametrize("change", [
    dict(N=-1), dict(D=-4), dict(c=-1.0), dict(dy=None), dict(states=None), dict(dx=None),
    dict(da=None), dict(db=None), dict(lam=None), dict(sdy=63), dict(sdx=63), dict(sda=63),
    dict(sdb=63), dict(cu=None, N=3), dict(cdt=_lib.XK_BF16)], ids=str)
def test_backward_refuses(change):
    assert _bwd(**change) == _lib.XK_ERR_INVALID


def test_backward_refuses_small_workspaces():
    need = _lib.lib().xk_gated_linear_recurrence_bwd_workspace_bytes(10, 2, 64)
    assert need > 0
    assert _bwd(ws=None) == _lib.XK_ERR_WORKSPACE
    assert _bwd(size=need - 1) == _lib.XK_ERR_WORKSPACE
    assert _bwd(ws=PTR + 4) == _lib.XK_ERR_WORKSPACE
    assert _bwd(dt=_lib.XK_I32) == _lib.XK_ERR_UNSUPPORTED


def _norm(**change):
    v = dict(x=PTR, sx=64, res=PTR, sr=64, gate=PTR, sg=64, post=PTR, scale=PTR, pre=PTR, h=PTR,
             sh=64, y=PTR, sy=64, r1=None, r2=None, M=4, N=64, eps=1e-6, off=0,
             dt=_lib.XK_BF16, rdt=_lib.XK_F32, wdt=_lib.XK_BF16, stream=None)
    v.update(change)
    return _lib.lib().xk_gated_residual_rms_norm(*v.values())


@pytest.mark.parametrize("change", [
    dict(M=-1), dict(N=0), dict(eps=-1.0), dict(x=None), dict(res=None), dict(h=None),
    dict(y=None), dict(sx=63), dict(sr=63), dict(sg=63), dict(sh=0), dict(sy=63)], ids=str)
def test_norm_refuses(change):
    assert _norm(**change) == _lib.XK_ERR_INVALID


def test_norm_refuses_types_and_takes_no_rows():
    assert _norm(dt=_lib.XK_I32) == _lib.XK_ERR_UNSUPPORTED
    assert _norm(rdt=_lib.XK_F16) == _lib.XK_ERR_UNSUPPORTED
    assert _norm(wdt=_lib.XK_F16) == _lib.XK_ERR_UNSUPPORTED
    assert _norm(M=0, x=None) == _lib.XK_OK


def _norm_bwd(**change):
    v = dict(dh=PTR, sdh=64, dy=PTR, sdy=64, x=PTR, sx=64, res=PTR, sr=64, gate=PTR, sg=64,
             post=PTR, scale=PTR, pre=PTR, r1=PTR, r2=PTR, dx=PTR, sdx=64, dres=PTR, sdr=64,
             dgate=PTR, sdg=64, dpost=PTR, dscale=PTR, dpre=PTR, M=4, N=64, off=0,
             dt=_lib.XK_BF16, rdt=_lib.XK_F32, wdt=_lib.XK_BF16, ws=PTR, size=1 << 30,
             stream=None)
    v.update(change)
    return _lib.lib().xk_gated_residual_rms_norm_bwd(*v.values())


@pytest.mark.parametrize("change", [
    dict(M=-1), dict(N=0), dict(x=None), dict(res=None), dict(dh=None, dy=None), dict(r1=None),
    dict(r2=None), dict(post=None), dict(scale=None), dict(pre=None), dict(gate=None),
    dict(sdh=63), dict(sdy=63), dict(sx=63), dict(sdx=63), dict(sdr=63), dict(sdg=63)], ids=str)
def test_norm_backward_refuses(change):
    assert _norm_bwd(**change) == _lib.XK_ERR_INVALID


def test_norm_backward_refuses_small_workspaces():
    need = _lib.lib().xk_gated_residual_rms_norm_bwd_workspace_bytes(4, 64)
    assert need > 0
    assert _norm_bwd(ws=None) == _lib.XK_ERR_WORKSPACE
    assert _norm_bwd(size=need - 1) == _lib.XK_ERR_WORKSPACE
    assert _norm_bwd(ws=PTR + 16) == _lib.XK_ERR_WORKSPACE


# ---------------------------------------------------------------------------
# the torch-level calls
# ---------------------------------------------------------------------------
def _x(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_recurrence_arguments(api):
    x, lam = _x(1, 6, 8), torch.zeros(8)
    f = api.npu_gated_linear_recurrence
    for args, match in [
            ((x[0], x[0], x[0], lam), "expects x"),
            ((x, x[:, :5], x, lam), "a must have"),
            ((x, x, x.float(), lam), "b must have"),
            ((x.long(), x.long(), x.long(), lam), "float32, bfloat16 or float16"),
            ((x, x, x, lam.bfloat16()), "lam must be"),
            ((x, x, x, lam[:7]), "lam must be"),
            ((x, x, x, lam, -1.0), "c must be"),
            ((x, x, x, lam, float("inf")), "c must be")]:
        with pytest.raises(REFUSED, match=match):
            f(*args)
    with pytest.raises(RuntimeError, match="GPU device"):
        f(x, x, x, lam)


def test_update_arguments(api):
    x, lam, pool = _x(3, 8), torch.zeros(8), torch.zeros(4, 8)
    idx = torch.zeros(3, dtype=torch.int32)
    f = api.npu_gated_linear_recurrence_update
    for args, match in [
            ((x[None, None],) * 3 + (lam, pool), "expects x"),
            ((x, x, x, lam, pool.bfloat16()), "state must be float32"),
            ((x, x, x, lam, pool[:, :7]), "state must be float32"),
            ((x, x, x, lam, torch.zeros(8, 4).t()), "contiguous channels"),
            ((x, x, x, lam, pool[:2]), "a slot for every sequence"),
            ((x, x, x, lam, pool, 8.0, idx.long()), "state_indices must be int32"),
            ((x, x, x, lam, pool, 8.0, idx[:2]), "state_indices must be int32"),
            ((x, x, x, lam, pool, 8.0, idx, idx), "needs state_indices"),
            ((x, x, x, lam, pool, 8.0, idx[:, None], idx[:2]), "num_accepted_tokens must be"),
            ((x, x, x, lam, pool, 8.0, idx, None, torch.zeros(4)), "cu_seqlens must be")]:
        with pytest.raises(REFUSED, match=match):
            f(*args)
    with pytest.raises(RuntimeError, match="GPU device"):
        f(x, x, x, lam, pool)


def test_backward_arguments(api):
    x, lam, st = _x(1, 20, 8), torch.zeros(8), torch.zeros(2, 8)
    f = api.npu_gated_linear_recurrence_bwd
    for args, match in [
            ((x[:, :5], x, x, x, lam, st), "dy must have"),
            ((x.float(), x, x, x, lam, st), "dy must have"),
            ((x, x, x, x, lam, st[:1]), "states must be"),
            ((x, x, x, x, lam, st.double()), "states must be")]:
        with pytest.raises(REFUSED, match=match):
            f(*args)


def test_norm_arguments(api):
    x, w = _x(3, 8), torch.ones(8, dtype=torch.bfloat16)
    f = api.npu_gated_residual_rms_norm
    for args, match in [
            ((x, x[:2]), "residual must have"),
            ((x, x.half()), "residual must have"),
            ((x.long(), x.long()), "float32, bfloat16 or float16"),
            ((x, x, w[:7]), "post_weight must be"),
            ((x, x, w.half()), "post_weight must have"),
            ((x, x, w, x.float()), "gate must have"),
            ((x, x, w, None, w.float()), "one dtype"),
            ((x, x, w, None, None, w, -1.0), "eps must not")]:
        with pytest.raises(REFUSED, match=match):
            f(*args)
    with pytest.raises(RuntimeError, match="GPU device"):
        f(x, x)


def test_norm_backward_arguments(api):
    x, w, r = _x(3, 8), torch.ones(8, dtype=torch.bfloat16), torch.ones(3)
    f = api.npu_gated_residual_rms_norm_bwd
    for args, match in [
            ((None, None, x, x, r, r, w, None, None, w), "needs dh or dy"),
            ((x, x, x, x, r, r), "dy needs pre_weight"),
            ((x.float(), None, x, x, r, r), "dh must have"),
            ((None, x[:2], x, x, r, r, None, None, None, w), "dy must have"),
            ((x, None, x, x, None, r, w), "rstd_post must be"),
            ((x, x, x, x, r, r[:2], w, None, None, w), "rstd_pre must be")]:
        with pytest.raises(REFUSED, match=match):
            f(*args)


def test_entry_points_are_operations_too():
    # The C symbols that csrc/torch_api/operations.h binds.
    lib = _lib.lib()
    for name in ("xk_gated_linear_recurrence", "xk_gated_linear_recurrence_update",
                 "xk_gated_linear_recurrence_bwd", "xk_gated_residual_rms_norm",
                 "xk_gated_residual_rms_norm_bwd"):
        assert ctypes.cast(getattr(lib, name), ctypes.c_void_p).value


def test_sizes_that_no_launch_holds_are_refused():
    # A launch has fewer than 2^32 threads, a pitch fewer than 2^25 elements.
    wide = dict(sx=1 << 26, sa=1 << 26, sb=1 << 26)
    for call, more in ((_glr, dict(sy=1 << 26)), (_bwd, dict(sdy=1 << 26, sdx=1 << 26,
                                                              sda=1 << 26, sdb=1 << 26))):
        assert call(total=1 << 30, size=1 << 62, ws=PTR) == _lib.XK_ERR_INVALID
        assert call(total=1 << 20, D=64 << 10, size=1 << 62, ws=PTR, **wide,
                    **more) == _lib.XK_ERR_INVALID
        assert call(total=0, D=1 << 25, size=1 << 62, ws=PTR) == _lib.XK_ERR_INVALID
        assert call(sx=1 << 25) == _lib.XK_ERR_INVALID
    assert _update(sy=1 << 25) == _lib.XK_ERR_INVALID
    assert _update(N=1 << 26, total=1 << 26) == _lib.XK_ERR_INVALID
    lib = _lib.lib()
    for total, D in ((1 << 30, 64), (1 << 20, 64 << 10), (16, 1 << 25), (-1, 64), (16, 0)):
        assert lib.xk_gated_linear_recurrence_workspace_bytes(total, D) == 0
        assert lib.xk_gated_linear_recurrence_bwd_workspace_bytes(total, 1, D) == 0
    # The largest that are taken: the workspace of 2^35 elements.
    assert lib.xk_gated_linear_recurrence_workspace_bytes(1 << 23, 1 << 12) > 0
    assert _norm(M=1, N=1 << 28) == _lib.XK_ERR_INVALID
    assert _norm_bwd(M=1, N=1 << 28, size=1 << 62) == _lib.XK_ERR_INVALID
    assert lib.xk_gated_residual_rms_norm_bwd_workspace_bytes(1, 1 << 28) == 0
    assert lib.xk_gated_residual_rms_norm_bwd_workspace_bytes(1, (1 << 28) - 1) > 0


def _documented_limits():
    """(n, p): the header's (ceil(total_tokens / 16) + n) * ceil(D / 64) < 2^p."""
    import pathlib
    import re
    path = pathlib.Path(__file__).parents[1] / "include" / "xk_ops.h"
    text = re.sub(r"\s*\n \*\s*", " ", path.read_text())
    at = re.search(r"\(ceil\(total_tokens / 16\) \+ (\d+)\) \* ceil\(D / 64\) must be below 2\^(\d+)",
                   text)
    return int(at[1]), int(at[2])


@pytest.mark.parametrize("D", [64, 65, 1000, 4096])
def test_the_documented_sizes_are_the_ones_that_are_taken(D):
    more, power = _documented_limits()
    lib = _lib.lib()
    blocks = -(-D // 64)
    windows = -(-(1 << power) // blocks) - more  # the first count of windows that is refused
    size = (lib.xk_gated_linear_recurrence_workspace_bytes,
            lambda t, d: lib.xk_gated_linear_recurrence_bwd_workspace_bytes(t, 1, d))
    for f in size:
        assert f((windows - 1) * 16, D) > 0
        assert f((windows - 1) * 16 + 1, D) == 0
    refused = dict(total=(windows - 1) * 16 + 1, D=D, size=1 << 62, ws=PTR)
    wide = dict.fromkeys(("sx", "sa", "sb", "sy"), D)
    assert _glr(**refused, **wide) == _lib.XK_ERR_INVALID
    # Taken as far as the workspace, which is missing.
    assert _glr(**{**refused, **wide, "total": (windows - 1) * 16, "ws": None}) == \
        _lib.XK_ERR_WORKSPACE


@pytest.mark.parametrize("call", [_glr, _update, _bwd])
def test_an_infinite_c_is_refused(call):
    assert call(c=float("inf")) == _lib.XK_ERR_INVALID


def test_a_c_that_is_infinite_in_fp32_is_refused(api):
    x, lam, pool = _x(1, 6, 8), torch.zeros(8), torch.zeros(6, 8)
    for c in (1e39, float("inf")):
        with pytest.raises(REFUSED, match="c must be"):
            api.npu_gated_linear_recurrence(x, x, x, lam, c)
        with pytest.raises(REFUSED, match="c must be"):
            api.npu_gated_linear_recurrence_update(x[0], x[0], x[0], lam, pool, c)
        with pytest.raises(REFUSED, match="c must be"):
            api.npu_gated_linear_recurrence_bwd(x, x, x, x, lam, torch.zeros(1, 8), c)
