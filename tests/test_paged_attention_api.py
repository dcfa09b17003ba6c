"""CPU checks of rotary positions, the paged cache and the attention over it:
the calls that are refused, by the C-ABI, the C++ API and its Python mirror,
before anything touches a GPU."""
import pytest
import torch

from torch_npu_ops_amd import _lib

PTR = 1 << 20  # aligned, never read: the calls are refused first
REFUSED = (RuntimeError, ValueError)
INVALID, UNSUPPORTED = _lib.XK_ERR_INVALID, _lib.XK_ERR_UNSUPPORTED


@pytest.fixture(params=["cpp", "py"])
def api(request):
    from torch_npu_ops_amd import _xk_torch, ops
    return _xk_torch if request.param == "cpp" else ops


def _rotary(**change):
    v = dict(q=PTR, qt=512, qh=64, qo=PTR, qot=512, qoh=64, Hq=8, k=PTR, kt=128, kh=64, ko=PTR,
             kot=128, koh=64, Hk=2, pos=PTR, pdt=_lib.XK_I64, freq=PTR, rot=64, inter=0,
             scale=1.0, inverse=0, T=4, D=64, dt=_lib.XK_BF16, stream=None)
    v.update(change)
    return _lib.lib().xk_rotary_embedding(*v.values())


@pytest.mark.parametrize("change,status", [
    (dict(T=-1), INVALID), (dict(D=0), INVALID), (dict(D=513), INVALID), (dict(rot=63), INVALID),
    (dict(rot=66), INVALID), (dict(rot=0), INVALID), (dict(rot=-2), INVALID),
    (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(Hq=-1), INVALID), (dict(Hk=4097), INVALID),
    (dict(q=None), INVALID), (dict(qo=None), INVALID), (dict(k=None), INVALID),
    (dict(ko=None), INVALID), (dict(pos=None), INVALID), (dict(freq=None), INVALID),
    (dict(pdt=_lib.XK_F32), UNSUPPORTED), (dict(dt=_lib.XK_I32), UNSUPPORTED),
    (dict(dt=_lib.XK_F8E4M3), UNSUPPORTED), (dict(T=0, q=None), _lib.XK_OK),
    (dict(Hq=0, Hk=0), _lib.XK_OK)], ids=str)
def test_rotary_refuses(change, status):
    assert _rotary(**change) == status


def _append(**change):
    v = dict(q=PTR, qt=512, qh=64, qo=PTR, qot=512, qoh=64, Hq=8, k=PTR, kt=128, kh=64, v=PTR,
             vt=128, vh=64, Hkv=2, kc=PTR, kcp=2048, kcs=128, kch=64, vc=PTR, vcp=2048, vcs=128,
             vch=64, cdt=_lib.XK_BF16, pages=4, page=16, slots=PTR, sdt=_lib.XK_I64, pos=PTR,
             pdt=_lib.XK_I64, freq=PTR, rot=64, inter=0, scale=1.0, ks=None, vs=None, T=4, D=64,
             dt=_lib.XK_BF16, stream=None)
    v.update(change)
    return _lib.lib().xk_rotary_cache_append(*v.values())


@pytest.mark.parametrize("change,status", [
    (dict(T=-1), INVALID), (dict(D=0), INVALID), (dict(rot=65), INVALID), (dict(rot=0), INVALID),
    (dict(Hkv=0), INVALID), (dict(Hq=4097), INVALID), (dict(pages=-1), INVALID),
    (dict(page=0), INVALID), (dict(pages=1 << 62, page=4), INVALID), (dict(k=None), INVALID),
    (dict(v=None), INVALID), (dict(slots=None), INVALID), (dict(kc=None), INVALID),
    (dict(vc=None), INVALID), (dict(q=None), INVALID), (dict(freq=None), INVALID),
    (dict(ks=PTR), INVALID), (dict(vs=PTR), INVALID), (dict(cdt=_lib.XK_F16), UNSUPPORTED),
    (dict(cdt=_lib.XK_F8E4M3, dt=_lib.XK_F32), UNSUPPORTED), (dict(sdt=_lib.XK_F32), UNSUPPORTED),
    (dict(pdt=_lib.XK_BF16), UNSUPPORTED), (dict(T=0, k=None), _lib.XK_OK)], ids=str)
def test_append_refuses(change, status):
    assert _append(**change) == status


def _attend(**change):
    v = dict(q=PTR, qs=512, qt=512, qh=64, kc=PTR, kcp=2048, kcs=128, kch=64, vc=PTR, vcp=2048,
             vcs=128, vch=64, cdt=_lib.XK_BF16, pages=4, page=16, table=PTR, row=2, width=2,
             lens=PTR, scale=0.125, window=0, ks=None, vs=None, o=PTR, os=512, ot=512, oh=64,
             lse=None, B=2, T=1, Hq=8, Hkv=2, D=64, dt=_lib.XK_BF16, ws=None, size=0, stream=None)
    v.update(change)
    return _lib.lib().xk_paged_attention(*v.values())


@pytest.mark.parametrize("change,status", [
    (dict(B=-1), INVALID), (dict(T=0), INVALID), (dict(Hq=7), INVALID), (dict(Hq=0), INVALID),
    (dict(Hkv=0), INVALID), (dict(D=0), INVALID), (dict(D=60), INVALID), (dict(D=264), INVALID),
    (dict(width=-1), INVALID), (dict(page=0), INVALID), (dict(width=1 << 20, page=1 << 10), INVALID),
    (dict(pages=-1), INVALID), (dict(pages=1 << 31), INVALID), (dict(window=-1), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(q=None), INVALID), (dict(o=None), INVALID),
    (dict(lens=None), INVALID), (dict(table=None), INVALID), (dict(kc=None), INVALID),
    (dict(vc=None), INVALID), (dict(ks=PTR), INVALID), (dict(kcs=-128), INVALID),
    (dict(vcs=1 << 26), INVALID), (dict(cdt=_lib.XK_F16), UNSUPPORTED),
    (dict(dt=_lib.XK_I32), UNSUPPORTED), (dict(dt=_lib.XK_F32, cdt=_lib.XK_F8E4M3), UNSUPPORTED),
    (dict(q=PTR + 2), UNSUPPORTED), (dict(kc=PTR + 8), UNSUPPORTED), (dict(vch=60), UNSUPPORTED),
    (dict(qt=66), UNSUPPORTED), (dict(oh=66), UNSUPPORTED), (dict(B=0, q=None), _lib.XK_OK)],
    ids=str)
def test_attention_refuses(change, status):
    assert _attend(**change) == status


@pytest.mark.parametrize("change", [
    # pages of 2^32 bytes, from place to place and from page to page of 2^35
    dict(page=1 << 20, width=1, kcs=1 << 12), dict(page=1 << 20, width=1, vcs=1 << 12),
    dict(kcp=1 << 34), dict(vcp=1 << 34), dict(vcp=-2048),
    # more positions than a sequence has, in one page and without a table
    dict(page=(1 << 28) + 1, width=1), dict(page=1 << 62, width=0),
    # a scale that is not finite as a power of two
    dict(scale=3e38), dict(scale=-3e38),
    dict(B=(1 << 24) + 1), dict(T=(1 << 20) + 1), dict(Hq=1 << 17), dict(B=1 << 23),
    # blocks
    dict(T=1 << 20, Hq=1 << 16, Hkv=1 << 16, row=1 << 14, width=1 << 14)], ids=str)
def test_attention_refuses_what_a_launch_does_not_hold(change):
    assert _attend(ws=PTR, size=1 << 60, **change) == INVALID


def test_attention_refuses_small_workspaces():
    lib = _lib.lib()
    need = lib.xk_paged_attention_workspace_bytes(2, 1, 8, 2, 64, 1000, 16, _lib.XK_BF16)
    assert need > 0 and need % 256 == 0
    for ws, size in ((None, need), (PTR, need - 1), (PTR + 8, need)):
        assert _attend(width=1000, row=1000, ws=ws, size=size) == _lib.XK_ERR_WORKSPACE
    # Few enough positions that no sequence is ever cut: no workspace.
    assert lib.xk_paged_attention_workspace_bytes(2, 1, 8, 2, 64, 2, 16, _lib.XK_BF16) == 0
    assert lib.xk_paged_attention_workspace_bytes(2, 1, 7, 2, 64, 2, 16, _lib.XK_BF16) == 0


# --------------------------------------------------------------------------
# The C++ API and the Python mirror
# --------------------------------------------------------------------------
BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _tokens(heads, d=64, t=4, dtype=BF16):
    return torch.zeros(t, heads, d, dtype=dtype)


def _ok(api, q=None, k=None, pos=None, freq=None, scale=1.0):
    return api.npu_rotary_embedding(
        _tokens(8) if q is None else q, _tokens(2) if k is None else k,
        torch.arange(4) if pos is None else pos, torch.ones(32) if freq is None else freq, False,
        scale)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(4, 64, dtype=BF16)), dict(q=_tokens(8, dtype=torch.int32)),
    dict(k=_tokens(2, 32)), dict(k=_tokens(2, t=3)), dict(k=_tokens(2, dtype=F32)),
    dict(q=_tokens(8, 520), k=_tokens(2, 520)), dict(pos=torch.arange(3)),
    dict(pos=torch.zeros(4)), dict(pos=torch.arange(4)[None]), dict(freq=torch.ones(33)),
    dict(freq=torch.ones(0)), dict(freq=torch.ones(32, dtype=torch.float64)),
    dict(freq=torch.ones(1, 32)), dict(scale=0.0), dict(scale=float("inf")), dict(scale=1e39),
    dict()], ids=lambda c: str(list(c)))  # the last: not on a GPU
def test_rotary_wrappers_refuse(api, change):
    with pytest.raises(REFUSED):
        _ok(api, **change)


def _append_call(api, **change):
    c = dict(q=_tokens(8), k=_tokens(2), v=_tokens(2), kc=torch.zeros(3, 16, 2, 64, dtype=BF16),
             vc=torch.zeros(3, 16, 2, 64, dtype=BF16), slots=torch.arange(4), pos=torch.arange(4),
             freq=torch.ones(32), ks=None, vs=None)
    c.update(change)
    return api.npu_rotary_cache_append(c["q"], c["k"], c["v"], c["kc"], c["vc"], c["slots"],
                                       c["pos"], c["freq"], False, 1.0, c["ks"], c["vs"])


@pytest.mark.parametrize("change", [
    dict(v=_tokens(3)), dict(v=_tokens(2, dtype=F32)), dict(k=_tokens(0), v=_tokens(0)),
    dict(slots=torch.arange(5)), dict(slots=torch.zeros(4)), dict(pos=None), dict(freq=None),
    dict(kc=torch.zeros(3, 16, 2, 32, dtype=BF16)), dict(kc=torch.zeros(3, 16, 128, dtype=BF16)),
    dict(vc=torch.zeros(3, 16, 3, 64, dtype=BF16)), dict(vc=torch.zeros(4, 16, 2, 64, dtype=BF16)),
    dict(kc=torch.zeros(3, 0, 2, 64, dtype=BF16), vc=torch.zeros(3, 0, 2, 64, dtype=BF16)),
    dict(kc=torch.zeros(1, 16, 2, 64, dtype=BF16).expand(3, 16, 2, 64)),
    dict(kc=torch.zeros(3, 16, 64, 2, dtype=BF16).transpose(2, 3)),
    dict(kc=torch.zeros(3, 16, 2, 64), vc=torch.zeros(3, 16, 2, 64)),
    dict(kc=torch.zeros(3, 16, 2, 64, dtype=FP8)), dict(ks=torch.ones(2)),
    dict(kc=torch.zeros(3, 16, 2, 64, dtype=FP8), vc=torch.zeros(3, 16, 2, 64, dtype=FP8),
         ks=torch.ones(3)),
    dict(kc=torch.zeros(3, 16, 2, 64, dtype=torch.float8_e5m2),
         vc=torch.zeros(3, 16, 2, 64, dtype=torch.float8_e5m2)),
    dict()], ids=lambda c: str(list(c)))
def test_append_wrappers_refuse(api, change):
    with pytest.raises(REFUSED):
        _append_call(api, **change)


def _attend_call(api, **change):
    c = dict(q=torch.zeros(3, 8, 64, dtype=BF16), kc=torch.zeros(3, 16, 2, 64, dtype=BF16),
             vc=torch.zeros(3, 16, 2, 64, dtype=BF16), table=torch.zeros(3, 2, dtype=torch.int32),
             lens=torch.ones(3, dtype=torch.int32), scale=None, window=0, ks=None, vs=None)
    c.update(change)
    return api.npu_paged_attention(*c.values())


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(3, 64, dtype=BF16)), dict(q=torch.zeros(3, 7, 64, dtype=BF16)),
    dict(q=torch.zeros(3, 0, 64, dtype=BF16)), dict(q=torch.zeros(3, 8, 64)),
    dict(q=torch.zeros(3, 8, 60, dtype=BF16), kc=torch.zeros(3, 16, 2, 60, dtype=BF16),
         vc=torch.zeros(3, 16, 2, 60, dtype=BF16)),
    dict(table=torch.zeros(2, 2, dtype=torch.int32)), dict(table=torch.zeros(3, 2)),
    dict(lens=torch.ones(3)), dict(lens=torch.ones(2, dtype=torch.int32)), dict(window=-1),
    dict(scale=float("inf")), dict(scale=float("nan")), dict(ks=torch.ones(2)),
    dict(kc=torch.zeros(3, 16, 2, 64, dtype=FP8)), dict()], ids=lambda c: str(list(c)))
def test_attention_wrappers_refuse(api, change):
    with pytest.raises(REFUSED):
        _attend_call(api, **change)
