"""CPU checks of what the Python functions of the gated linear recurrence and
the block-to-block norm hand to the C-ABI, with a library in its place that
takes every call and launches nothing."""
import contextlib

import pytest
import torch

from torch_npu_ops_amd import ops


class _Library:
    """Keeps the arguments of each call; a call succeeds, a size is 256 bytes."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return 256 if name.endswith("_bytes") else 0
        return call


@pytest.fixture
def library(monkeypatch):
    at = _Library()
    monkeypatch.setattr(ops, "lib", lambda: at)
    monkeypatch.setattr(ops, "_stream", lambda t: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    return at


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float64], ids=str)
def default_dtype(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield
    torch.set_default_dtype(before)


def test_fp32_outputs_do_not_follow_torchs_default_dtype(library, default_dtype):
    # The kernels write 4 bytes an element into each of these.
    f32, bf16 = torch.float32, torch.bfloat16
    x, lam, cu = torch.zeros(1, 40, 8, dtype=bf16), torch.zeros(8, dtype=f32), torch.arange(3)
    _, fin, states = ops.npu_gated_linear_recurrence(x, x, x, lam, 8.0, None, True, cu, True)
    dx, da, db, dlam, dh0 = ops.npu_gated_linear_recurrence_bwd(x, x, x, x, lam, states, 8.0,
                                                                cu_seqlens=cu)
    assert [t.dtype for t in (fin, states, dlam, dh0)] == [f32] * 4
    assert [t.dtype for t in (dx, da, db)] == [bf16] * 3
    w = torch.ones(8, dtype=bf16)
    h, y, r1, r2 = ops.npu_gated_residual_rms_norm(x, x.to(f32), w, x, w, w)
    assert (h.dtype, y.dtype, r1.dtype, r2.dtype) == (f32, bf16, f32, f32)


def test_rows_too_far_apart_for_a_tile_are_copied_in_prefill_and_backward_alone(library):
    # 2 tokens, 2^25 elements apart or one less.
    lam, cu = torch.zeros(8), torch.tensor([0, 2])
    near = torch.zeros(1, 2, 8, dtype=torch.bfloat16)
    states = torch.zeros(1, 8)
    for pitch, want in (((1 << 25) - 1, (1 << 25) - 1), (1 << 25, 8)):
        x = torch.empty(pitch + 8, dtype=torch.bfloat16).as_strided((1, 2, 8), (8, pitch, 1))
        ops.npu_gated_linear_recurrence(x, near, near, lam, cu_seqlens=cu)
        assert library.calls["xk_gated_linear_recurrence"][1] == want
        ops.npu_gated_linear_recurrence_bwd(x, near, x, near, lam, states, cu_seqlens=cu)
        assert library.calls["xk_gated_linear_recurrence_bwd"][1] == want
        assert library.calls["xk_gated_linear_recurrence_bwd"][5] == want
        ops.npu_gated_linear_recurrence_update(x[0], near[0], near[0], lam, torch.zeros(2, 8))
        assert library.calls["xk_gated_linear_recurrence_update"][1] == pitch
