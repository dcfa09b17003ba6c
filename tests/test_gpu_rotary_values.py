"""GPU check of the rotation's cosines and sines by themselves, within the bound
that oracle/rotary.py derives."""
import pytest
import torch

from oracle import rotary

pytestmark = pytest.mark.gpu


def _api(name):
    from torch_npu_ops_amd import _xk_torch, ops
    return {"cpp": _xk_torch, "py": ops}[name]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("reach", [8, 4096, 1 << 20, 1 << 29])
def test_cosines_and_sines(dev, interleaved, reach):
    """Pairs (1, 0) turn into (cos, sin) with no other rounding; every quarter
    turn, angles near their borders and near zero."""
    g = torch.Generator().manual_seed(reach)
    T, half = 3001, 128
    pos = torch.randint(1 - reach, reach, (T,), generator=g)
    f = torch.cat([(1e6 ** (-torch.arange(64) / 64)), torch.rand(60, generator=g),
                   torch.tensor([torch.pi / 2, torch.pi / 4, torch.pi, 1.0])]).float()
    x = torch.zeros(T, 1, 2 * half)
    x[..., ::2 if interleaved else 1][..., :half] = 1
    a = torch.outer(pos.double(), f.double())
    for api, back in (("cpp", False), ("py", True)):
        fn = getattr(_api(api), "npu_rotary_embedding" + ("_bwd" if back else ""))
        y = fn(x.to(dev), None, pos.to(dev), f.to(dev), interleaved)[0].cpu().double()[:, 0]
        c, s = (y[:, ::2], y[:, 1::2]) if interleaved else (y[:, :half], y[:, half:])
        assert (c - a.cos()).abs().max() <= rotary.TURN
        assert (s - a.sin() * (-1 if back else 1)).abs().max() <= rotary.TURN
