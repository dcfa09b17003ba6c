"""Pins of oracle/rotary.py (CPU): complex multiplication, the framework's other
rotations, the inverse and float64 autograd."""
import pytest
import torch

from oracle import rope, rotary


def _x(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


POS = torch.tensor([0, 1, 17, 4095, 1 << 20, -3])
FREQ = (1e4 ** (-torch.arange(8, dtype=torch.float64) / 8)).float()


def test_neighbours_are_a_complex_product():
    x = _x(1, 6, 3, 20)
    y, _ = rotary.turn(x, POS, FREQ, True, 1.25)
    z = torch.view_as_complex(x[..., :16].unflatten(-1, (8, 2)).contiguous())
    by = torch.polar(torch.tensor(1.25, dtype=torch.float64),
                     torch.outer(POS.double(), FREQ.double()))[:, None]
    torch.testing.assert_close(y[..., :16], torch.view_as_real(z * by).flatten(-2))
    assert torch.equal(y[..., 16:], x[..., 16:])


def test_halves_are_the_rotation_of_the_fused_norm():
    x = _x(2, 6, 3, 16)
    cos, sin = rope.neox_cos_sin(POS.clamp_min(0) % 4096, FREQ)
    want = x * cos.double()[:, None] + torch.cat([-x[..., 8:], x[..., :8]], -1) * sin.double()[:, None]
    y, _ = rotary.turn(x, POS.clamp_min(0) % 4096, FREQ)
    torch.testing.assert_close(y, want, rtol=0, atol=2e-3)  # fp32 angles up to 4096: 2^-12


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(interleaved):
    x, dy = _x(3, 6, 2, 18).requires_grad_(True), _x(4, 6, 2, 18)
    half = FREQ.numel()
    a = torch.outer(POS.double(), FREQ.double())[:, None]
    if interleaved:
        u, v = x[..., 0:16:2], x[..., 1:16:2]
    else:
        u, v = x[..., :half], x[..., half:16]
    p, q = 0.5 * (u * a.cos() - v * a.sin()), 0.5 * (v * a.cos() + u * a.sin())
    r = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    y = torch.cat([r, x[..., 16:]], -1)
    torch.testing.assert_close(rotary.turn(x.detach(), POS, FREQ, interleaved, 0.5)[0], y.detach())
    dx, = torch.autograd.grad(y, x, dy)
    torch.testing.assert_close(rotary.turn(dy, POS, FREQ, interleaved, 0.5, True)[0], dx)
