"""Tolerance of a result that was computed in fp32 and rounded once to its
type: the bound of the fp32 arithmetic (from the oracle) plus half a step of
the type, eps / 2 of the value; below the smallest normal number the step no
longer shrinks.  fp32 results carry their last rounding in the bound."""
import torch


def assert_within(actual, expected, err, what):
    dt, got = actual.dtype, actual.detach().cpu().double()
    assert got.shape == expected.shape, f"{what}: shape {tuple(got.shape)}"
    info = torch.finfo(dt)
    room = err + (info.eps / 2) * (expected.abs() + err) + info.tiny * info.eps
    off = (got - expected).abs()
    bad = ~((off <= room) | ((got == expected) & ~expected.isfinite()))
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} off, the worst by "
        f"{(off / room)[bad].max():.3g} of what is allowed; first at {bad.nonzero()[0].tolist()}: "
        f"{got[bad][0]} for {expected[bad][0]}")
