"""Cosines and sines of rotary positions, one rounding from the values in 64 bits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

# How far a cosine or sine of 32 bits may be off besides its own rounding, in units of 2**-24: 0.025 for the angle,
# which is known to 2**-32 of a turn (2 pi 2**-8); 0.03 for the terms left out of the series (x^11 / 11! at pi / 4);
# 0.37 for the roundings inside the terms after the first, at most x^3 / 6 = 0.081 of sine (0.016 of cosine): one
# unit of them each for x^2, x^3, the series over it and the product, a half for its first coefficient.  What of
# the angle stands behind its 24 bits is carried along.
UNITS = 0.025 + 0.03 + 0.37


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims", [128, 20])
@pytest.mark.parametrize("factor", [1.0, 1.1386, -2.5])
def test_turns_are_rounded_once(interleaved, dims, factor):
    """Pairs (1, 0) and (0, 1) come out as cosine and sine times the factor, over near and far positions."""
    from tritonkv_amd.rotary import Rotary, apply_rotary

    g = torch.Generator().manual_seed(dims)
    n = dims // 2
    w = torch.rand(n, generator=g, dtype=torch.float64) * 2
    N, D = 4096, 128
    pos = torch.randint(-2 ** 20, 2 ** 20, (1, N), generator=g, dtype=torch.int32)
    x = torch.zeros(1, 2, N, D)
    first = torch.arange(n) * 2 if interleaved else torch.arange(n)
    second = first + 1 if interleaved else first + n
    x[:, 0, :, first], x[:, 1, :, second] = 1.0, 1.0
    y = apply_rotary(x.cuda(), None, pos.cuda(), Rotary(inv_freq=w.cuda(), interleaved=interleaved, factor=factor))[0]
    y = y.cpu().double()
    f = float(torch.tensor(factor))  # as the 32-bit argument holds it
    angle = pos[0].double()[:, None] * w  # 2**21 radians in 64 bits: 2**-32 of one off at most
    cos, sin = f * angle.cos(), f * angle.sin()
    for got, want in ((y[0, 0][:, first], cos), (y[0, 0][:, second], sin), (y[0, 1][:, first], -sin),
                      (y[0, 1][:, second], cos)):
        off = (got - want).abs() * 2.0 ** 24
        rounding = torch.exp2(torch.floor(torch.log2(want.abs())))  # half a step, 0.5 for values of 1/2 to 1
        assert float((off - rounding - UNITS * abs(f)).max()) <= 0, float(off.max())
