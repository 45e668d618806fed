"""What a Rotary holds and which scalings it takes (no GPU)."""

from __future__ import annotations

import math

import pytest
import torch

from tritonkv_amd import rotary as ro


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_a_rotary_keeps_frequencies_of_its_own(dtype):
    """Those of a tensor that is changed later stay what its turns say."""
    w = torch.tensor([1.0, 0.25, 0.01], dtype=dtype)
    rot = ro.Rotary(inv_freq=w)
    before = rot.inv_freq.clone()
    w.mul_(2)
    assert torch.equal(rot.inv_freq, before) and torch.equal(rot.turns, ro._turns(before))
