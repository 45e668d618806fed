"""Where the 16-bit decode keeps rows whole: the plan takes the form that was measured faster
at each of these sizes (``plan_shares`` quotes the times)."""

from __future__ import annotations

import pytest


@pytest.mark.parametrize("D,S,units,whole", [
    (128, 512, 32, False), (128, 512, 64, False), (128, 512, 128, True), (128, 512, 256, True),
    (128, 384, 64, False), (128, 384, 128, True), (128, 256, 8, True),
    (64, 1024, 64, False), (64, 1024, 128, False), (64, 1024, 256, True), (64, 512, 8, True),
    (256, 256, 32, False), (256, 256, 64, True), (256, 128, 8, True),
    (128, 1024, 504, False), (128, 1024, 512, True), (128, 1040, 1024, False),
])
def test_whole_rows(D, S, units, whole):
    from tritonkv_amd.paged16 import plan_shares

    assert (plan_shares(units // 8, 8, 4, S, D)[1] == 0) is whole
