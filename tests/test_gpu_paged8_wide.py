"""The decode over 8-bit pages with more than 16 queries of a KV head to a workgroup."""

from __future__ import annotations

import pytest
import torch

from paged8_ref import E4M3, INT8
from test_gpu_paged8 import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [17, 33])
@pytest.mark.parametrize("M", [1, 2])
@pytest.mark.parametrize("code,dtype", [(E4M3, torch.float16), (E4M3, torch.bfloat16), (INT8, torch.float16),
                                        (INT8, torch.bfloat16)])
def test_two_tiles(D, G, M, code, dtype):
    run(2, G, 1, D, M, 64, 32, code, dtype, [95, 200], seed=G + M)
    run(2, G, 1, D, M, 64, 32, code, dtype, [300, 37], seed=G + M, piece=32)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_long_drafts(D, code):
    """32 queries a row and 9 of them, over cut rows."""
    run(2, 2, 2, D, 32, 32, 32, code, torch.bfloat16, [150, 70], counts=[32, 9], piece=64)
    run(2, 4, 2, D, 9, 32, 32, code, torch.float16, [33, 600], counts=[9, 1])
