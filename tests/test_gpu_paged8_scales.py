"""Scales that are none, and scores past 32-bit floats, in the decode over 8-bit pages."""

from __future__ import annotations

import math

import pytest
import torch

import paged8_ref as ref
from paged8_ref import E4M3, INT8

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("piece", [None, 32])
def test_a_block_without_a_scale_reaches_only_queries_that_see_it(which, code, bad, D, piece):
    """The last two of five tokens begin a block: the three queries before them see none of it."""
    from tritonkv_amd.paged8 import paged8_decode_attention

    L, M = 66, 5
    pools = [ref.make_pool(4, 2, 64, D, code, 32, s) for s in (1, 2)]
    table = ref.make_table(1, 2, 4, 3)
    pools["kv".index(which)].scale[int(table[0, 1]), :, 0] = bad
    q = torch.randn(1, 4, M, D, generator=torch.Generator().manual_seed(2)).half()
    clean = ref.decode(q[:, :, :3], *(ref.numbers(p) for p in pools), table, [L - 2], None, D ** -0.5)
    lse = torch.zeros(1, 4, M, device="cuda")
    got = paged8_decode_attention(q.cuda(), *pools, table.cuda(), ints([L]), lse=lse, piece_tokens=piece)
    ref.assert_within(got[:, :, :3], clean[0], clean[2], "out")
    ref.assert_within(lse[:, :, :3], clean[1], clean[3], "lse")
    if which == "v":
        assert not torch.isfinite(got[:, :, 3:]).any() and torch.isfinite(lse).all()
    elif math.isnan(bad):
        assert got[:, :, 3:].isnan().all() and lse[:, :, 3:].isnan().all()


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("HQ,M", [(2, 1), (20, 1), (2, 3)])
@pytest.mark.parametrize("piece", [None, 32])
def test_scores_past_32_bits_are_not_zeros(code, HQ, M, piece):
    """Scores over 2**128 have no softmax in 32 bits: NaN, for their query alone."""
    from tritonkv_amd.paged8 import paged8_decode_attention

    k, v = (ref.make_pool(4, 1, 64, 64, code, 32, s) for s in (1, 2))
    k.codes.copy_(k.codes.float().abs().clamp(min=1.0).to(code))
    k.scale.fill_(2.0 ** 40)
    table = ref.make_table(2, 2, 4, 3)
    q = torch.zeros(2, HQ, M, 64)
    q[:, 0] = 2.0 ** 100  # the score: 64 codes of 1 and more times 2^40 times 2^100 / 8, over 2^143
    q[:, 1:] = torch.randn(2, HQ - 1, M, 64, generator=torch.Generator().manual_seed(1)) * 2.0 ** -46
    q = q.bfloat16()
    lens = [100, 33]
    want = ref.decode(q, ref.numbers(k), ref.numbers(v), table, lens, None, 0.125)
    lse = torch.zeros(2, HQ, M, device="cuda")
    got = paged8_decode_attention(q.cuda(), k, v, table.cuda(), ints(lens), lse=lse, piece_tokens=piece)
    assert got[:, 0].isnan().all() and lse[:, 0].isnan().all()
    ref.assert_within(got[:, 1:], want[0][:, 1:], want[2][:, 1:], "out")
    ref.assert_within(lse[:, 1:], want[1][:, 1:], want[3][:, 1:], "lse")
