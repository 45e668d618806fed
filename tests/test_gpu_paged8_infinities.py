"""Infinities and magnitudes past 2**64 in every type that the 8-bit append takes, turned or not."""

from __future__ import annotations

import math

import pytest
import torch

import paged8_ref as ref
from paged8_ref import E4M3, INT8

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def append(kn, vn, code, pos=0, **kw):
    """Codes and scales of K and V after an append into pools whose scales are 2**-6."""
    from tritonkv_amd.paged8 import paged8_append

    pools = [ref.make_pool(2, kn.shape[1], 64, kn.shape[3], code, 32, s, spread=False) for s in (1, 2)]
    start = [ref.numbers(p) for p in pools]
    paged8_append(*pools, kn.cuda(), vn.cuda(), torch.tensor([[1]], dtype=torch.int32, device="cuda"),
                  torch.tensor([pos], dtype=torch.int32, device="cuda"), **kw)
    return [ref.numbers(p) for p in pools], start


def assert_same(got, want):
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0].isnan(), want[0].isnan()) and torch.equal(got[0].nan_to_num(), want[0].nan_to_num())


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("N,pos", [(3, 0), (3, 5), (40, 0), (40, 9)])
def test_infinities_count_as_two_to_the_64(code, dtype, N, pos):
    x = torch.randn(1, 2, N, 128, generator=torch.Generator().manual_seed(N)).to(dtype)
    x[0, 0, 1, 7], x[0, 0, 2, 9], x[0, 1, 0, 3] = math.inf, -math.inf, -math.inf
    x[0, 1, 2, 4] = math.nan
    y = x.flip(1)
    got, start = append(x, y, code, pos)
    table = torch.tensor([[1]])
    for (codes, scale), new, have in zip(start, (x, y), got):
        ref.append(codes, scale, new.double(), table, [pos], None, code, 32)
        assert_same(have, (codes, scale))
    assert float(got[0][1][1, 0, 0]) == (2.0 ** 56 if code is E4M3 else 2.0 ** 58)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("N", [2, 40])
def test_turned_keys_past_two_to_the_64(code, dtype, interleaved, N):
    """At position 0 nothing turns but the factor: 2**60 takes keys of 16 to 64 past 2**64."""
    from tritonkv_amd.rotary import Rotary

    D = 64
    w = torch.zeros(D // 2, dtype=torch.float64)  # no angle at any position
    rot = Rotary(inv_freq=w.cuda(), interleaved=interleaved, factor=2.0 ** 60)
    g = torch.Generator().manual_seed(N)
    x = (torch.randn(1, 1, N, D, generator=g) * 20).to(dtype)
    v = torch.randn(1, 1, N, D, generator=g).to(dtype)
    got, start = append(x, v, code, 0, rotary=rot)
    for (codes, scale), new, have in zip(start, (x.double() * 2.0 ** 60, v.double()), got):
        ref.append(codes, scale, new, torch.tensor([[1]]), [0], None, code, 32)
        assert_same(have, (codes, scale))
