"""Prompts long enough that a workgroup of the 8-bit append or read takes two heads and turns queries in tiles."""

from __future__ import annotations

import pytest
import torch

import paged8_ref as ref
from paged8_ref import E4M3, INT8

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


def rows(B, H, N, D, dtype, seed):
    """Token-major values whose size varies along the tokens, so that blocks get scales of their own."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, N, H, D, generator=g) * torch.exp2(torch.randint(-4, 5, (B, N, 1, 1), generator=g).float())
    return x.to(dtype).transpose(1, 2)


def append(B, HQ, HKV, N, D, page, block, code, dtype, pos, counts, dims=0, interleaved=False, seed=0):
    from tritonkv_amd.paged8 import paged8_append
    from tritonkv_amd.rotary import Rotary, apply_rotary

    width = -(-(max(pos) + N) // page)
    P = B * width + 1
    k, v = (ref.make_pool(P, HKV, page, D, code, block, seed + i) for i in (1, 2))
    table = ref.make_table(B, width, P, seed + 3)
    kn, vn = (rows(B, HKV, N, D, dtype, seed + i) for i in (4, 5))
    keys, turn = kn.double(), {}
    if dims:
        w = torch.tensor([10000.0 ** (-2.0 * i / dims) for i in range(dims // 2)], dtype=torch.float64)
        t = torch.tensor(pos)[:, None] + torch.arange(N)
        keys = ref.turn(keys, t[:, None], w, interleaved, 1.1)
        q = rows(B, HQ, N, D, dtype, seed + 6).cuda()
        rot = Rotary(inv_freq=w.cuda(), interleaved=interleaved, factor=1.1)
        turn = dict(rotary=rot, q=q, q_out=torch.full_like(q, 3.0))
    want = []
    for pool, new in ((k, keys), (v, vn.double())):
        c, s = ref.numbers(pool)
        ref.append(c, s, new, table, pos, counts, code, block)
        want.append((c, s))
    got = paged8_append(k, v, kn.cuda(), vn.cuda(), table.cuda(), ints(pos), ints(counts), **turn)
    (kc, ks), (vc, vs) = ref.numbers(k), ref.numbers(v)
    assert torch.equal(vs, want[1][1]) and torch.equal(vc, want[1][0])
    if not dims:
        assert torch.equal(ks, want[0][1]) and torch.equal(kc, want[0][0])
        return
    # A turned value is off by 8 * 2^-24 of its pair at most: its code may be the other neighbour where it lies
    # that close to the middle of two (16 * 2^-24 of a pair of up to 360 steps: under 4e-4 of them), its block's
    # scale the other power of two where the largest lies that close to one (about 1e-6 of the blocks).
    assert torch.equal(ks, want[0][1])
    d = (kc - want[0][0]).abs()
    step = torch.ones_like(d) if code is INT8 else torch.exp2(torch.floor(torch.log2(kc.abs().clamp(min=2.0 ** -6))) - 3)
    assert (d <= 2 * step).all() and (d > 0).double().mean() < 1e-3
    plain = apply_rotary(q, None, ints(pos), rot)[0]
    live = torch.ones(B, N, dtype=torch.bool) if counts is None else torch.arange(N) < torch.tensor(counts)[:, None]
    assert torch.equal(got, torch.where(live.cuda()[:, None, :, None], plain, 3.0))


@pytest.mark.parametrize("code,dtype", [(E4M3, BF16), (INT8, F16), (E4M3, F32), (INT8, F32)])
@pytest.mark.parametrize("HKV", [5, 6])
def test_two_heads_a_workgroup(code, dtype, HKV):
    """1095 and 1314 blocks of the rows' heads; of five heads the last one stands alone."""
    append(3, 0, HKV, 2300, 64, 64, 32, code, dtype, [0, 45, 31], [2300, 1001, 2299], seed=HKV)


@pytest.mark.parametrize("code,dtype", [(E4M3, F16), (INT8, BF16), (INT8, F32)])
def test_two_heads_of_the_largest_blocks(code, dtype):
    """128 tokens of 256 dims: 32 values a thread, 1080 blocks."""
    append(120, 0, 3, 130, 256, 128, 128, code, dtype, [7 * b % 127 for b in range(120)],
           [130 - b % 9 for b in range(120)])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("code,dtype,dims", [(E4M3, BF16, 128), (INT8, F16, 64), (E4M3, F32, 32)])
def test_two_heads_with_turns_and_queries_in_tiles(code, dtype, dims, interleaved):
    """3 * 2300 tokens: several to a workgroup of queries, the last ones ragged."""
    append(3, 7, 5, 2300, 128, 64, 32, code, dtype, [3, 45, 1000], [2300, 1001, 2299], dims, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_the_largest_blocks_with_turns(code, dtype, interleaved):
    append(2, 3, 3, 300, 256, 128, 128, code, dtype, [100, 0], [300, 211], 256, interleaved)
    append(2, 3, 3, 130, 256, 256, 128, code, dtype, [5, 127], None, 128, interleaved, seed=9)


@pytest.mark.parametrize("B,N", [(4100, 1), (1400, 3)])
def test_many_short_rows_with_queries_in_tiles(B, N):
    """One wave a workgroup, and over 4096 tokens."""
    append(B, 2, 1, N, 64, 32, 32, E4M3, BF16, [b % 29 for b in range(B)], None, 64)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("HKV,D", [(5, 64), (4, 128), (3, 256)])
def test_read_of_two_heads(code, dtype, HKV, D):
    """2085 blocks of 32 tokens of the rows' heads and more, counts and entries missing."""
    from tritonkv_amd.paged8 import paged8_read

    B, N, page = (3, 4400, 64) if D == 64 else (8, 3000, 96)
    P, width = 40, -(-(N + 50) // page)
    k, v = (ref.make_pool(P, HKV, page, D, code, 32, s) for s in (1, 2))
    g = torch.Generator().manual_seed(3)
    table = torch.randint(-2, P + 2, (B, width), generator=g, dtype=torch.int32)  # (rows may share pages)
    pos, counts = [(0, 31, 50)[b % 3] for b in range(B)], [N - 500 * b for b in range(B)]  # (below zero: none)
    got = paged8_read(k, v, table.cuda(), ints(pos), ints(counts),
                      out=tuple(torch.full((B, HKV, N, D), 5.0, dtype=dtype, device="cuda") for _ in range(2)))
    t = torch.tensor(pos)[:, None] + torch.arange(N)
    entry = table.long().gather(1, (t // page).clamp(max=width - 1))
    live = (torch.arange(N) < torch.tensor(counts)[:, None]) & (entry >= 0) & (entry < P) & (t < width * page)
    for pool, y in zip((k, v), got):
        c, s = ref.numbers(pool)
        full = (c.view(P, HKV, page // 32, 32, D) * s[..., None, None]).view(P, HKV, page, D).float().to(dtype)
        want = torch.where(live[..., None, None], full[entry.clamp(0, P - 1), :, t % page], 5.0).transpose(1, 2)
        assert torch.equal(y.cpu(), want)
