"""Attention over 8-bit pages against a plain softmax in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import paged8_ref as ref
from paged8_ref import E4M3, INT8

pytestmark = pytest.mark.gpu


def run(B, HQ, HKV, D, M, page, block, code, dtype, lens, counts=None, width=None, seed=0, sm_scale=None, piece=None,
        three=False, ws=None, dead=True):
    from tritonkv_amd.paged8 import paged8_decode_attention

    need = [-(-n // page) for n in lens]
    width = width or max(1, max(need))
    P = max(1, sum(need)) + 2
    k, v = (ref.make_pool(P, HKV, page, D, code, block, seed + i) for i in (1, 2))
    table = ref.make_table(B, width, P, seed + 3, need)
    if dead and code is E4M3:  # what lies past a row's tokens must not matter
        for b, n in enumerate(lens):
            if n % page:
                p = int(table[b, n // page])
                for pool in (k, v):
                    pool.codes.view(torch.int8)[p, :, n % page:] = 0x7f
    g = torch.Generator().manual_seed(seed + 4)
    q = torch.randn(B, M, HQ, D, generator=g).to(dtype).transpose(1, 2)
    sm = 1.0 / math.sqrt(D) if sm_scale is None else sm_scale
    want = ref.decode(q, ref.numbers(k), ref.numbers(v), table, lens, counts, sm)
    cuda = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    qd = q.cuda()
    qd = qd[:, :, 0] if three else qd
    out = torch.full(qd.shape, 7.0, device="cuda")
    lse = torch.full(qd.shape[:-1], 7.0, device="cuda")
    got = paged8_decode_attention(qd, k, v, table.cuda(), cuda(lens), sm_scale, out, lse, ws, counts=cuda(counts),
                                  piece_tokens=piece)
    assert got is out
    ref.assert_within(out.view(want[0].shape), want[0], want[2], "out")
    ref.assert_within(lse.view(want[1].shape), want[1], want[3], "lse")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_types_and_head_dims(D, code, dtype):
    run(3, 8, 2, D, 1, 64, 32, code, dtype, [1, 77, 130], three=True)
    run(2, 8, 2, D, 3, 64, 64, code, dtype, [200, 33], seed=5)


@pytest.mark.parametrize("G", [1, 3, 16, 17, 33])
@pytest.mark.parametrize("M", [1, 2])
def test_groups(G, M):
    run(2, 2 * G, 2, 64, M, 32, 32, E4M3, torch.float16, [95, 64], seed=G)


@pytest.mark.parametrize("block,pages", [(32, 1), (32, 3), (64, 2), (128, 1), (128, 2)])
def test_blocks_and_pages(block, pages):
    run(2, 4, 2, 128, 1, block * pages, block, E4M3, torch.bfloat16, [block * pages * 2 + 5, block - 1])


@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_lengths(n):
    run(2, 4, 2, 128, 1, 64, 32, INT8, torch.float16, [n, 100], width=8)
    run(2, 4, 2, 128, 4, 64, 32, E4M3, torch.float16, [n, 100], width=8)


@pytest.mark.parametrize("piece", [32, 96, 1024])
@pytest.mark.parametrize("M", [1, 5])
def test_cut_rows(piece, M):
    run(4, 8, 2, 128, M, 64, 32, E4M3, torch.bfloat16, [700, 0, 3, 333], piece=piece)


def test_wide_tables_and_default_cut():
    run(3, 8, 2, 128, 1, 32, 32, E4M3, torch.float16, [1500, 2, 999], width=300)
    run(3, 8, 2, 64, 2, 32, 32, INT8, torch.float16, [1500, 2, 999], width=300)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_drafts_of_other_counts(code):
    """Rows with fewer queries than M, none, more than they have tokens."""
    run(6, 4, 2, 128, 4, 64, 32, code, torch.bfloat16, [70, 70, 2, 0, 65, 33], counts=[4, 1, 4, 2, 0, 3])
    run(3, 4, 2, 128, 1, 64, 32, code, torch.bfloat16, [70, 1, 5], counts=[1, 0, 9])
    run(2, 4, 2, 64, 32, 64, 32, code, torch.float16, [40, 200], piece=32)


def test_many_rows():
    lens = [(7 * b) % 90 for b in range(130)]
    run(130, 4, 2, 64, 1, 32, 32, E4M3, torch.float16, lens, piece=64)
    run(130, 4, 2, 64, 1, 32, 32, INT8, torch.float16, lens)


def test_lengths_past_the_table_are_clamped():
    from tritonkv_amd.paged8 import paged8_decode_attention

    k, v = (ref.make_pool(4, 2, 32, 64, E4M3, 32, s) for s in (1, 2))
    table = ref.make_table(1, 2, 4, 3)
    q = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(1)).half()
    a = paged8_decode_attention(q.cuda(), k, v, table.cuda(), torch.tensor([999], dtype=torch.int32, device="cuda"))
    b = paged8_decode_attention(q.cuda(), k, v, table.cuda())
    assert torch.equal(a, b)
    want = ref.decode(q[:, :, None], ref.numbers(k), ref.numbers(v), table, [64], None, 0.125)
    ref.assert_within(a[:, :, None], want[0], want[2])


def test_scales_far_apart():
    """Blocks whose scales lie 2^60 apart, the smaller ones seen through p, and large and tiny queries."""
    from tritonkv_amd.paged8 import paged8_decode_attention

    k, v = (ref.make_pool(2, 1, 96, 64, E4M3, 32, s) for s in (1, 2))
    k.scale[:] = torch.tensor([2.0 ** -9, 2.0 ** -40, 2.0 ** -12]).cuda()
    v.scale[:] = torch.tensor([2.0 ** -30, 2.0 ** 30, 1.0]).cuda()
    table = torch.tensor([[1], [1]], dtype=torch.int32)
    for dtype, mul in ((torch.float16, 1.0), (torch.bfloat16, 1.0), (torch.bfloat16, 2.0 ** -20), (torch.float16, 2.0 ** 6)):
        q = (torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(1)) * mul).to(dtype)
        lens = [32, 96]
        want = ref.decode(q[:, :, None], ref.numbers(k), ref.numbers(v), table, lens, None, 0.125)
        got = paged8_decode_attention(q.cuda(), k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
        ref.assert_within(got[:, :, None], want[0], want[2], f"{dtype} {mul}")


@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_of_a_draft_reaches_only_those_that_see_it(which):
    """A NaN code in the last but one of five tokens: earlier queries are clean."""
    from tritonkv_amd.paged8 import paged8_decode_attention

    L, M = 70, 5
    pools = [ref.make_pool(3, 2, 64, 128, E4M3, 32, s) for s in (1, 2)]
    table = ref.make_table(1, 2, 3, 3)
    bad = L - 2
    pools["kv".index(which)].codes.view(torch.int8)[int(table[0, bad // 64]), 1, bad % 64, 5] = 0x7f
    q = torch.randn(1, 4, M, 128, generator=torch.Generator().manual_seed(2)).half()
    want = ref.decode(q, *(ref.numbers(p) for p in pools), table, [L], None, 128 ** -0.5)
    lens = torch.tensor([L], dtype=torch.int32, device="cuda")
    for piece in (None, 32):
        got = paged8_decode_attention(q.cuda(), *pools, table.cuda(), lens, piece_tokens=piece)
        assert not got[:, :, :M - 2].isnan().any() and not got[:, :2].isnan().any()
        sees = got[:, 2:, M - 2:]
        assert sees.isnan().all() if which == "k" else (sees[..., 5].isnan().all() and sees.isnan().sum() == sees[..., 5].numel())
        ref.assert_within(got, want[0], want[2])


def test_queries_that_are_not_finite():
    """As in softmax: a query of NaN gives NaN for itself alone."""
    from tritonkv_amd.paged8 import paged8_decode_attention

    k, v = (ref.make_pool(2, 1, 64, 64, INT8, 32, s) for s in (1, 2))
    table = torch.tensor([[0, 1]], dtype=torch.int32)
    for dtype in (torch.float16, torch.bfloat16):
        q = torch.randn(1, 3, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
        q[0, 1, 7] = math.nan
        got = paged8_decode_attention(q.cuda(), k, v, table.cuda(), torch.tensor([90], dtype=torch.int32, device="cuda"))
        assert got[0, 1].isnan().all() and not got[0, [0, 2]].isnan().any()
        q[0, 1] = 0.0
        want = ref.decode(q[:, :, None], ref.numbers(k), ref.numbers(v), table, [90], None, 0.125)
        got = paged8_decode_attention(q.cuda(), k, v, table.cuda(), torch.tensor([90], dtype=torch.int32, device="cuda"))
        ref.assert_within(got[:, :, None], want[0], want[2])


def test_strided_pools():
    """K and V as the halves of one token-major buffer, scales of their own strides."""
    from tritonkv_amd.paged8 import Paged8Pool, paged8_decode_attention

    P, HKV, page, D = 5, 2, 64, 128
    a, b = (ref.make_pool(P, HKV, page, D, E4M3, 32, s) for s in (1, 2))
    store = torch.empty(P, page, 2, HKV, D, dtype=E4M3, device="cuda")
    scales = torch.empty(2, 2, P, HKV, device="cuda")  # (block, k or v, page, head)
    pools = []
    for i, p in enumerate((a, b)):
        pools.append(Paged8Pool(store[:, :, i].transpose(1, 2), scales[:, i].permute(1, 2, 0)))
        pools[-1].codes.view(torch.int8).copy_(p.codes.view(torch.int8))
        pools[-1].scale.copy_(p.scale)
    table = ref.make_table(2, 2, P, 3).cuda()
    lens = torch.tensor([100, 65], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 128, device="cuda").half()
    assert torch.equal(paged8_decode_attention(q, a, b, table, lens), paged8_decode_attention(q, *pools, table, lens))


def test_kept_calls_streams_and_graphs():
    """One workspace over layers, on another stream, and a captured step that follows its lengths."""
    from tritonkv_amd.paged8 import paged8_decode_attention

    layers = [[ref.make_pool(40, 2, 32, 128, E4M3, 32, 10 * i + s) for s in (1, 2)] for i in range(2)]
    table = ref.make_table(2, 20, 40, 3).cuda()
    lens = torch.tensor([600, 17], dtype=torch.int32, device="cuda")
    qs = [torch.randn(2, 8, 128, device="cuda").bfloat16() for _ in range(2)]
    want = [paged8_decode_attention(q, *p, table, lens) for q, p in zip(qs, layers)]
    ws: dict = {}
    for _ in range(2):
        for q, p, w in zip(qs, layers, want):
            assert torch.equal(paged8_decode_attention(q, *p, table, lens, _workspace=ws), w)
    assert "call" in ws
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [paged8_decode_attention(q, *p, table, lens, _workspace=ws) for q, p in zip(qs, layers)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    outs = [torch.empty(2, 8, 128, device="cuda") for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for q, p, o in zip(qs, layers, outs):
            paged8_decode_attention(q, *p, table, lens, out=o, _workspace=ws)
    for new in ([600, 17], [1, 640], [333, 0]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        for q, p, o in zip(qs, layers, outs):
            assert torch.equal(o, paged8_decode_attention(q, *p, table, lens))


def test_long_cache_past_32_bits():
    """Pages that lie past 2^32 bytes of the pool."""
    from tritonkv_amd.paged8 import Paged8Pool, paged8_decode_attention

    small = [ref.make_pool(4, 4, 128, 128, INT8, 128, s) for s in (1, 2)]
    P = (1 << 32) // (4 * 128 * 128) + 8
    pools = []
    for p in small:
        codes = torch.zeros(P, 4, 128, 128, dtype=INT8, device="cuda")
        scale = torch.zeros(P, 4, 1, device="cuda")
        codes[-4:], scale[-4:] = p.codes, p.scale
        pools.append(Paged8Pool(codes, scale))
    q = torch.randn(1, 8, 128, device="cuda").half()
    lens = torch.tensor([401], dtype=torch.int32, device="cuda")
    table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device="cuda")
    assert torch.equal(paged8_decode_attention(q, *small, table, lens),
                       paged8_decode_attention(q, *pools, table + (P - 4), lens))
