"""Quantizing into 8-bit pages and reading them back, against the definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import paged8_ref as ref
from paged8_ref import E4M3, INT8

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")


def values(B, HKV, N, D, dtype, seed, token_major=False, grow=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*((B, N, HKV, D) if token_major else (B, HKV, N, D)), generator=g)
    x = x.transpose(1, 2) if token_major else x
    return (x * torch.linspace(1.0, grow, N)[:, None] ** 2).to(dtype)


def check(B, HKV, N, D, page, block, code, dtype, pos, counts=None, width=None, seed=0, token_major=False, grow=1.0,
          table=None, x=None, ws=None, pools=None):
    from tritonkv_amd.paged8 import paged8_append

    width = width or max(1, -(-(max(pos) + N) // page))
    P = B * width + 2
    kn, vn = x if x is not None else (values(B, HKV, N, D, dtype, seed + i, token_major, grow) for i in (1, 2))
    k, v = pools or (ref.make_pool(P, HKV, page, D, code, block, seed + i) for i in (3, 4))
    table = ref.make_table(B, width, P, seed + 5) if table is None else table
    want = []
    for pool, new in ((k, kn), (v, vn)):
        codes, scale = ref.numbers(pool)
        ref.append(codes, scale, new.double(), table, pos, counts, code, block)
        want.append((codes, scale))
    assert paged8_append(k, v, kn.cuda(), vn.cuda(), table.cuda(), ints(pos), ints(counts), ws) is None
    for pool, (codes, scale) in zip((k, v), want):
        got = ref.numbers(pool)
        assert torch.equal(got[1], scale)
        assert torch.equal(got[0].isnan(), codes.isnan())
        assert torch.equal(got[0].nan_to_num(), codes.nan_to_num())
    return k, v


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("block", [32, 64, 128])
def test_types_and_sizes(code, dtype, D, block):
    check(2, 2, block + 5, D, 2 * block, block, code, dtype, [0, 17])
    check(3, 2, 1, D, block, block, code, dtype, [0, 1, block + 7])


@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 32, 33, 100, 257])
def test_lengths(N):
    check(2, 2, N, 128, 64, 32, E4M3, BF16, [0, 45], seed=N)
    check(2, 1, N, 64, 32, 32, INT8, F16, [31, 5], seed=N, token_major=True)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_scales_rise(code):
    """Values that grow along the tokens, appended in pieces: earlier codes are rounded again."""
    k, v = check(1, 2, 10, 128, 64, 32, code, F32, [0], width=3, grow=1.0)
    table = ref.make_table(1, 3, 5, 5)
    at = 10
    for i, n in enumerate((1, 1, 3, 1, 9, 40, 1)):
        k, v = check(1, 2, n, 128, 64, 32, code, F32, [at], width=3, seed=20 + i, grow=30.0,
                     x=[values(1, 2, n, 128, F32, 40 + i + j, grow=3.0) * 4.0 ** i for j in (0, 50)], table=table,
                     pools=(k, v))
        at += n
    # a smaller value keeps the scale
    before = k.scale.clone()
    check(1, 2, 1, 128, 64, 32, code, F32, [at], x=[values(1, 2, 1, 128, F32, 9) * 1e-3] * 2, table=table, pools=(k, v))
    assert torch.equal(before, k.scale)


def test_first_slot_starts_the_block_anew():
    k, v = check(1, 2, 32, 64, 32, 32, E4M3, F16, [0], grow=9.0)
    check(1, 2, 1, 64, 32, 32, E4M3, F16, [0], x=[values(1, 2, 1, 64, F16, 9) * 0.01] * 2,
          table=ref.make_table(1, 1, 3, 5), pools=(k, v))


@pytest.mark.parametrize("old", [0.0, -1.0, math.nan, math.inf, 0.3, 2.0 ** -130, 1e-42])
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_scales_that_an_append_did_not_make(old, code):
    """None yet (0), no scale at all, one that is no power of two, subnormal ones."""
    from tritonkv_amd.paged8 import paged8_append

    k, v = (ref.make_pool(2, 1, 64, 64, code, 32, s) for s in (1, 2))
    k.scale.fill_(old)
    v.scale.fill_(old)
    table = torch.tensor([[1]], dtype=torch.int32)
    x = [values(1, 1, 3, 64, F32, s) * (1.0 if old != 0.3 else 5.0) for s in (1, 2)]
    want = [ref.numbers(p) for p in (k, v)]
    for (c, s), new in zip(want, x):
        ref.append(c, s, new.double(), table, [5], None, code, 32)
    paged8_append(k, v, *(y.cuda() for y in x), table.cuda(), ints([5]))
    for pool, (c, s) in zip((k, v), want):
        got = ref.numbers(pool)
        assert torch.equal(got[1].nan_to_num(7, 8, 9), s.nan_to_num(7, 8, 9))
        new = slice(5, 8)
        if old == 0.3:  # y / s in 32 bits may round to a border that 64 bits miss: half a step and 2^-24
            y = got[0][1, :, new] * s[1, :, :1, None]
            d = (y - x[0 if pool is k else 1].double()[0]).abs()
            step = s[1, 0, 0] / 2 if code is INT8 else torch.maximum(y.abs() / 16, s[1, 0, 0] * 2.0 ** -10)
            assert (d <= step * (1 + 2.0 ** -20)).all()
        else:
            assert torch.equal(got[0], c)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_values_that_are_not_finite_zero_and_tiny(code):
    x = torch.randn(4, 2, 5, 64, generator=torch.Generator().manual_seed(3))
    x[0, 0, 1, 3], x[0, 1, :, :] = math.nan, math.nan
    x[1, 0, 2, 5], x[1, 1, 0, 6] = math.inf, -math.inf
    x[2] = 0.0
    x[3] *= 2.0 ** -80
    x[3, 1, 0, 0] = 1e-42
    for dtype in (F32, BF16):
        check(4, 2, 5, 64, 32, 32, code, dtype, [0, 0, 0, 0], x=[x.to(dtype), x.flip(0).to(dtype)])
        check(4, 2, 5, 64, 32, 32, code, dtype, [9, 9, 9, 9], x=[x.to(dtype), x.flip(0).to(dtype)])


def test_magnitudes_next_to_the_largest_code():
    """448 * 2^k and 127 * 2^k just fit; the next value up needs the next scale."""
    from tritonkv_amd.paged8 import paged8_append

    for code in (E4M3, INT8):
        for k in (-3, 0, 5):
            edge = ref.TOP[code] * 2.0 ** k
            up = float(torch.nextafter(torch.tensor(edge), torch.tensor(math.inf)))
            for top, s in ((edge, 2.0 ** k), (up, 2.0 ** (k + 1))):
                pools = [ref.make_pool(1, 1, 32, 64, code, 32, i) for i in (1, 2)]
                x = torch.zeros(1, 1, 1, 64)
                x[..., 9] = top
                paged8_append(*pools, x.cuda(), -x.cuda(), ints([[0]]), ints([0]))
                assert float(pools[0].scale) == s and float(pools[1].scale) == s
                assert float(pools[0].codes[0, 0, 0, 9].float()) == float(ref.nearest(torch.tensor([top / s]).double(), code))


def test_counts_places_and_entries_that_are_not_written():
    """Padded rows, rows of none, negative positions, positions and entries outside."""
    table = torch.tensor([[0, 1], [2, 3], [4, -1], [5, 99], [6, 7], [-1, 8]], dtype=torch.int32)
    check(6, 2, 40, 64, 32, 32, E4M3, F16, [0, -5, 20, 20, 50, 3], counts=[7, 40, 40, 40, 40, 40], table=table, width=2)
    check(6, 2, 40, 64, 32, 32, INT8, F16, [0, -60, 2 ** 31 - 10, 63, 64, 0], counts=[0, 40, 40, -3, 40, 99],
          table=table, width=2)
    check(6, 2, 1, 64, 32, 32, INT8, F16, [0, -1, 2 ** 31 - 1, 63, 64, 0], table=table, width=2)


def test_strides_and_copies():
    """Token-major inputs as they lie, rows off 16 bytes through a copy, strided pools."""
    from tritonkv_amd.paged8 import Paged8Pool, paged8_append

    x = [values(2, 2, 40, 64, F16, s) for s in (1, 2)]
    table, pos = ref.make_table(2, 2, 4, 3).cuda(), ints([3, 30])
    a = [ref.make_pool(4, 2, 64, 64, E4M3, 32, 1) for _ in range(2)]
    paged8_append(*a, *(y.cuda() for y in x), table, pos)
    store = torch.empty(4, 64, 2, 2, 64, dtype=E4M3, device="cuda")
    scales = torch.empty(2, 2, 4, 2, device="cuda")
    b = [Paged8Pool(store[:, :, i].transpose(1, 2), scales[:, i].permute(1, 2, 0)) for i in range(2)]
    fresh = ref.make_pool(4, 2, 64, 64, E4M3, 32, 1)
    for p in b:
        p.codes.view(torch.int8).copy_(fresh.codes.view(torch.int8))
        p.scale.copy_(fresh.scale)
    odd = [torch.empty(2, 2, 40, 65, dtype=F16, device="cuda")[..., 1:] for _ in range(2)]
    for o, y in zip(odd, x):
        o.copy_(y)
    paged8_append(*b, *odd, table, pos)
    for p, q in zip(a, b):
        assert torch.equal(p.codes.view(torch.int8), q.codes.view(torch.int8)) and torch.equal(p.scale, q.scale)


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,dims,N", [(128, 128, 1), (128, 128, 50), (64, 32, 7), (256, 256, 40), (128, 16, 33)])
def test_rotary_on_the_way(code, interleaved, D, dims, N):
    """Keys are turned in 32 bits and rounded once, queries as by apply_rotary."""
    from tritonkv_amd.paged8 import paged8_append
    from tritonkv_amd.rotary import Rotary, apply_rotary

    B, HQ, HKV, page, block = 3, 4, 2, 64, 32
    pos, counts = [0, 37, 100], None if N == 1 else [N, N // 2, N - 1]
    k, v = (ref.make_pool(9, HKV, page, D, code, block, s) for s in (1, 2))
    table = ref.make_table(B, 3, 9, 3)
    kn, vn = (values(B, HKV, N, D, BF16, s, token_major=True) for s in (1, 2))
    q = values(B, HQ, N, D, BF16, 7, token_major=True)
    w = torch.tensor([10000.0 ** (-2.0 * i / dims) for i in range(dims // 2)], dtype=torch.float64)
    rot = Rotary(inv_freq=w.cuda(), interleaved=interleaved, factor=1.1)
    t = torch.tensor(pos)[:, None] + torch.arange(N)
    turned = ref.turn(kn.double(), t[:, None], w, interleaved, 1.1)
    want = []
    for pool, new in ((k, turned), (v, vn.double())):
        c, s = ref.numbers(pool)
        ref.append(c, s, new, table, pos, counts, code, block)
        want.append((c, s))
    out = torch.full((B, HQ, N, D), 3.0, device="cuda").bfloat16()
    got = paged8_append(k, v, kn.cuda(), vn.cuda(), table.cuda(), ints(pos), ints(counts), rotary=rot, q=q.cuda(),
                        q_out=out)
    assert got is out
    plain = apply_rotary(q.cuda(), None, ints(pos), rot)[0]
    for b in range(B):
        n = N if counts is None else counts[b]
        assert torch.equal(out[b, :, :n], plain[b, :, :n]) and (out[b, :, n:] == 3.0).all()
    (kc, ks), (vc, vs) = ref.numbers(k), ref.numbers(v)
    assert torch.equal(ks, want[0][1]) and torch.equal(vs, want[1][1]) and torch.equal(vc, want[1][0])
    # a code may be the other neighbour where the turned value lies on a border, at most 8 * 2^-24 of its pair off
    d = (kc - want[0][0]).abs()
    step = torch.ones_like(d) if code is INT8 else torch.exp2(torch.floor(torch.log2(kc.abs().clamp(min=2.0 ** -6))) - 3)
    assert (d <= 2 * step).all() and (d > 0).double().mean() < 1e-3
    # in place, and a new tensor of zeros
    q2 = q.cuda()
    assert paged8_append(k, v, kn.cuda(), vn.cuda(), table.cuda(), ints(pos), ints(counts), rotary=rot, q=q2, q_out=q2) is q2
    fresh = paged8_append(k, v, kn.cuda(), vn.cuda(), table.cuda(), ints(pos), ints(counts), rotary=rot, q=q.cuda())
    for b in range(B):
        n = N if counts is None else counts[b]
        assert torch.equal(q2[b, :, :n], plain[b, :, :n]) and torch.equal(q2[b, :, n:], q.cuda()[b, :, n:])
        assert torch.equal(fresh[b, :, :n], plain[b, :, :n]) and not fresh[b, :, n:].any()


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_read(code, dtype, D):
    """Code times scale, rounded once; rows behind a count and places outside are left alone."""
    from tritonkv_amd.paged8 import paged8_read

    k, v = (ref.make_pool(7, 2, 96, D, code, 32, s) for s in (1, 2))
    table = torch.tensor([[3, 0], [1, 6], [5, -1], [2, 77]], dtype=torch.int32)
    pos, counts, N = [0, 90, 95, -2], [130, 101, 50, 200], 101
    out = tuple(torch.full((4, N, 2, D), 5.0, device="cuda", dtype=dtype).transpose(1, 2) for _ in range(2))
    got = paged8_read(k, v, table.cuda(), ints(pos), ints(counts), out=out)
    assert got[0] is out[0] and got[1] is out[1]
    written = torch.zeros(4, 2, N, 1, dtype=torch.bool)
    for pool, y in zip((k, v), got):
        c, s = ref.numbers(pool)
        full = (c.view(7, 2, 3, 32, D) * s[..., None, None]).view(7, 2, 96, D)
        want = torch.full((4, 2, N, D), 5.0, dtype=torch.float64)
        for b in range(4):
            for n in range(min(N, counts[b])):
                t = pos[b] + n
                if 0 <= t < 192 and 0 <= int(table[b, t // 96]) < 7:
                    want[b, :, n] = full[int(table[b, t // 96]), :, t % 96]
                    written[b, :, n] = True
        assert torch.equal(y.cpu().double(), want.float().to(dtype).double())
    new = paged8_read(k, v, table.cuda(), ints(pos), ints(counts), tokens=N, dtype=dtype)
    assert torch.equal(new[0], torch.where(written.cuda(), out[0], 0.0))
    assert paged8_read(k, v, table.cuda(), tokens=0, dtype=dtype)[0].shape == (4, 2, 0, D)
    assert torch.equal(paged8_read(k, v, table.cuda()[:2], tokens=96, dtype=dtype)[1],
                       paged8_read(k, v, table.cuda()[:2], ints([0, 0]), ints([96, 96]), 96, dtype)[1])


def test_kept_calls_streams_and_graphs():
    from tritonkv_amd.paged8 import paged8_append, paged8_read
    from tritonkv_amd.rotary import Rotary

    table, pos = ref.make_table(2, 2, 4, 3).cuda(), ints([0, 33])
    rot = Rotary(64)
    x = [[values(2, h, 1, 64, BF16, 9 * i + h).cuda() for h in (2, 2, 4)] for i in range(3)]
    x = [(k, v + 1, q) for k, v, q in x]

    def fresh():
        return [[ref.make_pool(4, 2, 64, 64, E4M3, 32, 10 * i + s) for s in (1, 2)] for i in range(2)]

    def same(a, b):
        return all(torch.equal(p.codes.view(torch.int8), q.codes.view(torch.int8)) and torch.equal(p.scale, q.scale)
                   for r, s in zip(a, b) for p, q in zip(r, s))

    a, b = fresh(), fresh()
    ws: dict = {}
    outs = [torch.zeros_like(q) for _, _, q in x]
    for k, v, q in x:
        for layer_a, layer_b in zip(a, b):
            want = paged8_append(*layer_a, k, v, table, pos, rotary=rot, q=q)
            o = torch.zeros_like(q)
            assert torch.equal(paged8_append(*layer_b, k, v, table, pos, None, ws, rotary=rot, q=q, q_out=o), want)
        pos.add_(1)
    assert "call" in ws and same(a, b)
    # without rotary, the same workspace
    paged8_append(*a[0], x[0][0], x[0][1], table, pos)
    paged8_append(*b[0], x[0][0], x[0][1], table, pos, None, ws)
    assert same(a, b)
    # captured: follows the positions, on what the pools hold then
    graph, pools = torch.cuda.CUDAGraph(), fresh()[0]
    ws2: dict = {}
    read = tuple(torch.zeros(2, 2, 8, 64, device="cuda") for _ in range(2))
    paged8_append(*pools, x[1][0], x[1][1], table, pos, None, ws2, rotary=rot, q=x[1][2], q_out=outs[1])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        paged8_append(*pools, x[1][0], x[1][1], table, pos, None, ws2, rotary=rot, q=x[1][2], q_out=outs[1])
        paged8_read(*pools, table, pos, out=read, _workspace={})
    for p in ([5, 40], [0, 64], [100, 1]):
        pos.copy_(ints(p))
        eager = fresh()[0]
        for u, w in zip(eager, pools):
            u.codes.view(torch.int8).copy_(w.codes.view(torch.int8))
            u.scale.copy_(w.scale)
        want = paged8_append(*eager, x[1][0], x[1][1], table, pos, rotary=rot, q=x[1][2])
        back = paged8_read(*eager, table, pos, tokens=8, dtype=F32)
        for r in read:
            r.zero_()
        graph.replay()
        assert torch.equal(outs[1], want) and same([pools], [eager])
        assert all(torch.equal(r, w) for r, w in zip(read, back))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged8_append(*b[0], x[2][0], x[2][1], table, pos, None, ws)
    side.synchronize()
    paged8_append(*a[0], x[2][0], x[2][1], table, pos)
    assert same(a, b)


def test_a_serving_run():
    """A prompt, steps and a draft through append, fork, decode and read, against the same run in 64 bits."""
    from tritonkv_amd.pages import fork_rows, resize_rows
    from tritonkv_amd.paged8 import empty_paged8_pool, paged8_append, paged8_decode_attention, paged8_read
    from tritonkv_amd.rotary import Rotary

    B, HQ, HKV, D, page, block, P = 3, 4, 1, 64, 32, 32, 24
    k, v = (empty_paged8_pool(P, HKV, page, D, E4M3, block) for _ in range(2))
    for p in (k, v):
        p.codes.view(torch.int8).zero_()
    rot = Rotary(D)
    table = torch.full((B, 6), -1, dtype=torch.int32, device="cuda")
    lens, refs = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (B, P))
    w = rot.inv_freq.cpu()

    def step(n, counts, seed, host):
        kn, vn, q = (values(B, h, n, D, BF16, seed + i, token_major=True) for i, h in enumerate((HKV, HKV, HQ)))
        before = lens.clone()
        c = ints(counts)
        assert int(resize_rows([k, v], table, lens, refs, lens + c)) == 0
        qr = paged8_append(k, v, kn.cuda(), vn.cuda(), table, before, c, rotary=rot, q=q.cuda())
        t = before.cpu()[:, None] + torch.arange(n)
        turned = ref.turn(kn.double(), t[:, None], w)
        ref.append(*host[0], turned, table.cpu(), before.cpu(), counts, E4M3, block)
        ref.append(*host[1], vn.double(), table.cpu(), before.cpu(), counts, E4M3, block)
        (kc, ks), (vc, vs) = ref.numbers(k), ref.numbers(v)
        assert torch.equal(ks, host[0][1]) and torch.equal(vc, host[1][0])
        assert ((kc - host[0][0]) != 0).double().mean() < 1e-3
        return qr, c

    host = [[x.clone() for x in ref.numbers(p)] for p in (k, v)]
    step(50, [50, 33, 1], 1, host)
    for i in range(3):
        qr, c = step(1, [1, 1, 1], 10 + 3 * i, host)
        got = paged8_decode_attention(qr, k, v, table, lens)
        want = ref.decode(qr.cpu(), ref.numbers(k), ref.numbers(v), table.cpu(), lens.tolist(), None, 0.125)
        ref.assert_within(got, want[0], want[2])
    # row 2 goes on as a copy of row 0: the partial page is copied, scales too
    assert int(fork_rows([k, v], table, lens, refs, ints([0, 1, 0]))) == 0
    a, b = (paged8_read(k, v, table[[r]], tokens=53, dtype=F32) for r in (0, 2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and int(table[0, 1]) != int(table[2, 1])
    host = [[x.clone() for x in ref.numbers(p)] for p in (k, v)]
    qr, c = step(4, [4, 2, 3], 40, host)
    got = paged8_decode_attention(qr, k, v, table, lens, counts=c)
    want = ref.decode(qr.cpu(), ref.numbers(k), ref.numbers(v), table.cpu(), lens.tolist(), [4, 2, 3], 0.125)
    ref.assert_within(got, want[0], want[2])
