"""16-bit page pools on the GPU: the decode and the append against a plain
implementation in 64 bits, at the lengths, pages, strides and masks where they
can go wrong.

Tolerances, fixed before the first run.  Keys, values and queries are exact in
64 bits, so what separates the two is the kernel's own arithmetic:

* a score is a dot of D exact products accumulated in fp32; counted as D / 8
  sequential roundings of partial sums of at most ``A = max_t sum_d |q_d k_td|
  * scale``, plus 4 for the scale, the maximum and the exponential, its error is
  at most ``e = (D / 8 + 4) * 2**-24 * max(A, 1)``;
* p enters the products in terms that hold at least 22 bits, and the sums of p
  and of p * v run over at most n / 4 sequential steps of a wave and its joins,
  whose roundings average out: counted as sqrt(n) * 2**-24;
* numerator and denominator each carry that relative error, so ``|out - exact| <=
  2 * (e + 2**-21 + sqrt(n) * 2**-24) * max |v|``.

That bound is the worst case for one element; over a whole output the errors
have random signs, and the 2-norm of the difference stays below 1e-5 of the
result's (p rounded once to fp16 would give 2e-4, to bf16 2e-3).
``lse`` is the score's error plus one logarithm: ``e + 2**-21 * max(1, |lse|)``.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


def _table(lens, page, width, num_pages, g, spare=0):
    """Distinct pages in random order for every row's tokens, -1 after them."""
    order = torch.randperm(num_pages, generator=g).tolist()
    rows = []
    for n in lens:
        k = -(-max(0, min(n, width * page)) // page)
        rows.append([order.pop() for _ in range(k)] + [-1] * (width - k))
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def _case(lens, HQ, HKV, D, page, width, dtype, seed=0, poison=True):
    """q, pools and table; everything a row does not hold is NaN or Inf."""
    g = torch.Generator().manual_seed(seed)
    clamped = [max(0, min(n, width * page)) for n in lens]
    num_pages = sum(-(-n // page) for n in clamped) + 2
    table = _table(lens, page, width, num_pages, g)
    kp = torch.randn(num_pages, HKV, page, D, generator=g).to(dtype)
    vp = torch.randn(num_pages, HKV, page, D, generator=g).to(dtype)
    if poison:
        live = torch.zeros(num_pages, page, dtype=torch.bool)
        for row, n in zip(table.tolist(), clamped):
            for i, p in enumerate(row):
                if p >= 0:
                    live[p, :max(0, min(page, n - i * page))] = True
        kp.permute(0, 2, 1, 3)[~live] = math.nan
        vp.permute(0, 2, 1, 3)[~live] = math.inf
    q = torch.randn(len(lens), HQ, D, generator=g).to(dtype)
    return q.to(DEV), kp.to(DEV), vp.to(DEV), table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def _rows(pool, table, b, n):
    """Row b's first n tokens in 64 bits: (HKV, n, D)."""
    page = pool.shape[2]
    at = table[b, :-(-n // page)].long().clamp(0, pool.shape[0] - 1)
    return pool[at].double().transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def _reference(q, kp, vp, table, lens, scale=None):
    """out, lse and the two tolerances."""
    B, HQ, D = q.shape
    HKV, page = kp.shape[1], kp.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, HQ, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, HQ), -math.inf, dtype=torch.float64, device=q.device)
    e, vmax, longest = 0.0, 0.0, 1
    for b in range(B):
        n = table.shape[1] * page if lens is None else max(0, min(int(lens[b]), table.shape[1] * page))
        if not n:
            continue
        k, v = _rows(kp, table, b, n), _rows(vp, table, b, n)
        qb = q[b].double().view(HKV, HQ // HKV, D)
        s = torch.matmul(qb, k.transpose(1, 2).contiguous()) * scale
        out[b] = torch.matmul(torch.softmax(s, -1), v).view(HQ, D)
        lse[b] = torch.logsumexp(s, -1).view(HQ)
        size = float(torch.matmul(qb.abs(), k.abs().transpose(1, 2).contiguous()).max()) * abs(scale)
        e = max(e, (D / 8 + 4) * 2.0 ** -24 * max(size, 1.0))
        vmax, longest = max(vmax, float(v.abs().max())), max(longest, n)
    return out, lse, 2 * (e + 2.0 ** -21 + math.sqrt(longest) * 2.0 ** -24) * vmax, e


def _check(got, lse, q, kp, vp, table, lens, scale=None):
    want, wlse, tol, e = _reference(q, kp, vp, table, lens, scale)
    d = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert float(d.max()) <= tol, (float(d.max()), tol)
    norm = float(want.norm())
    assert norm == 0 or float(d.norm()) <= 1e-5 * norm, float(d.norm()) / norm
    if lse is not None:
        empty = torch.isinf(wlse)
        assert torch.equal(torch.isinf(lse), empty) and (lse[empty] < 0).all()
        dl = (lse.double() - wlse)[~empty].abs()
        if dl.numel():
            assert float((dl - 2.0 ** -21 * wlse[~empty].abs().clamp(min=1)).max()) <= e


def _decode(q, kp, vp, table, lens, **kw):
    from tritonkv_amd.paged16 import paged16_decode_attention

    lse = torch.full(q.shape[:2], math.nan, device=DEV)
    out = torch.full(q.shape, math.nan, device=DEV)
    got = paged16_decode_attention(q, kp, vp, table, lens, out=out, lse=lse, **kw)
    assert got is out
    return got, lse


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 384]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 48, 128])
@pytest.mark.parametrize("piece", [None, 32, 96, 4096], ids=["auto", "32", "96", "whole"])
def test_lengths_around_every_edge(dtype, D, page, piece):
    case = _case(EDGES, 6, 2, D, page, 384 // page, dtype, seed=D + page)
    _check(*_decode(*case, piece_tokens=piece), *case)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("HQ,HKV", [(1, 1), (2, 2), (5, 1), (12, 2), (16, 16), (16, 1), (17, 1), (24, 1),
                                    (40, 1), (64, 8), (66, 2)])
def test_head_layouts(dtype, HQ, HKV):
    case = _case([1, 130, 0, 511, 700], HQ, HKV, 128, 64, 12, dtype, seed=HQ)
    _check(*_decode(*case), *case)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("G", [16, 17, 31, 32, 33, 64])
def test_head_blocks_of_other_head_dims(D, G):
    case = _case([1, 300, 65], 2 * G, 2, D, 16, 20, BF16, seed=G)
    _check(*_decode(*case), *case)
    _check(*_decode(*case, piece_tokens=64), *case)


def test_thousands_of_rows_and_large_pages():
    g = torch.Generator().manual_seed(22)
    lens = torch.randint(0, 90, (5000,), generator=g).tolist()
    case = _case(lens, 2, 1, 64, 16, 40, F16, seed=22)  # tables of 640 tokens: cut, and joined
    out, lse = _decode(*case)
    at = list(range(0, 5000, 97)) + [4999]
    q, kp, vp, table, lens = case
    _check(out[at], lse[at], q[at], kp, vp, table[at], lens[at])
    case = _case([5000, 1, 4096, 4097], 4, 2, 128, 4096, 2, BF16, seed=23)
    _check(*_decode(*case), *case)


def test_one_workspace_for_every_layer():
    from tritonkv_amd.paged16 import paged16_append, paged16_decode_attention

    ws, wa = {}, {}
    for seed in range(3):
        q, kp, vp, table, lens = _case([300, 5, 64], 8, 2, 128, 64, 8, BF16, seed=seed)
        new = torch.randn(2, 3, 2, 1, 128, device=DEV).to(BF16)
        want_k, want_v = kp.clone(), vp.clone()
        paged16_append(want_k, want_v, new[0], new[1], table, lens - 1)
        paged16_append(kp, vp, new[0], new[1], table, lens - 1, _workspace=wa)
        assert torch.equal(kp.view(torch.int16), want_k.view(torch.int16))
        assert torch.equal(vp.view(torch.int16), want_v.view(torch.int16))
        out = paged16_decode_attention(q, kp, vp, table, lens, _workspace=ws)
        _check(out, None, q, kp, vp, table, lens)
        prep = (ws["call"], wa["call"]) if seed == 0 else prep
        assert (ws["call"], wa["call"]) == prep


def test_two_calls_at_once():
    from tritonkv_amd.paged16 import paged16_decode_attention

    cases = [_case([9000, 20, 400], 8, 2, 128, 64, 160, BF16, seed=s) for s in (30, 31)]
    want = [paged16_decode_attention(*c) for c in cases]
    streams, ws = [torch.cuda.Stream() for _ in cases], [{} for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged16_decode_attention(*cases[i], _workspace=ws[i]))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)


def test_expanded_queries_and_one_pool_for_both():
    q, kp, vp, table, lens = _case([300, 5, 64], 8, 2, 128, 64, 8, F16, seed=32)
    one = q[:1].expand(3, 8, 128)
    _check(*_decode(one, kp, kp.clone(), table, lens), one, kp, kp, table, lens)
    got, _ = _decode(one, kp, kp, table, lens)
    assert torch.equal(got, _decode(one.contiguous(), kp, kp.clone(), table, lens)[0])


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (256, F16)])
def test_a_long_row_among_short_ones(D, dtype):
    case = _case([20011, 3, 0, 1000, 64], 8, 2, D, 64, 400, dtype, seed=3)
    _check(*_decode(*case), *case)
    _check(*_decode(*case, piece_tokens=20032), *case)  # 157 chunks a wave: the tiles are looked up anew


def test_many_rows():
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 700, (333,), generator=g).tolist()
    case = _case(lens, 4, 2, 64, 32, 25, F16, seed=9)
    _check(*_decode(*case), *case)
    _check(*_decode(*case, piece_tokens=64), *case)
    case = _case([0] * 100, 4, 2, 64, 32, 25, F16, seed=9)
    out, lse = _decode(*case)
    assert not out.any() and torch.isinf(lse).all()


def test_lengths_outside_the_table_are_clamped():
    case = _case([500, 96, 0], 4, 1, 128, 32, 3, F16, seed=4)
    q, kp, vp, table, lens = case
    lens.copy_(torch.tensor([2 ** 31 - 1, 96, -2 ** 31], device=DEV))
    _check(*_decode(*case), *case)
    q, kp, vp, table, _ = _case([96, 96], 4, 1, 128, 32, 3, F16, seed=5)
    out, lse = _decode(q, kp, vp, table, None)  # every row holds its table's capacity
    _check(out, lse, q, kp, vp, table, None)


def test_table_entries_outside_the_pool_are_clamped():
    q, kp, vp, table, lens = _case([96, 96], 4, 1, 128, 32, 3, F16, seed=6, poison=False)
    table[0, 1], table[1, 2] = -7, 2 ** 31 - 1
    out, lse = _decode(q, kp, vp, table, lens)
    _check(out, lse, q, kp, vp, table.clamp(0, kp.shape[0] - 1), lens)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.5])
def test_scales(scale):
    case = _case([1, 77, 300], 8, 2, 128, 64, 5, BF16, seed=7)
    _check(*_decode(*case, sm_scale=scale, piece_tokens=96), *case, scale)


def test_sharp_and_far_scores():
    """One token far above the others, and all scores far from zero."""
    q, kp, vp, table, lens = _case([300, 300], 4, 1, 128, 64, 5, F16, seed=8)
    q.mul_(6)
    _check(*_decode(q, kp, vp, table, lens, piece_tokens=64), q, kp, vp, table, lens)
    kp[..., 0] = torch.where(torch.isnan(kp[..., 0]), kp[..., 0], 60.0)
    q[..., 0] = -20.0
    _check(*_decode(q, kp, vp, table, lens, piece_tokens=64), q, kp, vp, table, lens)


def test_flat_scores_over_a_long_row_keep_their_precision():
    """Every p small beside the largest: the low terms of P carry them."""
    q, kp, vp, table, lens = _case([8192], 2, 1, 128, 128, 64, F16, seed=10)
    kp[int(table[0, 0]), 0, 5] = 14 * q[0, 0] / q[0, 0].norm()
    for dtype in (F16, BF16):
        c = (q.to(dtype), kp.to(dtype), vp.to(dtype), table, lens)
        _check(*_decode(*c), *c)


def test_nonfinite_values_in_the_row_show_as_in_softmax():
    q, kp, vp, table, lens = _case([200, 200, 200, 200], 4, 2, 128, 64, 4, F16, seed=11)
    kp[int(table[0, 1]), 0, 3, 7] = math.nan     # row 0, kv head 0: scores NaN
    vp[int(table[1, 0]), 1, 2, 9] = math.inf     # row 1, kv head 1, dim 9
    kp[int(table[2, 2]), 1, 1] = -math.inf * q[2, 2].sign()  # heads 2, 3 of row 2
    out, lse = _decode(q, kp, vp, table, lens, piece_tokens=64)
    assert torch.isnan(out[0, :2]).all() and torch.isnan(lse[0, :2]).all()
    assert torch.isfinite(out[0, 2:]).all()
    assert torch.isinf(out[1, 2:, 9]).all() and torch.isfinite(out[1, :2]).all()
    assert torch.isfinite(out[1, 2:, :9]).all() and torch.isfinite(out[1, 2:, 10:]).all()
    assert torch.isfinite(out[3]).all() and torch.isfinite(out[2, :3]).all()  # head 2: one score of -inf


def test_a_row_whose_scores_are_all_minus_infinity_is_zero():
    q, kp, vp, table, lens = _case([70, 70], 2, 1, 64, 32, 3, F16, seed=12)
    q[0] = 0
    q[0, :, 0] = 1
    live = ~torch.isnan(kp[..., 0])
    kp[..., 0] = torch.where(live, torch.tensor(-math.inf, dtype=F16, device=DEV), kp[..., 0])
    q[1, :, 0] = 1
    for piece in (32, 96):
        out, lse = _decode(q, kp, vp, table, lens, piece_tokens=piece)
        assert not out.any() and (lse == -math.inf).all()


def _views(kp, vp, form):
    if form == "token_major":
        return [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kp, vp)]
    if form == "paired":  # K and V of a page side by side
        both = torch.stack([kp, vp], 1)
        return [both[:, 0], both[:, 1]]
    wide = [torch.full((*x.shape[:3], 2 * x.shape[3]), math.nan, dtype=x.dtype, device=x.device) for x in (kp, vp)]
    for w, x in zip(wide, (kp, vp)):
        w[..., 8:8 + x.shape[3]] = x
    return [w[..., 8:8 + kp.shape[3]] for w in wide]


@pytest.mark.parametrize("form", ["token_major", "paired", "wide_rows"])
@pytest.mark.parametrize("append", [False, True])
def test_strided_pools_and_queries(form, append):
    q, kp, vp, table, lens = _case([1, 100, 0, 290], 8, 4, 128, 48, 8, BF16, seed=13)
    kw = {}
    if append:
        new = torch.randn(4, 2, 4, 128, device=DEV).to(BF16)
        kw = dict(k_new=new[:, 0], v_new=new[:, 1])
    qkv = torch.randn(4, 16, 128, device=DEV).to(BF16)  # q as rows of a joint projection
    ws = {}
    for _ in range(2):
        ks, vs = _views(kp, vp, form)
        want, wl = _decode(q, kc := kp.clone(), vc := vp.clone(), table, lens, **kw)
        got, gl = _decode(q, ks, vs, table, lens, _workspace=ws, **kw)
        assert torch.equal(got, want) and torch.equal(gl, wl)
        assert torch.equal(ks.nan_to_num(), kc.nan_to_num()) and torch.equal(vs.nan_to_num(), vc.nan_to_num())
    got, _ = _decode(qkv[:, 4:12], ks, vs, table, lens, _workspace=ws, **kw)
    assert torch.equal(got, _decode(qkv[:, 4:12].contiguous(), ks, vs, table, lens, **kw)[0])
    odd = torch.randn(4, 8, 129, device=DEV).to(BF16)[..., 1:]  # rows off their 16 bytes: copied
    assert torch.equal(_decode(odd, ks, vs, table, lens, _workspace=ws, **kw)[0],
                       _decode(odd.contiguous(), ks, vs, table, lens, **kw)[0])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("HQ", [4, 40])
@pytest.mark.parametrize("piece", [None, 32], ids=["auto", "32"])
def test_the_fused_append_is_the_append_and_the_decode(dtype, D, HQ, piece):
    from tritonkv_amd.paged16 import paged16_append

    q, kp, vp, table, lens = _case(EDGES, HQ, 2, D, 48, 8, dtype, seed=14)
    new = torch.randn(2, len(EDGES), 2, D, device=DEV).to(dtype)
    ka, va = kp.clone(), vp.clone()
    paged16_append(ka, va, new[0][:, :, None], new[1][:, :, None], table, lens - 1)
    want = _decode(q, ka, va, table, lens, piece_tokens=piece)
    got = _decode(q, kp, vp, table, lens, k_new=new[0], v_new=new[1], piece_tokens=piece)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    bits = torch.int16
    assert torch.equal(kp.view(bits), ka.view(bits)) and torch.equal(vp.view(bits), va.view(bits))
    _check(*got, q, kp, vp, table, lens)


def test_a_new_token_without_a_page_is_attended_and_not_stored():
    q, kp, vp, table, lens = _case([33, 40], 4, 2, 128, 32, 2, F16, seed=15)
    table[0, 1] = -1
    new = torch.randn(2, 2, 2, 128, device=DEV).to(F16)
    kb, vb = kp.clone(), vp.clone()
    out, _ = _decode(q, kp, vp, table, lens, k_new=new[0], v_new=new[1])
    kb[int(table[1, 1]), :, 7], vb[int(table[1, 1]), :, 7] = new[0, 1], new[1, 1]
    bits = torch.int16
    assert torch.equal(kp.view(bits), kb.view(bits)) and torch.equal(vp.view(bits), vb.view(bits))
    spare = torch.cat([kp, kp[:1]]), torch.cat([vp, vp[:1]])
    spare[0][-1, :, 0], spare[1][-1, :, 0] = new[0, 0], new[1, 0]
    table[0, 1] = kp.shape[0]
    _check(out, None, q, *spare, table, lens)


def test_joining_two_caches_by_their_lse():
    q, kp, vp, table, lens = _case([500, 37], 8, 2, 128, 32, 16, F16, seed=16)
    want, wl = _decode(q, kp, vp, table, lens)
    first = torch.tensor([256, 32], dtype=torch.int32, device=DEV)
    a, la = _decode(q, kp, vp, table, first)
    rest = torch.stack([torch.roll(table[0], -8), torch.roll(table[1], -1)]).contiguous()
    b, lb = _decode(q, kp, vp, rest, lens - first)
    l = torch.logaddexp(la, lb)
    joined = a * (la - l).exp()[..., None] + b * (lb - l).exp()[..., None]
    assert torch.allclose(joined, want, atol=1e-5, rtol=0) and torch.allclose(l, wl, atol=1e-5, rtol=0)


def test_captured_step_follows_lengths_and_tables():
    """A graph of the step with its append, replayed while rows grow; its workspace is
    used by an eager call and another graph in between."""
    from tritonkv_amd.paged16 import paged16_decode_attention

    q, kp, vp, table, lens = _case([500, 40, 0, 900], 8, 2, 128, 64, 16, F16, seed=17, poison=False)
    full = _case([1024] * 4, 8, 2, 128, 64, 16, F16, seed=18, poison=False)
    kp, vp, table = full[1], full[2], full[3]
    new = torch.randn(2, 4, 2, 128, device=DEV).to(F16)
    ws = {}
    outs = [torch.empty(4, 8, 128, device=DEV) for _ in range(2)]

    def step(out):
        paged16_decode_attention(q, kp, vp, table, lens, out=out, _workspace=ws, k_new=new[0], v_new=new[1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(outs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for out in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(out)
        graphs.append(graph)
    for n in range(4):
        lens.copy_(torch.tensor([500 + 33 * n, 40 + n, n, 1024 - n], device=DEV))
        new.copy_(torch.randn(2, 4, 2, 128, device=DEV))
        graphs[n % 2].replay()
        small = paged16_decode_attention(q[:2], kp, vp, table[:2], lens[:2], _workspace=ws, piece_tokens=64)
        torch.cuda.synchronize()
        _check(outs[n % 2], None, q, kp, vp, table, lens)
        _check(small, None, q[:2], kp, vp, table[:2], lens[:2])


def test_another_stream_and_repeated_calls():
    from tritonkv_amd.paged16 import paged16_decode_attention

    case = _case([300, 5, 64], 8, 2, 128, 64, 8, BF16, seed=19)
    q, kp, vp, table, lens = case
    want = paged16_decode_attention(*case)
    ws, out = {}, torch.empty(3, 8, 128, device=DEV)
    paged16_decode_attention(*case, out=out, _workspace=ws)
    prep = ws.get("call")
    assert torch.equal(out, want) and prep is not None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.empty(1 << 26, device=DEV).zero_()  # the call has to wait for its own stream
        q2 = (q.float() * (1 + big[:1])).to(BF16)
        got = paged16_decode_attention(q2, kp, vp, table, lens, _workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and ws["call"] is prep
    lens.fill_(17)  # lengths change in place; row 1 holds 5 tokens, the rest of its page is NaN
    got = paged16_decode_attention(*case, _workspace=ws)
    assert ws["call"] is prep and torch.isnan(got[1]).all()
    _check(got[::2], None, q[::2], kp, vp, table[::2], lens[::2])
    lens[1] = 5
    for other in ((q, kp, vp, table.clone(), lens), (q, kp, vp, table, lens.clone()), (q, kp.clone(), vp, table, lens)):
        assert torch.equal(paged16_decode_attention(*other, _workspace=ws), paged16_decode_attention(*other))
    assert torch.equal(paged16_decode_attention(*case, sm_scale=0.2, _workspace=ws),
                       paged16_decode_attention(*case, sm_scale=0.2))
    with pytest.raises(TypeError):
        paged16_decode_attention(q.to(F16), kp, vp, table, lens, out=out, _workspace=ws)
    with pytest.raises(ValueError):
        paged16_decode_attention(q, kp, vp, table, lens.long(), out=out, _workspace=ws)


def test_the_result_does_not_depend_on_the_call():
    case = _case([3000, 1, 777, 0], 8, 2, 128, 64, 48, F16, seed=20)
    first = _decode(*case)
    for _ in range(3):
        again = _decode(*case)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_a_pool_past_32_bit_offsets():
    """Pages beyond 4 GiB of a pool are read and written at their place."""
    from tritonkv_amd.paged16 import paged16_append, paged16_decode_attention

    D, page, HKV = 128, 64, 8
    num_pages = (9 << 30) // (HKV * page * D * 2)
    kp = torch.zeros(num_pages, HKV, page, D, dtype=F16, device=DEV)
    vp = torch.zeros_like(kp)
    table = torch.tensor([[num_pages - 1, 0, num_pages // 2 + 1, -1]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(21)
    x = torch.randn(2, 1, HKV, 180, D, generator=g).to(F16).to(DEV)
    paged16_append(kp, vp, x[0], x[1], table, torch.zeros(1, dtype=torch.int32, device=DEV))
    assert torch.equal(kp[num_pages // 2 + 1, :, :52], x[0, 0, :, 128:])
    assert torch.equal(vp[num_pages - 1], x[1, 0, :, :64])
    q = torch.randn(1, 8, D, generator=g).to(F16).to(DEV)
    lens = torch.tensor([180], dtype=torch.int32, device=DEV)
    _check(paged16_decode_attention(q, kp, vp, table, lens), None, q, kp, vp, table, lens)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------


def _append_plain(pool, x, table, pos, counts):
    pool = pool.clone()
    page = pool.shape[2]
    for b in range(x.shape[0]):
        for n in range(x.shape[2] if counts is None else max(0, min(int(counts[b]), x.shape[2]))):
            t = int(pos[b]) + n
            if 0 <= t < table.shape[1] * page:
                p = int(table[b, t // page])
                if 0 <= p < pool.shape[0]:
                    pool[p, :, t % page] = x[b, :, n].to(pool.dtype)
    return pool


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("x", [F16, BF16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 48), (256, 32)])
@pytest.mark.parametrize("layout", ["head_major", "token_major", "odd"])
def test_append_bit_for_bit(dtype, x, D, page, layout):
    from tritonkv_amd.paged16 import paged16_append

    B, HKV, N, width = 5, 3, 37, 4
    g = torch.Generator().manual_seed(D)
    num_pages = B * width
    kp, vp = (torch.randn(num_pages, HKV, page, D, generator=g).to(dtype) for _ in range(2))
    table = torch.randperm(num_pages, generator=g).to(torch.int32).view(B, width)
    table[1, 1], table[2, 0] = -1, num_pages
    pos = torch.tensor([0, page - 1, 5, -3, width * page - 10], dtype=torch.int32)
    if layout == "head_major":
        new = [torch.randn(B, HKV, N, D, generator=g).to(x) for _ in range(2)]
    elif layout == "token_major":
        new = [torch.randn(B, N, HKV, D, generator=g).to(x).transpose(1, 2) for _ in range(2)]
    else:
        new = [torch.randn(B, HKV, N, D + 1, generator=g).to(x)[..., 1:] for _ in range(2)]
    new[0][0, 0, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, 1e30]).to(x)
    for counts in (None, torch.tensor([37, 5, 0, 99, -4], dtype=torch.int32)):
        want = [_append_plain(p, n, table, pos, counts) for p, n in zip((kp, vp), new)]
        got = [kp.to(DEV), vp.to(DEV)]
        ws = {}
        for _ in range(2):
            dev = [n.to(DEV) if n.is_contiguous() else
                   (n.transpose(1, 2).to(DEV).transpose(1, 2) if layout == "token_major" else
                    torch.cat([n[..., :1], n], -1).to(DEV)[..., 1:]) for n in new]
            r = paged16_append(got[0], got[1], dev[0], dev[1], table.to(DEV), pos.to(DEV),
                               None if counts is None else counts.to(DEV), _workspace=ws)
            assert r is None
        for a, b in zip(got, want):
            a = a.cpu()
            nan = torch.isnan(b)
            assert torch.equal(torch.isnan(a), nan) and torch.equal(a[~nan], b[~nan])


def test_append_one_token_per_row_and_captured():
    from tritonkv_amd.paged16 import paged16_append

    B, HKV, D, page, width = 33, 8, 128, 64, 3
    kp, vp = (torch.zeros(B * width, HKV, page, D, dtype=BF16, device=DEV) for _ in range(2))
    table = torch.randperm(B * width, device=DEV).to(torch.int32).view(B, width)
    pos = torch.zeros(B, dtype=torch.int32, device=DEV)
    new = torch.randn(2, B, HKV, 1, D, device=DEV).to(BF16)
    ws = {}
    paged16_append(kp, vp, new[0], new[1], table, pos, _workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged16_append(kp, vp, new[0], new[1], table, pos, _workspace=ws)
    wk, wv = kp.clone(), vp.clone()
    for n in range(4):
        pos.fill_(50 + n).add_(torch.arange(B, device=DEV, dtype=torch.int32))
        new.copy_(torch.randn(2, B, HKV, 1, D, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for pool, x in ((wk, new[0]), (wv, new[1])):
            t = pos.long()
            pool[table[torch.arange(B), t // page].long(), :, t % page] = x[:, :, 0]
        assert torch.equal(kp, wk) and torch.equal(vp, wv)
    paged16_append(kp, vp, new[0, :0], new[1, :0], table[:0], pos[:0])
    paged16_append(kp, vp, new[0][:, :, :0], new[1][:, :, :0], table, pos)
    assert torch.equal(kp, wk) and torch.equal(vp, wv)
