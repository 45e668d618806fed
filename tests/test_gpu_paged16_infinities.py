"""Infinities and NaN among the values and keys of live tokens: the 16-bit paged decode gives
what softmax in 32 bits gives, infinite where one sign of infinity is met, NaN where both are.

The oracle is the definition in 64 bits.  Where it is finite the kernel's error is that of
any other row: with scores below 16 and rows of at most 400 tokens of |v| < 8 it is below
2 * ((D / 8 + 4) * 2**-24 * 16 + 2**-21 + 20 * 2**-24) * 8 < 2**-10 for D up to 256.  Scores lie within
60 of each other, so that no p leaves the range of 32 bits."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16
PAGE, WIDTH = 32, 13
LENS = [400, 1, 33, 64, 0, 257]


def _case(dtype, D, HQ, HKV, seed):
    """Rows whose values hold infinities in some dims; everything past a row is NaN."""
    g = torch.Generator().manual_seed(seed)
    B, N = len(LENS), len(LENS) * WIDTH
    table = torch.randperm(N, generator=g).to(torch.int32).view(B, WIDTH)
    k, v = (torch.randn(B, HKV, WIDTH * PAGE, D, generator=g).clamp(-7, 7) for _ in range(2))
    for b, n in enumerate(LENS):
        if n == 0:
            continue
        for dim in range(0, D, 3):  # one infinity, or several of one sign, anywhere in the row
            for t in torch.randint(0, n, (1 + dim % 2,), generator=g).tolist():
                v[b, dim % HKV, t, dim] = math.inf if dim % 4 < 2 else -math.inf
        v[b, :, n - 1, 1], v[b, :, 0, 1] = math.inf, -math.inf  # both signs (the last one's where n is 1)
        v[b, :, n // 2, 4] = math.nan
    q = 0.5 * torch.randn(B, HQ, D, generator=g)
    return q.to(dtype), k.to(dtype), v.to(dtype), table


def _pools(x, table):
    """Rows (B, HKV, T, D) as pages, NaN past the rows."""
    B, HKV, T, D = x.shape
    x = x.clone()
    for b, n in enumerate(LENS):
        x[b, :, n:] = math.nan
    pool = torch.empty(table.numel(), HKV, PAGE, D, dtype=x.dtype)
    pool[table.long()] = x.view(B, HKV, WIDTH, PAGE, D).transpose(1, 2)
    return pool.to(DEV)


def _exact(q, k, v):
    B, HQ, D = q.shape
    HKV = k.shape[1]
    out = torch.zeros(B, HQ, D, dtype=torch.float64)
    for b, n in enumerate(LENS):
        if n == 0:
            continue
        for h in range(HQ):
            kb, vb = k[b, h * HKV // HQ, :n].double(), v[b, h * HKV // HQ, :n].double()
            out[b, h] = (torch.softmax(kb @ q[b, h].double() * D ** -0.5, 0)[:, None] * vb).sum(0)
    return out


def _same(got, want):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    for sign in (1, -1):
        assert torch.equal(got == sign * math.inf, want == sign * math.inf)
    fin = torch.isfinite(want)
    assert float((got - want)[fin].abs().max()) < 2.0 ** -10
    assert fin.any() and torch.isinf(want).any() and torch.isnan(want).any()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("HQ,HKV", [(2, 2), (12, 2), (40, 2), (40, 1)])
@pytest.mark.parametrize("append", [False, True], ids=["decode", "append"])
def test_infinite_values_are_infinite(dtype, D, HQ, HKV, append):
    from tritonkv_amd.paged16 import paged16_decode_attention

    q, k, v, table = _case(dtype, D, HQ, HKV, seed=D + HQ)
    want = _exact(q, k, v)
    lens = torch.tensor(LENS, dtype=torch.int32, device=DEV)
    for piece in (None, 32, 96, 4096):
        kp, vp, kw = _pools(k, table), _pools(v, table), {}
        if append:
            at = [max(0, n - 1) for n in LENS]
            kw = dict(k_new=k[range(len(LENS)), :, at].to(DEV), v_new=v[range(len(LENS)), :, at].to(DEV))
            for b, n in enumerate(LENS):  # their places hold NaN until the call
                if n:
                    for pool in (kp, vp):
                        pool[int(table[b, (n - 1) // PAGE]), :, (n - 1) % PAGE] = math.nan
        got = paged16_decode_attention(q.to(DEV), kp, vp, table.to(DEV), lens, piece_tokens=piece, **kw)
        _same(got, want)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_a_long_row_with_one_infinity(dtype):
    """Many chunks a wave, the infinity in the first one, beside a NaN key elsewhere."""
    from tritonkv_amd.paged16 import paged16_decode_attention

    g = torch.Generator().manual_seed(5)
    n, D = 9000, 128
    q, k, v = (torch.randn(s, generator=g).to(dtype) for s in ((2, 4, D), (2, 2, n, D), (2, 2, n, D)))
    v[0, 0, 3, 7], v[0, 1, n - 1, 8] = math.inf, -math.inf
    k[1, 0, 4500, 0] = math.nan
    pages = -(-n // 64)
    pad = torch.full((2, 2, pages * 64 - n, D), math.nan, dtype=dtype)
    kp, vp = (torch.cat([x, pad], 2).view(2, 2, pages, 64, D).transpose(1, 2).reshape(2 * pages, 2, 64, D).to(DEV)
              for x in (k, v))
    table = torch.arange(2 * pages, dtype=torch.int32, device=DEV).view(2, pages)
    lens = torch.tensor([n, n], dtype=torch.int32, device=DEV)
    for piece in (None, 9024, 512):
        out = paged16_decode_attention(q.to(DEV), kp, vp, table, lens, piece_tokens=piece)
        assert (out[0, :2, 7] == math.inf).all() and (out[0, 2:, 8] == -math.inf).all()
        assert int(torch.isfinite(out[0]).sum()) == 4 * D - 4
        assert torch.isnan(out[1, :2]).all() and torch.isfinite(out[1, 2:]).all()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_an_infinite_value_of_a_token_without_weight(dtype):
    """A score of -inf is a weight of 0: times infinity NaN, as in softmax; any other weight, infinity."""
    from tritonkv_amd.paged16 import paged16_decode_attention

    q = torch.zeros(2, 2, 64, dtype=dtype, device=DEV)
    q[:, :, 0] = 1
    kp, vp = (torch.zeros(4, 1, 32, 64, dtype=dtype, device=DEV) for _ in range(2))
    kp[0, 0, 5, 0] = -math.inf
    kp[2, 0, 5, 0] = -8 * 60  # a weight of e**-60
    vp[0, 0, 5, 3] = vp[2, 0, 5, 3] = math.inf
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    for piece in (32, 64):
        out = paged16_decode_attention(q, kp, vp, table, torch.tensor([50, 50], dtype=torch.int32, device=DEV),
                                       piece_tokens=piece)
        assert torch.isnan(out[0, :, 3]).all() and (out[1, :, 3] == math.inf).all()
        assert not out[..., :3].any() and not out[..., 4:].any()
