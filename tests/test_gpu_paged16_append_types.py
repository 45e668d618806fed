"""Tokens of the other 16-bit type into 16-bit page pools: rounded by the kernel itself, bit for
bit as torch rounds them from fp32, from where they lie, without an allocation."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16


def _same(got, want):
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan].view(torch.int16), want[~nan].view(torch.int16))


@pytest.mark.parametrize("x,pool", [(F16, BF16), (BF16, F16)], ids=["fp16_to_bf16", "bf16_to_fp16"])
def test_every_value_of_the_other_type(x, pool):
    from tritonkv_amd.paged16 import paged16_append

    D, HKV, N = 128, 2, 256
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(x).view(1, HKV, N, D).to(DEV)
    kp, vp = (torch.zeros(4, HKV, 64, D, dtype=pool, device=DEV) for _ in range(2))
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(1, 4)
    paged16_append(kp, vp, every, every.flip(2), table, torch.zeros(1, dtype=torch.int32, device=DEV))
    for p, new in ((kp, every), (vp, every.flip(2))):
        _same(p.transpose(0, 1).reshape(1, HKV, N, D), new.float().to(pool))


@pytest.mark.parametrize("x,pool", [(F16, BF16), (BF16, F16)], ids=["fp16_to_bf16", "bf16_to_fp16"])
@pytest.mark.parametrize("layout", ["head_major", "token_major"])
def test_a_kept_call_reads_them_where_they_lie(x, pool, layout):
    from tritonkv_amd.paged16 import paged16_append

    B, HKV, N, D, page = 3, 4, 21, 64, 16
    kp, vp = (torch.zeros(9, HKV, page, D, dtype=pool, device=DEV) for _ in range(2))
    table = torch.randperm(9, device=DEV).to(torch.int32).view(B, 3)
    pos = torch.tensor([0, 5, 27], dtype=torch.int32, device=DEV)
    counts = torch.tensor([21, 3, 20], dtype=torch.int32, device=DEV)
    shape = (B, HKV, N, D) if layout == "head_major" else (B, N, HKV, D)
    news = [[torch.randn(shape, device=DEV).to(x) for _ in range(2)] for _ in range(3)]
    if layout == "token_major":
        news = [[t.transpose(1, 2) for t in n] for n in news]
    ws, before, prep = {}, 0, None
    for i, (k, v) in enumerate(news):
        wk, wv = kp.clone(), vp.clone()
        for b in range(B):
            for n in range(int(counts[b])):
                t = int(pos[b]) + n
                for w, new in ((wk, k), (wv, v)):
                    w[int(table[b, t // page]), :, t % page] = new[b, :, n].float().to(pool)
        if i:
            before = torch.cuda.memory_stats()["allocation.all.allocated"]
        paged16_append(kp, vp, k, v, table, pos, counts, _workspace=ws)
        if i:
            assert torch.cuda.memory_stats()["allocation.all.allocated"] == before and ws["call"] is prep
        prep = ws["call"]
        _same(kp, wk)
        _same(vp, wv)


def test_types_side_by_side_on_one_workspace():
    from tritonkv_amd.paged16 import paged16_append

    kp, vp = (torch.zeros(2, 1, 16, 64, dtype=F16, device=DEV) for _ in range(2))
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
    ws = {}
    for i, t in enumerate((F16, BF16, torch.float32, BF16, F16)):
        new = torch.randn(1, 1, 1, 64, device=DEV).to(t)
        paged16_append(kp, vp, new, -new, table, torch.tensor([3 * i], dtype=torch.int32, device=DEV), _workspace=ws)
        at = kp[1 if 3 * i < 16 else 0, 0, 3 * i % 16], vp[1 if 3 * i < 16 else 0, 0, 3 * i % 16]
        _same(at[0], new[0, 0, 0].float().to(F16))
        _same(at[1], -new[0, 0, 0].float().to(F16))
