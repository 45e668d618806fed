"""The fused append of the 16-bit paged decode on rows that fill their tables or whose lengths
are past them: what the append and the decode after it do, bit for bit."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged16 import BF16, DEV, F16, _case, _check, _decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("HQ", [4, 80])
@pytest.mark.parametrize("piece", [None, 32, 96], ids=["auto", "32", "whole"])
def test_rows_at_and_past_the_end_of_their_tables(dtype, HQ, piece):
    from tritonkv_amd.paged16 import paged16_append

    S = 96
    q, kp, vp, table, lens = _case([S, S, S, S - 1, S, 1, 0], HQ, 2, 128, 32, 3, dtype, seed=HQ)
    lens.copy_(torch.tensor([S, S + 1, 2 ** 31 - 1, S - 1, S + 32, 1, 0], device=DEV))
    new = torch.randn(2, 7, 2, 128, device=DEV).to(dtype)
    before = kp.clone(), vp.clone()
    ka, va = kp.clone(), vp.clone()
    paged16_append(ka, va, new[0][:, :, None], new[1][:, :, None], table, lens - 1)
    want = _decode(q, ka, va, table, lens, piece_tokens=piece)
    got = _decode(q, kp, vp, table, lens, k_new=new[0], v_new=new[1], piece_tokens=piece)
    bits = torch.int16
    for b in (1, 2, 4):  # past their tables: as they were
        for pool, old in zip((kp, vp), before):
            assert torch.equal(pool[table[b].long()].view(bits), old[table[b].long()].view(bits))
    assert torch.equal(kp.view(bits), ka.view(bits)) and torch.equal(vp.view(bits), va.view(bits))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _check(*got, q, kp, vp, table, lens)
    got = _decode(q, kp, vp, table, None, k_new=new[0], v_new=new[1], piece_tokens=piece)  # all rows full
    for pool, x in zip((kp, vp), new):
        assert torch.equal(pool[table[[0, 1, 2, 4], 2].long(), :, 31], x[[0, 1, 2, 4]])
