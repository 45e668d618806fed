"""Two forms of the 16-bit paged decode at the sizes that reach them: few long streams in place
of many short ones, and a fused append whose heads take several workgroups.  Tolerances
are those of ``test_gpu_paged16``, derived there."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_paged16 import BF16, DEV, EDGES, F16, _case, _check, _decode

pytestmark = pytest.mark.gpu


def _long_lengths(G, D, S, off):
    """A batch over 16 KV heads whose chunks of 32 tokens are ``off`` more than long streams need,
    in tables of S tokens, and the workgroups that a KV head should get."""
    from tritonkv_amd.paged16 import plan_shares

    least, workgroups, few, long = plan_shares(5, 16, G, S, D, DEV)
    need = few * long
    assert 5 <= few < workgroups
    lens = [0, 32 * (need + off - 26) - 7, 33, 1, 700]  # 1 (no tokens), 2, 1 and 22 chunks beside the long row
    assert max(lens) <= S and sum(max(1, -(-n // 32)) for n in lens) == need + off
    return lens, few if off >= 0 else min(workgroups, -(-(need + off) // least))


def _shares(ws, B):
    """Workgroups of a KV head that the rows were cut over, as the device noted them."""
    (rows,) = [t for key, t in ws.items() if key[0] == "row_pieces16"]
    return int(rows[:2 * B].view(B, 2).sum(1).max())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D,G,page", [(128, 1, 64), (128, 4, 16), (128, 20, 64), (256, 2, 48), (64, 1, 64)])
@pytest.mark.parametrize("off", [-1, 0, 1, 75])
def test_long_streams(dtype, D, G, page, off):
    S = (1 << 17) // page * page
    lens, workgroups = _long_lengths(G, D, S, off)
    if D == 64 and off not in (-1, 0):
        pytest.skip("65536 tokens: the two sides of the threshold suffice")
    q, kp, vp, table, lens = case = _case(lens, 16 * G, 16, D, page, S // page, dtype, seed=off + 2)
    ws = {}
    got, lse = _decode(*case, _workspace=ws)
    assert _shares(ws, 5) == workgroups
    _check(got, lse, *case)
    new = torch.randn(2, 5, 16, D, device=DEV).to(dtype)
    want_k, want_v = kp.clone(), vp.clone()
    from tritonkv_amd.paged16 import paged16_append

    paged16_append(want_k, want_v, new[0][:, :, None], new[1][:, :, None], table, lens - 1)
    want = _decode(q, want_k, want_v, table, lens)
    got = _decode(q, kp, vp, table, lens, k_new=new[0], v_new=new[1])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(kp.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(vp.view(torch.int16), want_v.view(torch.int16))
    _check(*got, q, kp, vp, table, lens)


def test_long_streams_of_equal_rows_and_a_captured_batch_that_grows_into_them():
    from tritonkv_amd.paged16 import paged16_decode_attention, plan_shares

    least, workgroups, few, long = plan_shares(4, 16, 2, 8192, 128, DEV)
    assert 4 <= few < workgroups and few * long <= 4 * 256  # 4 rows of 8192 tokens have 1024 chunks
    q, kp, vp, table, _ = _case([8192] * 4, 32, 16, 128, 64, 128, F16, seed=3, poison=False)
    out, lse = _decode(q, kp, vp, table, None)
    _check(out, lse, q, kp, vp, table, None)
    lens, ws = torch.tensor([100, 8192, 0, 33], dtype=torch.int32, device=DEV), {}
    paged16_decode_attention(q, kp, vp, table, lens, out=out, _workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged16_decode_attention(q, kp, vp, table, lens, out=out, _workspace=ws)
    assert few * long == 256  # chunks that long streams need
    for n, chunks in (([1, 960, 32, 1], 33), ([32 * 252, 0, 32, 5], 255), ([32 * 253, 0, 32, 5], 256),
                      ([8192, 33, 1, 0], 260), ([8192] * 4, 1024), ([5, 0, 0, 1], 4)):
        lens.copy_(torch.tensor(n, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        assert _shares(ws, 4) == (few if chunks >= 256 else min(workgroups, -(-chunks // least)))
        _check(out, None, q, kp, vp, table, lens)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [33, 64, 128])
@pytest.mark.parametrize("piece", [None, 32, 384], ids=["auto", "32", "whole"])
def test_the_fused_append_of_wide_groups(dtype, D, G, piece):
    """More than 32 heads on a KV head: every block of them puts the new token in its row's
    place, one of them stores it."""
    from tritonkv_amd.paged16 import paged16_append

    q, kp, vp, table, lens = _case(EDGES, 2 * G, 2, D, 48, 8, dtype, seed=G)
    new = torch.randn(2, len(EDGES), 2, D, device=DEV).to(dtype)
    for b, n in enumerate(EDGES):  # the token's place holds NaN until the call
        if n:
            for pool in (kp, vp):
                pool[int(table[b, (n - 1) // 48]), :, (n - 1) % 48] = float("nan")
    ka, va = kp.clone(), vp.clone()
    paged16_append(ka, va, new[0][:, :, None], new[1][:, :, None], table, lens - 1)
    want = _decode(q, ka, va, table, lens, piece_tokens=piece)
    got = _decode(q, kp, vp, table, lens, k_new=new[0], v_new=new[1], piece_tokens=piece)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(kp.view(torch.int16), ka.view(torch.int16))
    assert torch.equal(vp.view(torch.int16), va.view(torch.int16))
    _check(*got, q, kp, vp, table, lens)
