"""What the 8-bit page calls and apply_rotary refuse: outputs over the tensors that say where tokens lie, and more."""

from __future__ import annotations

import pytest
import torch

from tritonkv_amd import paged8 as p8
from tritonkv_amd import rotary as ro

I32 = torch.int32


def pool():
    return p8.empty_paged8_pool(4, 2, 64, 64, torch.int8, 32, device="cpu")


def over(t, like):
    """A tensor of like's form over t's memory."""
    return torch.empty(0, dtype=like.dtype).set_(t.untyped_storage(), 0, like.shape, like.stride())


def test_read_refuses_outputs_over_its_other_tensors():
    k, v, table, n = pool(), pool(), torch.zeros(1, 64, dtype=I32), torch.zeros(1, dtype=I32)
    out = tuple(torch.zeros(1, 2, 8, 64) for _ in range(2))
    for kw in (dict(block_table=over(out[0], table)), dict(positions=over(out[1], n)), dict(counts=over(out[0], n))):
        with pytest.raises(ValueError, match="share"):
            p8.paged8_read(k, v, **{**dict(block_table=table), **kw}, out=out)


def append(q_out):
    return dict(k_pool=pool(), v_pool=pool(), k_new=torch.zeros(2, 2, 3, 64), v_new=torch.zeros(2, 2, 3, 64),
                block_table=torch.zeros(2, 2, dtype=I32), positions=torch.zeros(2, dtype=I32),
                counts=torch.zeros(2, dtype=I32), rotary=ro.Rotary(64, device="cpu"), q=torch.zeros(2, 4, 3, 64),
                q_out=q_out)


def test_append_refuses_queries_over_its_other_tensors():
    q_out = torch.zeros(2, 4, 3, 64)
    for name in ("block_table", "positions", "counts"):
        a = append(q_out)
        a[name] = over(q_out, a[name])
        with pytest.raises(ValueError, match="share"):
            p8.paged8_append(**a)
    a = append(q_out)
    a["rotary"].turns = over(q_out, a["rotary"].turns)
    with pytest.raises(ValueError, match="share"):
        p8.paged8_append(**a)


def test_rotary_refuses_outputs_over_its_turns():
    q, pos, rot = torch.zeros(2, 4, 3, 64), torch.zeros(2, dtype=I32), ro.Rotary(64, device="cpu")
    out = torch.zeros_like(q)
    rot.turns = over(out, rot.turns)
    with pytest.raises(ValueError, match="share"):
        ro.apply_rotary(q, None, pos, rot, out=(out, None))


def test_a_kept_read_still_checks_its_tokens(monkeypatch):
    """``tokens`` must be the outputs', in the call that is kept and in those after it."""
    from tritonkv_amd import _lib

    class Kept:
        def __init__(self, key):
            self.key = key

        def run(self, *tensors):
            return True

    monkeypatch.setattr(p8, "_require_gpu", lambda *a: None)
    monkeypatch.setattr(p8, "_keep16", lambda ws, key, *a: ws.update(call=Kept(key)))
    monkeypatch.setattr(_lib, "launch", lambda *a: 0)
    table, out = torch.zeros(1, 2, dtype=I32), tuple(torch.zeros(1, 2, 8, 64) for _ in range(2))
    for first in (None, 8):
        ws: dict = {}
        p8.paged8_read(pool(), pool(), table, tokens=first, out=out, _workspace=ws)
        assert "call" in ws
        with pytest.raises(ValueError, match="tokens"):
            p8.paged8_read(pool(), pool(), table, tokens=9, out=out, _workspace=ws)
        assert p8.paged8_read(pool(), pool(), table, tokens=8, out=out, _workspace=ws)[0] is out[0]


def test_decode_refuses_queries_that_require_grad():
    """It records no gradient, and says so, also where a call is kept."""
    q = torch.zeros(1, 4, 64).half().requires_grad_()
    args = q, pool(), pool(), torch.zeros(1, 2, dtype=I32)
    for kw in (dict(), dict(_workspace={})):
        with pytest.raises(ValueError, match="requires grad"):
            p8.paged8_decode_attention(*args, **kw)
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU|HIP"):
            p8.paged8_decode_attention(*args, **kw)
        with pytest.raises(RuntimeError, match="GPU|HIP"):
            p8.paged8_decode_attention(q.detach(), *args[1:], **kw)
