"""Kept calls of the 8-bit pages and of apply_rotary refuse what their first call refuses: tensors over each other."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tritonkv_amd import _lib
from tritonkv_amd import paged8 as p8
from tritonkv_amd import rotary as ro

I32 = torch.int32
_ENTRY = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p)(lambda args, stream: 0)


@pytest.fixture
def kept(monkeypatch):
    """keep(call): the tensors' check of the call that ``call`` leaves in its workspace, with an entry that does
    nothing: whether it would launch them."""
    found = {}

    def keep16(ws, key, args, entry, what, device, buffers, slots):
        found["call"] = _lib.host().prepare(bytes(args), ctypes.cast(_ENTRY, ctypes.c_void_p).value, 0, slots, None)
        found["slots"] = slots

    for module in (p8, ro):
        monkeypatch.setattr(module, "_require_gpu", lambda *a: None)
        monkeypatch.setattr(module, "_keep16", keep16)
    monkeypatch.setattr(_lib, "launch", lambda *a: 0)

    def keep(call):
        call()
        names = [t for t, *_ in found["slots"]]

        def taken(**change):
            """change: slot number (as s0, s1, ...) to another tensor."""
            tensors = [change.get(f"s{i}", t) for i, t in enumerate(names)]
            try:
                return _lib.host().run(found["call"], *tensors) is not None
            except RuntimeError:  # past the tensors: the device is asked for, and there is none
                return True

        assert taken()
        return taken

    return keep


def pool(P=4, HKV=2, page=64, D=64, dtype=torch.int8, block=32):
    return p8.empty_paged8_pool(P, HKV, page, D, dtype, block, device="cpu")


def room(*shape):
    """A tensor at the start of a storage that holds any of these tests' tensors."""
    n = torch.Size(shape).numel()
    return torch.zeros(2 ** 16)[:n].view(shape)


def over(t, like):
    """A tensor of like's form over t's memory."""
    raw = t.untyped_storage()
    assert 4 * sum((n - 1) * m for n, m in zip(like.shape, like.stride())) < raw.nbytes()
    return torch.empty(0, dtype=like.dtype).set_(raw, 0, like.shape, like.stride())


def test_read(kept):
    k, v = pool(), pool()
    out = tuple(room(1, 2, 8, 64) for _ in range(2))
    table, n = torch.zeros(1, 64, dtype=I32), torch.zeros(1, dtype=I32)
    taken = kept(lambda: p8.paged8_read(k, v, table, n, n.clone(), out=out, _workspace={}))
    # slots: k codes, scale, v codes, scale, table, positions, counts, out, out
    assert taken(s7=out[0].clone(), s8=out[1].clone()) and taken(s0=v.codes, s2=k.codes) and taken(s6=n)
    assert not taken(s7=out[1]) and not taken(s8=out[0])
    for t in (k.codes, v.codes):
        assert not taken(s7=over(t, out[0])) and not taken(s8=over(t, out[1]))
    for i, t in ((1, k.scale), (3, v.scale), (4, table), (5, n), (6, n)):
        assert not taken(**{f"s{i}": over(out[0], t)}) and not taken(**{f"s{i}": over(out[1], t)})


def append(**kw):
    a = dict(k_pool=pool(), v_pool=pool(), k_new=torch.zeros(2, 2, 3, 64), v_new=torch.zeros(2, 2, 3, 64),
             block_table=torch.zeros(2, 2, dtype=I32), positions=torch.zeros(2, dtype=I32),
             counts=torch.zeros(2, dtype=I32), rotary=ro.Rotary(64, device="cpu"), q=torch.zeros(2, 4, 3, 64))
    a.update(kw)
    return a


# slots of an append: k codes, scale, v codes, scale, k_new, v_new, table, positions, counts, turns, q, q_out


def test_append_into_another_tensor(kept):
    q_out = room(2, 4, 3, 64)
    a = append(q_out=q_out)
    taken = kept(lambda: p8.paged8_append(**a, _workspace={}))
    assert taken(s11=q_out.clone()) and taken(s4=a["v_new"])
    for i, t in ((0, a["k_pool"].codes), (1, a["k_pool"].scale), (2, a["v_pool"].codes), (3, a["v_pool"].scale),
                 (4, a["k_new"]), (5, a["v_new"]), (6, a["block_table"]), (7, a["positions"]), (8, a["counts"]),
                 (9, a["rotary"].turns), (10, a["q"])):
        assert not taken(**{f"s{i}": over(q_out, t)}), i


def test_append_in_place(kept):
    q = room(2, 4, 3, 64)
    a = append(q=q, q_out=q)
    taken = kept(lambda: p8.paged8_append(**a, _workspace={}))
    other = torch.zeros_like(q)
    assert taken(s10=other, s11=other) and taken(s4=a["v_new"])
    for i, t in ((0, a["k_pool"].codes), (1, a["k_pool"].scale), (2, a["v_pool"].codes), (3, a["v_pool"].scale),
                 (4, a["k_new"]), (5, a["v_new"]), (6, a["block_table"]), (7, a["positions"]), (8, a["counts"]),
                 (9, a["rotary"].turns)):
        assert not taken(**{f"s{i}": over(q, t)}), i


# slots of apply_rotary: q, k, q_out, k_out, positions, turns


def test_rotary_into_other_tensors(kept):
    q, k, pos, rot = room(2, 4, 3, 64), room(2, 4, 3, 64), torch.zeros(2, dtype=I32), ro.Rotary(64, device="cpu")
    out = room(2, 4, 3, 64), room(2, 4, 3, 64)
    taken = kept(lambda: ro.apply_rotary(q, k, pos, rot, out=out, _workspace={}))
    assert taken(s0=k) and taken(s2=out[1], s3=out[0])
    assert not taken(s2=q) and not taken(s2=k) and not taken(s3=q) and not taken(s2=out[1])
    assert not taken(s4=over(out[0], pos)) and not taken(s5=over(out[1], rot.turns))


def test_rotary_in_place(kept):
    q, k, pos, rot = room(2, 4, 3, 64), room(2, 4, 3, 64), torch.zeros(2, dtype=I32), ro.Rotary(64, device="cpu")
    taken = kept(lambda: ro.apply_rotary(q, k, pos, rot, out=(q, k), _workspace={}))
    other = torch.zeros_like(q)
    assert taken(s0=other, s2=other)
    assert not taken(s0=k, s2=k) and not taken(s1=q, s3=q)
    assert not taken(s4=over(q, pos)) and not taken(s4=over(k, pos)) and not taken(s5=over(k, rot.turns))


def fused(B=2, N=3, HQ=4, HKV=2, D=64):
    """Queries, keys and values that lie in turn in one projection's output."""
    x = torch.zeros(B, N, HQ + 2 * HKV, D)
    return tuple(x[:, :, a:b].transpose(1, 2) for a, b in ((0, HQ), (HQ, HQ + HKV), (HQ + HKV, HQ + 2 * HKV)))


def test_tensors_in_turn_stay_kept(kept):
    """They interleave, and share nothing: as in the first call."""
    (q, k, v), pos, rot = fused(), torch.zeros(2, dtype=I32), ro.Rotary(64, device="cpu")
    taken = kept(lambda: ro.apply_rotary(q, k, pos, rot, out=(q, k), _workspace={}))
    q2, k2, _ = fused()
    assert taken(s0=q2, s1=k2, s2=q2, s3=k2)
    over_q = torch.as_strided(q, k.shape, k.stride(), q.storage_offset() + 64)
    assert not taken(s1=over_q, s3=over_q)
    taken = kept(lambda: p8.paged8_append(**append(q=q, q_out=q, k_new=k, v_new=v), _workspace={}))
    assert taken() and not taken(s4=over_q) and not taken(s5=over_q)
