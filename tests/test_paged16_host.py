"""Host side of the 16-bit page pools without a GPU: argument checks before any
backend call, the pieces' plan, and the C entries' own refusals."""

from __future__ import annotations

import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, BF16 = torch.float16, torch.bfloat16


def test_pool_rules():
    from tritonkv_amd.paged16 import empty_paged16_pool

    assert empty_paged16_pool(3, 2, 48, 64, BF16, device="cpu").shape == (3, 2, 48, 64)
    for bad in ((3, 2, 40, 64), (3, 2, 0, 64), (0, 2, 32, 64), (3, 0, 32, 64), (3, 2, 32, 96)):
        with pytest.raises(ValueError):
            empty_paged16_pool(*bad, device="cpu")
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        empty_paged16_pool(3, 2, 32, 64, torch.float32, device="cpu")


def _call(**kw):
    a = dict(q=torch.zeros(2, 8, 128, dtype=F16), k_pool=torch.zeros(4, 2, 32, 128, dtype=F16),
             v_pool=torch.zeros(4, 2, 32, 128, dtype=F16), block_table=torch.zeros(2, 3, dtype=torch.int32))
    a.update(kw)
    from tritonkv_amd.paged16 import paged16_decode_attention

    return paged16_decode_attention(**a)


Z = torch.zeros


@pytest.mark.parametrize("kw,error,match", [
    (dict(k_pool=Z(4, 2, 32, 128)), TypeError, "k_pool must be float16 or bfloat16"),
    (dict(v_pool=Z(4, 2, 32, 128, dtype=BF16)), ValueError, "same shape, dtype"),
    (dict(v_pool=Z(5, 2, 32, 128, dtype=F16)), ValueError, "same shape"),
    (dict(k_pool=Z(2, 32, 128, dtype=F16)), ValueError, "num_pages, HKV, page_size, D"),
    (dict(k_pool=Z(4, 2, 24, 128, dtype=F16), v_pool=Z(4, 2, 24, 128, dtype=F16)), ValueError, "multiple of 16"),
    (dict(k_pool=Z(4, 2, 32, 96, dtype=F16), v_pool=Z(4, 2, 32, 96, dtype=F16)), ValueError, "head_dim"),
    (dict(k_pool=Z(0, 2, 32, 128, dtype=F16), v_pool=Z(0, 2, 32, 128, dtype=F16)), ValueError, "empty"),
    (dict(k_pool=Z(4, 2, 32, 132, dtype=F16)[..., 4:]), ValueError, "16-byte"),
    (dict(k_pool=Z(4, 2, 128, 32, dtype=F16).transpose(2, 3)), ValueError, "densely"),
    (dict(k_pool=Z(1, 2, 32, 128, dtype=F16).expand(4, 2, 32, 128)), ValueError, "densely"),
    (dict(q=Z(2, 8, 128, dtype=BF16)), TypeError, "pools' dtype"),
    (dict(q=Z(2, 8, 128)), TypeError, "pools' dtype"),
    (dict(q=Z(2, 8, 64, dtype=F16)), ValueError, "q must be"),
    (dict(q=Z(2, 7, 128, dtype=F16)), ValueError, "multiple of HKV"),
    (dict(q=Z(0, 8, 128, dtype=F16)), ValueError, "neither zero"),
    (dict(q=Z(2, 0, 128, dtype=F16)), ValueError, "neither zero"),
    (dict(block_table=Z(2, 3, dtype=torch.int64)), ValueError, "block_table"),
    (dict(block_table=Z(3, 3, dtype=torch.int32)), ValueError, "block_table"),
    (dict(block_table=Z(2, 0, dtype=torch.int32)), ValueError, "column"),
    (dict(seq_lens=Z(2, dtype=torch.int64)), ValueError, "seq_lens"),
    (dict(seq_lens=Z(3, dtype=torch.int32)), ValueError, "seq_lens"),
    (dict(seq_lens=Z(2, 1, dtype=torch.int32)), ValueError, "seq_lens"),
    (dict(out=Z(2, 8, 128, dtype=F16)), ValueError, "out must be"),
    (dict(out=Z(2 * 8 * 128 + 1)[1:].view(2, 8, 128)), ValueError, "16-byte"),
    (dict(lse=Z(2, 7)), ValueError, "lse"),
    (dict(lse=Z(2, 8, dtype=F16)), ValueError, "lse"),
    (dict(lse=[0.0]), ValueError, "lse"),
    (dict(k_new=Z(2, 2, 128, dtype=F16)), ValueError, "together"),
    (dict(k_new=Z(2, 2, 128, dtype=F16), v_new=Z(2, 2, 64, dtype=F16)), ValueError, "v_new must have shape"),
    (dict(k_new=Z(2, 2, 128), v_new=Z(2, 2, 128)), TypeError, "pools' dtype"),
    (dict(piece_tokens=0), ValueError, "piece_tokens"),
    (dict(piece_tokens=1 << 60), RuntimeError, "HIP"),
])
def test_decode_refuses_before_the_backend(kw, error, match):
    with pytest.raises(error, match=match):
        _call(**kw)


def test_decode_without_a_gpu():
    with pytest.raises(RuntimeError, match="HIP"):
        _call()
    with pytest.raises(RuntimeError, match="HIP"):
        _call(k_new=Z(2, 2, 1, 128, dtype=F16), v_new=Z(2, 2, 1, 128, dtype=F16), lse=Z(2, 8), _workspace={})


@pytest.mark.parametrize("kw,error,match", [
    (dict(k_new=Z(2, 3, 5, 128, dtype=F16)), ValueError, "k_new must be"),
    (dict(v_new=Z(2, 2, 6, 128, dtype=F16)), ValueError, "same shape and dtype"),
    (dict(v_new=Z(2, 2, 5, 128)), ValueError, "same shape and dtype"),
    (dict(k_new=Z(2, 2, 5, 128, dtype=torch.int16)), TypeError, "float16, bfloat16 or float32"),
    (dict(block_table=Z(1, 3, dtype=torch.int32)), ValueError, "block_table"),
    (dict(positions=Z(2, dtype=torch.int64)), ValueError, "positions"),
    (dict(positions=None), ValueError, "positions"),
    (dict(counts=Z(3, dtype=torch.int32)), ValueError, "counts"),
    (dict(k_pool=Z(4, 2, 24, 128, dtype=F16), v_pool=Z(4, 2, 24, 128, dtype=F16)), ValueError, "multiple of 16"),
    (dict(), RuntimeError, "GPU"),
])
def test_append_refuses(kw, error, match):
    from tritonkv_amd.paged16 import paged16_append

    a = dict(k_pool=Z(4, 2, 32, 128, dtype=F16), v_pool=Z(4, 2, 32, 128, dtype=F16),
             k_new=Z(2, 2, 5, 128, dtype=F16), v_new=Z(2, 2, 5, 128, dtype=F16),
             block_table=Z(2, 3, dtype=torch.int32), positions=Z(2, dtype=torch.int32))
    a.update(kw)
    with pytest.raises(error, match=match):
        paged16_append(**a)


@pytest.mark.parametrize("B", [1, 7, 256, 60000])
@pytest.mark.parametrize("HKV,G", [(1, 1), (8, 4), (2, 40)])
@pytest.mark.parametrize("S", [16, 512, 4096, 1 << 20])
def test_the_shares_cover_every_chunk_once(B, HKV, G, S):
    """Whatever the lengths: shares follow each other, none is empty, and the share that a
    chunk is looked up in holds it (the device's arithmetic, restated)."""
    import random

    from tritonkv_amd.paged16 import MAX_WORKGROUPS, plan_shares

    rng = random.Random(B * S)
    for piece in (None, 48, S):
        try:
            least, groups, few, long = plan_shares(B, HKV, G, S, 128, "cpu", piece)
        except ValueError:
            assert piece is not None and -(-B * -(-S // 32) // -(-piece // 32)) > MAX_WORKGROUPS
            continue
        assert 0 <= groups <= MAX_WORKGROUPS and least > 0
        if groups == 0:
            assert S <= 1024 if piece is None else S <= 32 * least
            continue
        assert 0 <= few <= groups and (few == 0 or long > 0)
        for lens in ([S] * B, [0] * B, [S] + [0] * (B - 1), [rng.randint(0, S) for _ in range(B)]):
            total = sum(max(1, -(-n // 32)) for n in lens)
            W = few if B <= few and total >= few * long else min(groups, -(-total // least))
            each, more = divmod(total, W)
            assert each > 0

            def start(i):
                return i * each + min(i, more)

            def of(chunk):
                big = more * (each + 1)
                return chunk // (each + 1) if chunk < big else more + (chunk - big) // each

            assert start(0) == 0 and start(W) == total
            for i in rng.sample(range(W), min(W, 50)):
                assert of(start(i)) == of(start(i + 1) - 1) == i


def test_argument_blocks_match_the_header():
    from tritonkv_amd import _lib

    for struct, name in ((_lib.Paged16Args, "tkv_paged16_args"), (_lib.Paged16AppendArgs, "tkv_paged16_append_args")):
        fields = [f for f, _ in struct._fields_]
        src = '#include <stdio.h>\n#include <stddef.h>\n#include "tkv.h"\nint main(void) { printf("%zu", sizeof(' \
            + name + "));\n" + "".join(f'printf(" %zu", offsetof({name}, {f}));\n' for f in fields) + "return 0; }"
        with tempfile.TemporaryDirectory() as d:
            c = os.path.join(d, "l.c")
            open(c, "w").write(src)
            subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", c[:-2]], check=True)
            vals = [int(x) for x in subprocess.run([c[:-2]], capture_output=True, text=True, check=True).stdout.split()]
        assert vals == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


def _decode_args():
    from tritonkv_amd import _lib

    d = 0x1000
    return _lib.Paged16Args(q=d, q_strides=(1024, 128), k=d, v=d, k_strides=(8192, 4096, 128),
                            v_strides=(8192, 4096, 128), block_table=d, out=d, partials=d, row_pieces=d, B=2,
                            HQ=8, HKV=2, D=128, block_table_stride=4, max_pages=4, page_size=32, num_pages=4,
                            sm_scale=0.1, least_chunks=2, workgroups=4)


@pytest.mark.parametrize("field,value", [
    ("q", None), ("q", 0x1008), ("k", None), ("v", 0x1008), ("out", 0x1004), ("block_table", None),
    ("partials", None), ("partials", 0x1008), ("row_pieces", 0x1004), ("k_new", 0x1000), ("B", 0), ("HQ", 7),
    ("HKV", 0), ("page_size", 24), ("page_size", 0), ("max_pages", 0), ("num_pages", 0),
    ("block_table_stride", 3), ("max_pages", 1 << 27), ("least_chunks", 0), ("workgroups", -1),
    ("workgroups", 65536), ("long_workgroups", 5), ("long_workgroups", -1), ("long_chunks", -1),
    ("long_workgroups", 2),  ("k_strides", (8192, 4096, 132)),
    ("v_strides", (8192, 4096, 0)), ("k_strides", (8192, 4096, 1 << 26)), ("k_strides", (-8, 4096, 128)),
    ("q_strides", (1024, 4))])
def test_c_entry_refuses(field, value):
    from tritonkv_amd import _lib

    a = _decode_args()
    setattr(a, field, value)
    assert _lib.load().tkv_paged16_decode_attention(ctypes.byref(a), None) == _lib.TKV_EINVAL


def test_c_entry_refuses_other_head_dims_and_null():
    from tritonkv_amd import _lib

    a = _decode_args()
    a.D = 96
    assert _lib.load().tkv_paged16_decode_attention(ctypes.byref(a), None) == _lib.TKV_EUNSUPPORTED
    assert _lib.load().tkv_paged16_decode_attention(None, None) == _lib.TKV_EINVAL
    assert _lib.load().tkv_paged16_append(None, None) == _lib.TKV_EINVAL


@pytest.mark.parametrize("field,value", [
    ("k_new", None), ("k_new", 0x1008), ("v", None), ("positions", None), ("block_table", None), ("B", 0),
    ("N", 0), ("D", 12), ("page_size", 0), ("num_pages", 0), ("block_table_stride", 1),
    ("k_new_strides", (8, 8, 4)), ("v_strides", (8192, 4096, 4))])
def test_c_append_refuses(field, value):
    from tritonkv_amd import _lib

    d = 0x1000
    a = _lib.Paged16AppendArgs(k_new=d, v_new=d, k_new_strides=(8, 8, 8), v_new_strides=(8, 8, 8), k=d, v=d,
                               k_strides=(8192, 4096, 128), v_strides=(8192, 4096, 128), block_table=d,
                               positions=d, B=2, HKV=2, N=3, D=128, block_table_stride=4, max_pages=4,
                               page_size=32, num_pages=4)
    setattr(a, field, value)
    assert _lib.load().tkv_paged16_append(ctypes.byref(a), None) == _lib.TKV_EINVAL
