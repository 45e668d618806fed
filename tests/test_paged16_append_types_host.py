"""The append's type of new rows in the C interface, without a GPU."""

from __future__ import annotations

import ctypes

import pytest


@pytest.mark.parametrize("kind", [-1, 3])
def test_unknown_types_are_refused(kind):
    from tritonkv_amd import _lib

    d = 0x1000
    a = _lib.Paged16AppendArgs(k_new=d, v_new=d, k_new_strides=(64, 64, 64), v_new_strides=(64, 64, 64), k=d, v=d,
                               k_strides=(1024, 1024, 64), v_strides=(1024, 1024, 64), block_table=d, positions=d,
                               new_is_fp32=kind, B=1, HKV=1, N=1, D=64, block_table_stride=1, max_pages=1,
                               page_size=16, num_pages=1)
    assert _lib.load().tkv_paged16_append(ctypes.byref(a), None) == _lib.TKV_EINVAL
    a.new_is_fp32, a.k_new_strides = 2, (64, 64, 4)  # rows of 16 bits on 16 bytes
    assert _lib.load().tkv_paged16_append(ctypes.byref(a), None) == _lib.TKV_EINVAL
