"""Rows with room made ahead, without a GPU: the rule that ``fork_rows`` follows with
``written`` keeps every row's tokens its own, and the argument's checks."""

from __future__ import annotations

import ctypes
import os
import random
import subprocess

import pytest
import torch

from tests.rows_with_room import Rows, step

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def Z(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("seed", range(40))
def test_rows_keep_their_tokens(seed):
    rng = random.Random(seed)
    m = Rows(rng.choice([1, 2, 5, 9]), rng.choice([1, 3, 8]), 60, rng.choice([2, 5, 16]))
    for _ in range(40):
        m.fork(*step(rng, m))
        for b in rng.sample(range(m.B), rng.randint(0, m.B)):
            for _ in range(rng.randint(0, m.page + 1)):
                m.append(b)
        assert all(m.row(b) == m.tokens[b] for b in range(m.B))
        used = [p for row, n in zip(m.table, m.lens) for p in row[:-(-n // m.page)]]
        assert m.refs == [used.count(p) for p in range(m.N)]


def test_room_that_counts_as_written_is_shared():
    """20 tokens with room for 40, forked as 40 tokens: both rows write into one page."""
    for use, same in ((False, True), (True, False)):
        m = Rows(2, 4, 12, 16)
        m.fork(None, [40, 0])
        for _ in range(20):
            m.append(0)
        assert m.fork([0, 0], None, use)[0] == 0
        assert (m.table[0][1] == m.table[1][1]) is same
        m.append(0), m.append(1)
        assert (m.row(0) != m.tokens[0]) is same and m.row(1) == m.tokens[1]


POOL = torch.zeros(6, 2, 16, 64, dtype=torch.float16)
T, R, L = Z(2, 3), Z(6), Z(2)


@pytest.mark.parametrize("written,error,match", [
    (Z(3), ValueError, "written"),
    (Z(2, dtype=torch.int64), ValueError, "written"),
    (Z(2, 1), ValueError, "written"),
    ([1, 2], ValueError, "written"),
    (L, ValueError, "share memory"),
    (R[2:4], ValueError, "share memory"),
    (T[1, 1:], ValueError, "share memory"),
    (Z(4)[::2], RuntimeError, "GPU"),
    (Z(2), RuntimeError, "GPU"),
])
def test_refusals(written, error, match):
    from tritonkv_amd.pages import fork_rows, resize_rows

    with pytest.raises(error, match=match):
        fork_rows([POOL], T, L, R, Z(2), written=written)
    with pytest.raises(error, match=match):
        resize_rows([POOL], T, L, R, Z(2), written=written, _workspace={})


def test_argument_block_matches_the_header(tmp_path):
    from tritonkv_amd import _lib

    c = tmp_path / "l.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tkv.h"\nint main(void) { printf("%zu %zu %zu", '
                 "sizeof(tkv_fork_written_args), offsetof(tkv_fork_written_args, rows.page_size), "
                 "offsetof(tkv_fork_written_args, written)); return 0; }")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(tmp_path / "l")], check=True)
    got = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()
    a = _lib.ForkWrittenArgs
    assert [int(x) for x in got] == [ctypes.sizeof(a), a.page_size.offset, a.written.offset]


def test_c_entry_refuses():
    from tritonkv_amd import _lib

    d = 0x1000
    fn = _lib.load().tkv_fork_rows_written
    a = _lib.ForkWrittenArgs(block_table=d, seq_lens=d, refs=d, status=d, work=0x1004, table_stride=3, B=2,
                             max_pages=3, page_size=16, num_pages=6, written=d)
    assert fn(ctypes.byref(a), None) == _lib.TKV_EINVAL and fn(None, None) == _lib.TKV_EINVAL
    a.work, a.B = d, 8193
    assert fn(ctypes.byref(a), None) == _lib.TKV_EUNSUPPORTED
