"""Pools and tables that lie in turn in one buffer share no memory, without a GPU."""

from __future__ import annotations

import pytest
import torch

F16 = torch.float16


def Z(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


def _shared(a, b):
    at = lambda t: set((torch.arange(t.untyped_storage().nbytes() // t.element_size()).as_strided(
        t.shape, t.stride(), t.storage_offset())).flatten().tolist())
    return bool(at(a) & at(b))


@pytest.mark.parametrize("width,a,b", [
    (8, (0, 4), (4, 8)), (8, (0, 4), (3, 8)), (8, (4, 8), (0, 4)), (8, (4, 8), (0, 5)), (8, (0, 8), (0, 8)),
    (8, (2, 3), (3, 4)), (8, (2, 3), (2, 3)), (8, (0, 1), (7, 8)), (8, (7, 8), (0, 8)), (9, (0, 5), (5, 9)),
])
@pytest.mark.parametrize("rows_a,rows_b", [((0, 5), (0, 5)), ((0, 3), (2, 5)), ((2, 5), (0, 3)), ((0, 2), (3, 5)),
                                           ((0, 1), (0, 5)), ((4, 5), (0, 5))])
def test_columns_of_one_table(width, a, b, rows_a, rows_b):
    from tritonkv_amd.pages import _overlap

    t = Z(5, width)
    x, y = t[rows_a[0]:rows_a[1], a[0]:a[1]], t[rows_b[0]:rows_b[1], b[0]:b[1]]
    assert _overlap(x, y) is _overlap(y, x) is _shared(x, y)


def test_other_strides_count_as_shared():
    from tritonkv_amd.pages import _overlap

    t = Z(64)
    assert _overlap(t[:32].view(4, 8)[:, :4], t[4:28].view(4, 6)[:, :1])
    assert _overlap(t[:32].view(4, 8)[:, :4], t[4:6]) and not _overlap(t[:32].view(4, 8), t[32:34])


def test_calls_take_them():
    from tritonkv_amd.pages import compact_pages, copy_pages, fork_rows

    both = torch.zeros(6, 2, 2, 16, 64, dtype=F16)
    with pytest.raises(RuntimeError, match="GPU"):
        copy_pages([both[:, 0]], Z(1), Z(1), [both[:, 1]])
    with pytest.raises(ValueError, match="share memory"):
        copy_pages([both[:, 0]], Z(1), Z(1), [both[1:, 0]])
    with pytest.raises(ValueError, match="share memory"):
        copy_pages([both[:, 0], both[:, 1]], Z(1), Z(1), [both[:, 1], torch.zeros(6, 2, 16, 64, dtype=F16)])
    tables, refs = Z(2, 8), Z(6)
    with pytest.raises(RuntimeError, match="GPU"):
        compact_pages([both[:, 0]], tables[:, :3], refs, out=(tables[:, 3:6], Z(6)))
    with pytest.raises(ValueError, match="share memory"):
        compact_pages([both[:, 0]], tables[:, :3], refs, out=(tables[:, 2:5], Z(6)))
    with pytest.raises(ValueError, match="share memory"):
        fork_rows([both[:, 0]], tables[:, :3], tables[0, 3:5], refs, Z(2))
