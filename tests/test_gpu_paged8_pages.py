"""Pages of 8-bit pools copied and compacted: codes and scales alike."""

from __future__ import annotations

import pytest
import torch

import paged8_ref as ref
from paged8_ref import E4M3, INT8

pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(a.codes.view(torch.int8), b.codes.view(torch.int8)) and torch.equal(a.scale, b.scale)


def pools(code, HKV, page, block, seed):
    return [ref.make_pool(12, HKV, page, 64, code, block, seed + i) for i in (1, 2)]


@pytest.mark.parametrize("code,HKV,page,block", [(E4M3, 2, 64, 32), (INT8, 3, 96, 32), (E4M3, 1, 128, 128), (INT8, 5, 64, 64)])
def test_copies(code, HKV, page, block):
    """Within the pools and into others; scales of 4, 9, 1 and 5 a page, with room after them."""
    from tritonkv_amd.pages import copy_pages

    src, dst = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([3, 0, -1, 7, 99], [5, 11, 2, 6, 1]))
    a, b = pools(code, HKV, page, block, 0), pools(code, HKV, page, block, 20)
    want_in, want_out = pools(code, HKV, page, block, 0), pools(code, HKV, page, block, 20)
    for x, y, z in zip(want_in, want_out, pools(code, HKV, page, block, 0)):
        for s, d in ((3, 5), (0, 11), (7, 6)):
            for w in (x, y):
                w.codes.view(torch.int8)[d] = z.codes.view(torch.int8)[s]
                w.scale[d] = z.scale[s]
    ws: dict = {}
    copy_pages(a, src, dst, b, _workspace=ws)
    assert all(same(x, y) for x, y in zip(b, want_out))
    for _ in range(2):
        copy_pages(a, src, dst, _workspace=ws)
        assert all(same(x, y) for x, y in zip(a, want_in))


@pytest.mark.parametrize("code,HKV,page,block", [(E4M3, 2, 64, 32), (INT8, 3, 96, 32)])
def test_compaction_keeps_what_rows_hold(code, HKV, page, block):
    from tritonkv_amd.pages import compact_pages
    from tritonkv_amd.paged8 import paged8_read

    a = pools(code, HKV, page, block, 0)
    table = torch.tensor([[9, 4, -1], [2, -1, -1], [9, 11, 7]], dtype=torch.int32, device="cuda")
    refs = torch.zeros(12, dtype=torch.int32, device="cuda")
    for p in (9, 4, 2, 9, 11, 7):
        refs[p] += 1
    counts = torch.tensor([2 * page, page, 3 * page], dtype=torch.int32, device="cuda")
    held = sorted(refs.tolist())
    before = paged8_read(*a, table, None, counts, tokens=3 * page, dtype=torch.float32)
    new_table, new_refs, live = compact_pages(a, table, refs)
    assert int(live) == 5 and int((new_table >= 0).sum()) == 6 and int(new_table.max()) == 4
    after = paged8_read(*a, new_table, None, counts, tokens=3 * page, dtype=torch.float32)
    assert all(torch.equal(x, y) for x, y in zip(before, after))
    assert sorted(new_refs.tolist()) == held
