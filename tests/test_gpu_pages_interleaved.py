"""Pages copied between the halves of paired pools, and a compaction into other columns of
its table's buffer, on the GPU: equal bytes and entries."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("pairs", [3, 700])
def test_copies_between_the_halves_of_paired_pages(pairs):
    from tritonkv_amd.pages import copy_pages

    both = torch.randn(1500, 2, 2, 16, 1024 if pairs > 100 else 64, device=DEV).half()
    want = both.clone()
    g = torch.Generator().manual_seed(pairs)
    src = torch.randperm(1500, generator=g)[:pairs].to(DEV)
    dst = torch.randperm(1500, generator=g)[:pairs].to(DEV)
    want[dst, 1] = want[src, 0]
    ws = {}
    for _ in range(2):
        copy_pages([both[:, 0]], src.int(), dst.int(), [both[:, 1]], _workspace=ws)
        assert torch.equal(both, want)


def test_a_compaction_into_other_columns():
    from tritonkv_amd.pages import compact_pages

    pool = torch.randn(10, 2, 16, 64, device=DEV).half()
    before = pool.clone()
    tables = torch.full((2, 8), -1, dtype=torch.int32, device=DEV)
    tables[0, 0], tables[1, 0], tables[1, 1] = 9, 1, 6
    refs = torch.zeros(10, dtype=torch.int32, device=DEV)
    refs[[1, 6, 9]] = 1
    ws = {}
    for _ in range(2):
        table, out_refs, live = compact_pages([pool], tables[:, :3], refs, out=(tables[:, 4:7], torch.empty_like(refs)),
                                              _workspace=ws)
        assert live.tolist() == [3] and out_refs.tolist() == [1] * 3 + [0] * 7
        assert tables.tolist() == [[9, -1, -1, -1, 2, -1, -1, -1], [1, 6, -1, -1, 1, 0, -1, -1]]
        assert torch.equal(pool[0], before[6]) and torch.equal(pool[2], before[9])
