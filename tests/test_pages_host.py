"""Host side of the page bookkeeping without a GPU: argument checks before any
launch, the work sizes, and the C entries' own refusals."""

from __future__ import annotations

import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16 = torch.float16


def Z(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


def _pool(n=6, HKV=2, page=16, D=64, dtype=F16):
    return torch.zeros(n, HKV, page, D, dtype=dtype)


def _quant(n=6):
    from tritonkv_amd.paged import empty_paged_pool

    return empty_paged_pool(n, 2, 32, 64, 4, 32, device="cpu")


@pytest.mark.parametrize("kw,error,match", [
    (dict(pools=_pool()), TypeError, "list or tuple"),
    (dict(pools=[]), ValueError, "empty"),
    (dict(pools=[3]), TypeError, "page pool"),
    (dict(pools=[_pool(), _pool(5)]), ValueError, "of 6 pages"),
    (dict(pools=[_pool()[0]]), ValueError, "num_pages, HKV"),
    (dict(pools=[_pool(6, 2, 16, 128)[..., :64]]), ValueError, "dense"),
    (dict(pools=[_pool(1).expand(6, 2, 16, 64)]), ValueError, "overlap"),
    (dict(pools=[_pool(6, 1, 1, 4)]), ValueError, "16 bytes"),
    (dict(pools=[torch.zeros(6 * 2048 + 1, dtype=F16)[1:].view(6, 2, 16, 64)]), ValueError, "16 bytes"),
    (dict(src=Z(3, dtype=torch.int64)), ValueError, "src must be"),
    (dict(src=[0, 1, 2]), ValueError, "src must be"),
    (dict(dst=Z(2)), ValueError, "dst must be"),
    (dict(dst_pools=[]), ValueError, "as many tensors"),
    (dict(dst_pools=[_pool(4, 2, 32, 64)]), ValueError, "shapes"),
    (dict(dst_pools=[_pool(4, dtype=torch.bfloat16)]), ValueError, "dtypes"),
    (dict(dst_pools=[_pool(4, 16, 2, 64).transpose(1, 2)]), ValueError, "order"),
    (dict(), RuntimeError, "GPU"),
    (dict(dst_pools=[_pool(4)]), RuntimeError, "GPU"),
    (dict(pools=[_quant(), _pool(6, 2, 32)]), RuntimeError, "GPU"),
])
def test_copy_refuses(kw, error, match):
    from tritonkv_amd.pages import copy_pages

    a = dict(pools=[_pool()], src=Z(3), dst=Z(3))
    a.update(kw)
    with pytest.raises(error, match=match):
        copy_pages(**a)


def test_copy_between_pools_of_one_memory_is_refused():
    from tritonkv_amd.pages import copy_pages

    p = _pool(8)
    with pytest.raises(ValueError, match="share memory"):
        copy_pages([p[:5]], Z(1), Z(1), [p[4:]])
    with pytest.raises(ValueError, match="share memory"):
        copy_pages([p, p.clone()], Z(1), Z(1), [p.clone(), p])
    with pytest.raises(RuntimeError, match="GPU"):  # parts of one allocation that do not meet
        copy_pages([p[:4]], Z(1), Z(1), [p[4:]])
    with pytest.raises(RuntimeError, match="GPU"):  # one KV head: its stride says nothing
        copy_pages([_pool(6, 1)], Z(1), Z(1), [_pool(6, 16, 1).transpose(1, 2)])


BIG = Z(2, 3)
LENS = Z(2)


@pytest.mark.parametrize("kw,error,match", [
    (dict(refs=Z(6, dtype=torch.int64)), ValueError, "refs"),
    (dict(refs=Z(0)), ValueError, "refs"),
    (dict(refs=Z(12)[::2]), ValueError, "refs"),
    (dict(block_table=Z(2, 3, dtype=torch.int64)), ValueError, "block_table"),
    (dict(block_table=Z(2, 0)), ValueError, "block_table"),
    (dict(block_table=Z(3, 2).t()), ValueError, "dense rows"),
    (dict(block_table=Z(1, 3).expand(2, 3)), ValueError, "dense rows"),
    (dict(block_table=Z(8193, 3), seq_lens=Z(8193), parents=Z(8193)), ValueError, "8192 rows"),
    (dict(block_table=Z(2, 1 << 27)), ValueError, "tokens"),
    (dict(pools=[]), ValueError, "empty"),
    (dict(pools=[_pool(5)]), ValueError, "of 6 pages"),
    (dict(pools=[_pool(), _pool(6, 2, 32)]), ValueError, "one page_size"),
    (dict(seq_lens=Z(3)), ValueError, "seq_lens"),
    (dict(seq_lens=Z(4)[::2]), ValueError, "seq_lens"),
    (dict(parents=Z(3)), ValueError, "parents"),
    (dict(new_lens=Z(2, dtype=torch.float32)), ValueError, "new_lens"),
    (dict(status=Z(2)), ValueError, "status"),
    (dict(seq_lens=LENS, new_lens=LENS), ValueError, "share memory"),
    (dict(block_table=BIG, parents=BIG[0, :2]), ValueError, "share memory"),
    (dict(), RuntimeError, "GPU"),
    (dict(parents=None, new_lens=Z(2), status=Z(1), _workspace={}), RuntimeError, "GPU"),
])
def test_fork_refuses(kw, error, match):
    from tritonkv_amd.pages import fork_rows

    a = dict(pools=[_pool()], block_table=Z(2, 3), seq_lens=Z(2), refs=Z(6), parents=Z(2))
    a.update(kw)
    with pytest.raises(error, match=match):
        fork_rows(**a)


def test_state_may_lie_in_one_buffer():
    from tritonkv_amd.pages import fork_rows

    state = Z(20)
    with pytest.raises(RuntimeError, match="GPU"):
        fork_rows([_pool()], state[:6].view(2, 3), state[6:8], state[8:14], state[14:16], state[16:18], state[18:19])
    with pytest.raises(ValueError, match="share memory"):
        fork_rows([_pool()], state[:6].view(2, 3), state[5:7], state[8:14], state[14:16])


def test_resize_needs_lengths():
    from tritonkv_amd.pages import resize_rows

    with pytest.raises(ValueError, match="new_lens"):
        resize_rows([_pool()], Z(2, 3), Z(2), Z(6), None)


T, R = Z(2, 3), Z(6)


@pytest.mark.parametrize("kw,error,match", [
    (dict(out=(Z(2, 4), Z(6))), ValueError, "shapes"),
    (dict(out=(Z(2, 3), Z(7))), ValueError, "shapes"),
    (dict(block_table=T, out=(T, Z(6))), ValueError, "share memory"),
    (dict(refs=R, out=(Z(2, 3), R)), ValueError, "share memory"),
    (dict(live=Z(2)), ValueError, "live"),
    (dict(refs=R, live=R[:1]), ValueError, "share memory"),
    (dict(pools=[]), ValueError, "empty"),
    (dict(pools=[_pool(7)]), ValueError, "of 6 pages"),
    (dict(), RuntimeError, "GPU"),
])
def test_compact_refuses(kw, error, match):
    from tritonkv_amd.pages import compact_pages

    a = dict(pools=[_pool()], block_table=Z(2, 3), refs=Z(6))
    a.update(kw)
    with pytest.raises(error, match=match):
        compact_pages(**a)


def test_argument_blocks_match_the_header():
    from tritonkv_amd import _lib

    for struct, name in ((_lib.PageSet, "tkv_page_set"), (_lib.CopyPagesArgs, "tkv_copy_pages_args"),
                         (_lib.ForkRowsArgs, "tkv_fork_rows_args"),
                         (_lib.CompactPagesArgs, "tkv_compact_pages_args")):
        fields = [f for f, _ in struct._fields_]
        src = '#include <stdio.h>\n#include <stddef.h>\n#include "tkv.h"\nint main(void) { printf("%zu", sizeof(' \
            + name + "));\n" + "".join(f'printf(" %zu", offsetof({name}, {f}));\n' for f in fields) + "return 0; }"
        with tempfile.TemporaryDirectory() as d:
            c = os.path.join(d, "l.c")
            open(c, "w").write(src)
            subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", c[:-2]], check=True)
            vals = [int(x) for x in subprocess.run([c[:-2]], capture_output=True, text=True, check=True).stdout.split()]
        assert vals == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


def test_work_sizes():
    from tritonkv_amd import _lib

    lib = _lib.load()
    c = _lib.CopyPagesArgs(set=_set(_lib), src=0x1000, dst=0x1000, n=4096, src_pages=100, dst_pages=7)
    assert lib.tkv_copy_pages_work(c) == 0  # 4096 pages of 4 KiB
    c.n = 4097
    assert lib.tkv_copy_pages_work(c) >= 107 + 2 * 4097
    c.n, c.set.bytes[0], c.set.src_stride[0], c.set.dst_stride[0] = 32, 1 << 20, 1 << 20, 1 << 20
    assert lib.tkv_copy_pages_work(c) >= 107 + 2 * 32
    assert lib.tkv_fork_rows_work(4, 10, 100, 1) - lib.tkv_fork_rows_work(4, 10, 100, 0) == 40
    assert lib.tkv_fork_rows_work(4, 10, 100, 0) >= 6 * 4 + 100
    assert lib.tkv_compact_pages_work(100) >= 250
    c.n = 0
    for bad in (lib.tkv_copy_pages_work(c), lib.tkv_fork_rows_work(0, 1, 1, 0),
                lib.tkv_compact_pages_work(0)):
        assert bad == -1


def _set(_lib):
    s = _lib.PageSet(count=1)
    s.src[0] = s.dst[0] = 0x1000
    s.src_stride[0] = s.dst_stride[0] = s.bytes[0] = 4096
    return s


@pytest.mark.parametrize("change", [dict(count=33), dict(count=-1), dict(src=0), dict(dst=0x1008), dict(bytes=0),
                                    dict(bytes=4104), dict(src_stride=4088), dict(dst_stride=2048)])
def test_c_entries_refuse_page_sets(change):
    from tritonkv_amd import _lib

    lib, d = _lib.load(), 0x1000
    s = _set(_lib)
    for name, value in change.items():
        if name == "count":
            s.count = value
        else:
            getattr(s, name)[0] = value
    c = _lib.CopyPagesArgs(set=s, src=d, dst=d, work=d, n=3, src_pages=6, dst_pages=6, same=1)
    f = _lib.ForkRowsArgs(set=s, block_table=d, seq_lens=d, refs=d, status=d, work=d, table_stride=3, B=2,
                          max_pages=3, page_size=16, num_pages=6)
    p = _lib.CompactPagesArgs(set=s, block_table=d, refs=d, out_table=d, out_refs=d, work=d, table_stride=3,
                              out_stride=3, B=2, max_pages=3, num_pages=6)
    assert lib.tkv_copy_pages(ctypes.byref(c), None) == _lib.TKV_EINVAL
    assert lib.tkv_fork_rows(ctypes.byref(f), None) == _lib.TKV_EINVAL
    assert lib.tkv_compact_pages(ctypes.byref(p), None) == _lib.TKV_EINVAL
    assert lib.tkv_copy_planned(ctypes.byref(s), d, 3, None) == _lib.TKV_EINVAL


@pytest.mark.parametrize("kind,field,value", [
    ("copy", "src", None), ("copy", "dst", None), ("copy", "n", 0), ("copy", "src_pages", 0),
    ("copy", "dst_pages", 0), ("copy", "dst_pages", 7), ("copy", "n", 8193), ("copy", "n", -1),
    ("fork", "block_table", None), ("fork", "seq_lens", None), ("fork", "refs", None), ("fork", "status", None),
    ("fork", "work", None), ("fork", "work", 0x1004), ("fork", "B", 0), ("fork", "max_pages", 0),
    ("fork", "num_pages", 0), ("fork", "page_size", 0), ("fork", "table_stride", 2),
    ("fork", "page_size", 1 << 30),
    ("compact", "block_table", None), ("compact", "out_refs", None), ("compact", "work", 0x1008),
    ("compact", "out_stride", 2), ("compact", "num_pages", 0)])
def test_c_entries_refuse(kind, field, value):
    from tritonkv_amd import _lib

    lib, d = _lib.load(), 0x1000
    s = _set(_lib)
    a, fn = {
        "copy": (_lib.CopyPagesArgs(set=s, src=d, dst=d, n=3, src_pages=6, dst_pages=6, same=1),
                 lib.tkv_copy_pages),
        "fork": (_lib.ForkRowsArgs(set=s, block_table=d, seq_lens=d, refs=d, status=d, work=d, table_stride=3, B=2,
                                   max_pages=3, page_size=16, num_pages=6), lib.tkv_fork_rows),
        "compact": (_lib.CompactPagesArgs(set=s, block_table=d, refs=d, out_table=d, out_refs=d, work=d,
                                          table_stride=3, out_stride=3, B=2, max_pages=3, num_pages=6),
                    lib.tkv_compact_pages)}[kind]
    setattr(a, field, value)
    assert fn(ctypes.byref(a), None) == _lib.TKV_EINVAL
    assert fn(None, None) == _lib.TKV_EINVAL


def test_too_many_rows_for_the_c_entry():
    from tritonkv_amd import _lib

    d = 0x1000
    f = _lib.ForkRowsArgs(set=_set(_lib), block_table=d, seq_lens=d, refs=d, status=d, work=d, table_stride=3,
                          B=8193, max_pages=3, page_size=16, num_pages=6)
    assert _lib.load().tkv_fork_rows(ctypes.byref(f), None) == _lib.TKV_EUNSUPPORTED


def test_too_many_pages():
    from tritonkv_amd import _lib
    from tritonkv_amd.pages import copy_pages, fork_rows

    lib, d, n = _lib.load(), 0x1000, 2 ** 30 + 1
    s = _set(_lib)
    for kw in (dict(n=n), dict(src_pages=n, dst_pages=n, same=1), dict(src_pages=n)):
        c = _lib.CopyPagesArgs(set=s, src=d, dst=d, work=d, **(dict(n=3, src_pages=6, dst_pages=6) | kw))
        assert lib.tkv_copy_pages(ctypes.byref(c), None) == _lib.TKV_EUNSUPPORTED
        assert lib.tkv_copy_pages_work(ctypes.byref(c)) == _lib.TKV_EUNSUPPORTED
    f = _lib.ForkRowsArgs(set=s, block_table=d, seq_lens=d, refs=d, status=d, work=d, table_stride=3, B=2,
                          max_pages=3, page_size=16, num_pages=n)
    p = _lib.CompactPagesArgs(set=s, block_table=d, refs=d, out_table=d, out_refs=d, work=d, table_stride=3,
                              out_stride=3, B=2, max_pages=3, num_pages=n)
    assert lib.tkv_fork_rows(ctypes.byref(f), None) == _lib.TKV_EUNSUPPORTED
    assert lib.tkv_compact_pages(ctypes.byref(p), None) == _lib.TKV_EUNSUPPORTED
    many = torch.empty(1, dtype=torch.uint8).expand(n, 1, 16, 16)
    with pytest.raises(ValueError, match="at most"):
        copy_pages([many], Z(1), Z(1))
    with pytest.raises(ValueError, match="at most"):
        copy_pages([_pool()], Z(1).expand(n), Z(1).expand(n))
    wide = torch.empty(2, 2 ** 30, dtype=torch.int32)  # (never touched)
    with pytest.raises(ValueError, match="at most"):
        fork_rows([_pool()], wide, Z(2), Z(6), Z(2))


def test_a_kept_call_refuses_what_shares_memory():
    from tritonkv_amd import _lib
    from tritonkv_amd.pages import _APART, _WRITTEN

    b = Z(64)
    table, status, parents = b[:8].view(2, 4), b[8:9], b[16:18]
    call = _lib.host().prepare(bytes(_lib.ForkRowsArgs()), _lib.address("tkv_fork_rows"), 0,
                               ((table, -1, 4, 1 | _WRITTEN), (status, 0, 4, _WRITTEN), (parents, 8, 4, _APART),
                                (parents, 16, 4, _APART)), None)
    run = _lib.host().run
    # (a call without these faults would ask for the device's stream)
    for s, p0, p1 in ((b[7:8], parents, parents), (status, b[7:9], parents), (status, parents, b[6:8]),
                      (b[17:18], parents, parents), (b[20:21], parents, b[19:21])):
        assert run(call, table, s, p0, p1) is None
    with pytest.raises(ValueError, match="too many"):
        _lib.host().prepare(b"", 0, 0, ((table, -1, 4, _APART),) * 17, None)
