"""Pages of a cache on the device: copied, forked, handed out, taken back, compacted.

A paged cache is page pools (of any layer, K and V; 2/4-bit
:class:`~tritonkv_amd.quantize.QuantizedTensor` pools of
:mod:`tritonkv_amd.paged`, 8-bit ones of :mod:`tritonkv_amd.paged8` or 16-bit tensors of
:mod:`tritonkv_amd.paged16`)
that share page numbers, and three int32 tensors that say which row owns what:

* ``block_table`` ``(B, max_pages)``: row b's pages in order, -1 after them;
* ``seq_lens`` ``(B,)``: its tokens, or as many as it has room for; it uses
  ``ceil(seq_lens[b] / page_size)`` pages;
* ``refs`` ``(num_pages,)``: how many used table entries name each page, 0 for
  a free one.  (A caller may add counts of its own to keep pages alive.)

An empty cache is a table of -1 and two tensors of zeros.  From there
:func:`resize_rows` makes room, truncates and frees, :func:`fork_rows` makes
rows out of other rows (parallel samples, beams, a shared prefix), sharing
their full pages, and :func:`compact_pages` moves the live pages to the low end
of the pools.  A page that is not full belongs to one row alone, so the appends
(:func:`~tritonkv_amd.paged.paged_append`, ``paged16_append`` and the decodes'
fused ones) never write into another row's tokens.  Where rows hold room made ahead,
whose pages are full only by ``seq_lens``, this takes ``written``, the tokens that
they really hold: :func:`fork_rows`.

Everything runs on the current stream, in two launches, from device tensors
alone: nothing is copied to the host and no call synchronises.  Calls that may
overlap in time must not share a ``_workspace``.
"""

from __future__ import annotations

import torch

from . import _lib
from .paged8 import Paged8Pool
from .paged16 import _buffer, _int32_arg, _keep16, _offset
from .kernels.fused_decode_attn import _prepared
from .quantize import QuantizedTensor, _require_gpu

MAX_ROWS = 8192
MAX_PAGES = 2 ** 30


def _tensors(pools) -> list:
    """The page tensors of pools, in order."""
    if isinstance(pools, (QuantizedTensor, Paged8Pool, torch.Tensor)):
        raise TypeError("pools must be a list or tuple of page pools")
    found = []
    for p in pools:
        if isinstance(p, QuantizedTensor):
            found += [p.packed, p.scale, p.zero]
        elif isinstance(p, Paged8Pool):
            found += p.page_tensors()
        elif isinstance(p, torch.Tensor):
            found.append(p)
        else:
            raise TypeError(f"a page pool is a QuantizedTensor, a Paged8Pool or a tensor, got {type(p).__name__}")
    return found


def _page_size(pools) -> int:
    pages = [p.packed if isinstance(p, QuantizedTensor) else p.codes if isinstance(p, Paged8Pool) else p for p in pools]
    sizes = {p.shape[2] for p in pages if p.dim() == 4}
    if len(sizes) != 1:
        raise ValueError(f"the pools must be (num_pages, HKV, page_size, ...) of one page_size, got {sorted(sizes)}")
    return sizes.pop()


def _check_pages(tensors: list, num_pages: int | None, device, what: str) -> list:
    """``(address, page stride in bytes, bytes of a page)`` of every page tensor."""
    found = []
    for t in tensors:
        if t.dim() != 4 or t.numel() == 0 or (num_pages is not None and t.shape[0] != num_pages):
            raise ValueError(f"{what} must hold (num_pages, HKV, page_size, ...) tensors"
                             + ("" if num_pages is None else f" of {num_pages} pages") + f", got {tuple(t.shape)}")
        if t.shape[0] > MAX_PAGES:
            raise ValueError(f"{what}: at most {MAX_PAGES} pages, got {t.shape[0]}")
        if t.device != device:
            raise ValueError(f"{what} must be on {device}, got a tensor on {t.device}")
        if t.is_contiguous():
            size = stride = t.numel() // t.shape[0] * t.element_size()
        else:
            dense = 1  # a page is one block of memory, in whatever order of its axes
            for stride, n in sorted((s, n) for s, n in zip(t.stride()[1:], t.shape[1:]) if n > 1):
                if stride != dense:
                    raise ValueError(f"{what}: a page must be one dense block, got strides {tuple(t.stride())}")
                dense *= n
            size = dense * t.element_size()
            stride = t.stride(0) * t.element_size() if t.shape[0] > 1 else size
        if stride < size:
            raise ValueError(f"{what}: pages overlap, got strides {tuple(t.stride())}")
        if size % 16 or stride % 16 or t.data_ptr() % 16:
            raise ValueError(f"{what}: pages must start on 16 bytes and be a multiple of them, got {size} bytes "
                             f"every {stride}")
        found.append((t.data_ptr(), stride, size))
    return found


def _page_sets(src: list, dst: list) -> list:
    """The tensors as sets of at most ``PAGE_TENSORS``; one empty set without any."""
    n = _lib.PAGE_TENSORS
    sets = []
    for first in range(0, max(1, len(src)), n):
        one = _lib.PageSet(count=len(src[first:first + n]))
        from_, to, from_stride, to_stride, size = one.src, one.dst, one.src_stride, one.dst_stride, one.bytes
        for i, (s, d) in enumerate(zip(src[first:first + n], dst[first:first + n])):
            from_[i], from_stride[i], size[i] = s
            to[i], to_stride[i], _ = d
        sets.append(one)
    return sets


def _work(ws: dict | None, name: str, n: int, device) -> torch.Tensor:
    return _buffer({} if ws is None else ws, name, n, torch.int32, device)


def _check_rows(block_table, refs) -> tuple:
    """B and max_pages of a table that is written in place, and the pages of refs."""
    if not isinstance(refs, torch.Tensor) or refs.dtype != torch.int32 or refs.dim() != 1 or refs.numel() == 0 \
            or not refs.is_contiguous():
        raise ValueError("refs must be a contiguous int32 (num_pages,) tensor")
    if not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32 or block_table.dim() != 2 \
            or block_table.numel() == 0 or block_table.device != refs.device or _row_stride(block_table) is None:
        raise ValueError("block_table must be an int32 (B, max_pages) tensor with dense rows on refs' device")
    if refs.numel() > MAX_PAGES or block_table.numel() > 2 ** 31 - 1:
        raise ValueError(f"at most {MAX_PAGES} pages and 2**31 - 1 table entries, got {refs.numel()} and "
                         f"{block_table.numel()}")
    return block_table.shape


def _row_stride(t: torch.Tensor) -> int | None:
    """Entries between the rows of a table, None if its rows are not dense or overlap."""
    B, P = t.shape
    if P > 1 and t.stride(1) != 1:
        return None
    stride = t.stride(0) if B > 1 else P
    return stride if stride >= P else None


def _span(t: torch.Tensor) -> tuple:
    """First and last address of t's entries."""
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() - 1


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a and b share memory.  Two that lie in turn at one stride, such as the halves of a
    pool of paired pages or columns of one table, do not; at different strides, meeting
    address ranges count as shared."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a0 > b1 or b0 > a1:
        return False
    stride = a.stride(0) * a.element_size()
    if a.dim() < 2 or b.dim() < 2 or stride <= 0 or stride != b.stride(0) * b.element_size():
        return True
    size = [_span(t[0]) for t in (a, b)]
    between = (b0 - a0) % stride
    return between <= size[0][1] - size[0][0] or between + size[1][1] - size[1][0] >= stride


_C = {f: _offset(_lib.CopyPagesArgs, f) for f in ("src", "dst")}
_F = {f: _offset(_lib.ForkWrittenArgs, f) for f in ("parents", "new_lens", "status", "written")}
_P = {f: _offset(_lib.CompactPagesArgs, f) for f in ("live",)}
_APART, _WRITTEN = 2, 4  # flags of a kept call's tensors: apart from written ones; written


def copy_pages(pools, src: torch.Tensor, dst: torch.Tensor, dst_pools=None, _workspace: dict | None = None) -> None:
    """Page ``dst[i]`` := page ``src[i]`` in every one of ``pools``, for all pairs of one call.

    pools: a list of page pools that share page numbers; ``src`` and ``dst``:
    int32 ``(n,)`` tensors on their device.  With ``dst_pools``, a list of
    pools of the same pages in other memory, pages go from ``pools`` to
    those.  A pair with a number outside the pools is skipped (-1 marks one
    that is not wanted).  Of several pairs with one destination the first is
    carried out.  Within one set of pools a page that the call reads is
    never written: a pair whose destination is a pair's source is skipped.
    """
    tensors = _tensors(pools)
    others = None if dst_pools is None else _tensors(dst_pools)
    key = None
    if _workspace is not None:
        key = ("copy_pages", len(tensors), others is None)
        prep = _prepared(_workspace, key)
        if prep is not None and prep.run(src, dst, *tensors, *(others or ())):
            return
    if not tensors:
        raise ValueError("pools is empty")
    device = tensors[0].device
    from_ = _check_pages(tensors, tensors[0].shape[0], device, "pools")
    to = from_
    src_pages = dst_pages = tensors[0].shape[0]
    if others is not None:
        if len(others) != len(tensors):
            raise ValueError(f"dst_pools must hold as many tensors as pools: {len(others)} and {len(tensors)}")
        dst_pages = others[0].shape[0] if others[0].dim() else 0
        to = _check_pages(others, dst_pages, device, "dst_pools")
        for a, b in zip(tensors, others):
            order = [sorted((i for i in range(1, 4) if t.shape[i] > 1), key=t.stride) for t in (a, b)]
            if a.shape[1:] != b.shape[1:] or a.dtype != b.dtype or order[0] != order[1]:
                raise ValueError(f"dst_pools must have pools' page shapes, order and dtypes: {tuple(a.shape)} "
                                 f"{a.dtype} and {tuple(b.shape)} {b.dtype}")
        if any(_overlap(a, b) for a in tensors for b in others):
            raise ValueError("dst_pools must not share memory with pools")
    if not isinstance(src, torch.Tensor):
        raise ValueError("src must be an int32 tensor of page numbers")
    n = src.numel()
    if n > MAX_PAGES:
        raise ValueError(f"at most {MAX_PAGES} pairs, got {n}")
    s, d = (_int32_arg(x, n, device, name, "page numbers, as many as the other")
            for name, x in (("src", src), ("dst", dst)))
    _require_gpu(tensors[0], "copy_pages")
    if n == 0:
        return
    sets = _page_sets(from_, to)
    work = None
    for one in sets:
        args = _lib.CopyPagesArgs(set=one, src=s.data_ptr(), dst=d.data_ptr(), n=n, src_pages=src_pages,
                                  dst_pages=dst_pages, same=int(others is None))
        words = _lib.load().tkv_copy_pages_work(args)
        if words > 0:
            work = _work(_workspace, "copy_pages", words, device)
            args.work = work.data_ptr()
        _lib.check(_lib.launch(device, "tkv_copy_pages", args), "copy_pages")
    if key is not None and len(sets) == 1:
        _keep16(_workspace, key, args, "tkv_copy_pages", "copy_pages", device, (work,),
                ((src, _C["src"], 4), (dst, _C["dst"], 4),
                 *((t, -1, 16, 1) for t in (*tensors, *(others or ())))))


def fork_rows(pools, block_table: torch.Tensor, seq_lens: torch.Tensor, refs: torch.Tensor,
              parents: torch.Tensor | None, new_lens: torch.Tensor | None = None,
              status: torch.Tensor | None = None, _workspace: dict | None = None, *,
              written: torch.Tensor | None = None) -> torch.Tensor:
    """Make every row of a block table out of an old row, in place.

    Row b becomes the first ``min(new_lens[b], seq_lens[a])`` tokens of old
    row ``a = parents[b]``, with pages for ``new_lens[b]`` tokens;
    ``new_lens=None`` keeps ``a``'s length, ``parents=None`` every row's own
    tokens, and a parent outside ``[0, B)`` (say -1) empties the row.  So

    * ``parents = arange(B)`` with some entries changed forks rows into empty
      or finished ones, a beam search's choice of beams reorders them;
    * a smaller ``new_lens`` truncates, 0 or a parent of -1 frees;
    * a larger one makes room: tokens from the old length on are whatever the
      new pages hold until they are written.

    ``written``, an int32 ``(B,)`` tensor, says how many of its ``seq_lens`` tokens
    every old row holds (None: all of them).  It is needed where an old row has room
    that was made ahead and is not written yet: without it the full pages of that room
    would be shared, and the rows would write their next tokens over each other's.
    With it only full pages of written tokens are shared; the pages of room stay with
    the row that keeps the partial page, and other rows get new ones.  (The rows made
    hold ``min(written[parents[b]], new_lens[b])`` tokens.)

    Full pages are shared (``refs`` counts the rows).  The page that a row ends
    in, if not full, stays with one row -- the parent itself, else its first
    child -- if no other row keeps it, and is copied for every other one, in
    all of ``pools``, by the same launch that rewrites the table.  New pages are
    the lowest that were free before the call, in row order, whatever runs
    in parallel.  At most 8192 rows.

    Returns ``status``, an int32 ``(1,)`` tensor: 0, or 1 where the free
    pages, or 2 where a row's table entries, do not suffice; then nothing was
    changed.  It is on the device, so reading it is what waits for the call.
    """
    tensors = _tensors(pools)
    key = None
    if _workspace is not None:
        key = ("fork_rows", len(tensors))
        prep = _prepared(_workspace, key)
        if prep is not None:
            got = status
            if got is None and isinstance(refs, torch.Tensor):
                got = torch.empty(1, dtype=torch.int32, device=refs.device)
            if prep.run(block_table, seq_lens, refs, parents, new_lens, written, got, *tensors):
                return got
    B, max_pages = _check_rows(block_table, refs)
    device, num_pages = refs.device, refs.numel()
    if B > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows, got {B}")
    if not tensors:
        raise ValueError("pools is empty")
    pages = _check_pages(tensors, num_pages, device, "pools")
    page_size = _page_size(pools)
    if max_pages * page_size > 2 ** 31 - 1:
        raise ValueError(f"{max_pages} pages of {page_size} tokens a row: at most 2**31 - 1 tokens")
    if not isinstance(seq_lens, torch.Tensor) or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous int32 tensor of B lengths: it is written in place")
    _int32_arg(seq_lens, B, device, "seq_lens", "B lengths")
    par = None if parents is None else _int32_arg(parents, B, device, "parents", "B rows")
    new = None if new_lens is None else _int32_arg(new_lens, B, device, "new_lens", "B lengths")
    held = None if written is None else _int32_arg(written, B, device, "written", "B token counts")
    outputs = [block_table, seq_lens, refs]
    if status is None:
        status_given = torch.empty(1, dtype=torch.int32, device=device)
    else:
        status_given = _int32_arg(status, 1, device, "status", "one entry")
        outputs.append(status)
    inputs = [x for x in (parents, new_lens, written) if x is not None]
    for i, a in enumerate(outputs):
        if any(_overlap(a, b) for b in outputs[i + 1:] + inputs):
            raise ValueError("block_table, seq_lens, refs and status are written: they must not share memory "
                             "with each other, parents, new_lens or written")
    _require_gpu(refs, "fork_rows")
    words = _lib.load().tkv_fork_rows_work(B, max_pages, num_pages, int(par is not None))
    work = _work(_workspace, "fork_rows", words, device)
    sets = _page_sets(pages, pages)
    args = _lib.ForkWrittenArgs(
        set=sets[0], block_table=block_table.data_ptr(), seq_lens=seq_lens.data_ptr(), refs=refs.data_ptr(),
        parents=_lib.ptr(par), new_lens=_lib.ptr(new), written=_lib.ptr(held), status=status_given.data_ptr(),
        work=work.data_ptr(),
        table_stride=_row_stride(block_table), B=B, max_pages=max_pages, page_size=page_size, num_pages=num_pages)
    _lib.check(_lib.launch(device, "tkv_fork_rows_written", args), "fork_rows")
    for one in sets[1:]:
        _lib.check(_lib.launch(device, "tkv_copy_planned", one, work.data_ptr(), B), "fork_rows")
    if key is not None and len(sets) == 1:
        _keep16(_workspace, key, args, "tkv_fork_rows_written", "fork_rows", device, (work,),
                ((block_table, -1, 4, 1 | _WRITTEN), (seq_lens, -1, 4, _WRITTEN), (refs, -1, 4, _WRITTEN),
                 (parents, _F["parents"], 4, _APART), (new_lens, _F["new_lens"], 4, _APART),
                 (written, _F["written"], 4, _APART),
                 (status_given, _F["status"], 4, _WRITTEN), *((t, -1, 16, 1) for t in tensors)))
    return status_given


def resize_rows(pools, block_table: torch.Tensor, seq_lens: torch.Tensor, refs: torch.Tensor,
                new_lens: torch.Tensor, status: torch.Tensor | None = None,
                _workspace: dict | None = None, *, written: torch.Tensor | None = None) -> torch.Tensor:
    """Give every row ``new_lens[b]`` tokens: :func:`fork_rows` with every row its own parent.

    Rows that grow get pages, rows that shrink return theirs, a length of 0
    frees the row.  A row cut inside a page that it shares gets its own
    copy of that page.  ``written`` as there; rows keep the room that is their own.
    """
    if new_lens is None:
        raise ValueError("new_lens must be an int32 tensor of B lengths")
    return fork_rows(pools, block_table, seq_lens, refs, None, new_lens, status, _workspace, written=written)


def compact_pages(pools, block_table: torch.Tensor, refs: torch.Tensor, out=None,
                  live: torch.Tensor | None = None, _workspace: dict | None = None) -> tuple:
    """Move the live pages (``refs > 0``) to the low end of the pools.

    With n of them, the i-th live page at or past n is copied to the i-th free
    page below n in every one of ``pools``; afterwards pages n and up are free,
    and the pools' tails may be given back or lent out.  Returns
    ``(block_table, refs, live)`` with the new numbers and counts, ``live`` an
    int32 ``(1,)`` tensor holding n.  ``out``: a table and counts to write
    instead of the given ones, which then stay valid, as do the pages they
    name, until something is written to the pools: readers may go on with the
    old table and be switched over later.
    """
    tensors = _tensors(pools)
    out_table, out_refs = (block_table, refs) if out is None else out
    key = None
    if _workspace is not None:
        key = ("compact_pages", len(tensors))
        prep = _prepared(_workspace, key)
        if prep is not None:
            got = live
            if got is None and isinstance(refs, torch.Tensor):
                got = torch.empty(1, dtype=torch.int32, device=refs.device)
            if prep.run(block_table, refs, out_table, out_refs, got, *tensors):
                return out_table, out_refs, got
    B, max_pages = _check_rows(block_table, refs)
    device, num_pages = refs.device, refs.numel()
    if out is not None:
        _check_rows(out_table, out_refs)
        if out_table.shape != block_table.shape or out_refs.shape != refs.shape or out_refs.device != device:
            raise ValueError("out must be a table and counts of the given ones' shapes on their device")
        if _overlap(out_table, block_table) or _overlap(out_refs, refs) or _overlap(out_table, refs) \
                or _overlap(out_refs, block_table):
            raise ValueError("out must not share memory with block_table or refs")
    if _overlap(out_table, out_refs):
        raise ValueError("block_table and refs must not share memory")
    if not tensors:
        raise ValueError("pools is empty")
    pages = _check_pages(tensors, num_pages, device, "pools")
    if live is None:
        live_given = torch.empty(1, dtype=torch.int32, device=device)
    else:
        live_given = _int32_arg(live, 1, device, "live", "one entry")
        if any(_overlap(live, t) for t in (block_table, refs, out_table, out_refs)):
            raise ValueError("live must not share memory with the tables or counts")
    _require_gpu(refs, "compact_pages")
    words = _lib.load().tkv_compact_pages_work(num_pages)
    work = _work(_workspace, "compact_pages", words, device)
    sets = _page_sets(pages, pages)
    args = _lib.CompactPagesArgs(
        set=sets[0], block_table=block_table.data_ptr(), refs=refs.data_ptr(), out_table=out_table.data_ptr(),
        out_refs=out_refs.data_ptr(), live=live_given.data_ptr(), work=work.data_ptr(),
        table_stride=_row_stride(block_table), out_stride=_row_stride(out_table), B=B, max_pages=max_pages,
        num_pages=num_pages)
    _lib.check(_lib.launch(device, "tkv_compact_pages", args), "compact_pages")
    for one in sets[1:]:
        _lib.check(_lib.launch(device, "tkv_copy_planned", one, work.data_ptr(), num_pages // 2), "compact_pages")
    if key is not None and len(sets) == 1:
        _keep16(_workspace, key, args, "tkv_compact_pages", "compact_pages", device, (work,),
                ((block_table, -1, 4, 1 | _APART), (refs, -1, 4, _APART), (out_table, -1, 4, 1 | _APART),
                 (out_refs, -1, 4, _APART), (live_given, _P["live"], 4, _WRITTEN),
                 *((t, -1, 16, 1) for t in tensors)))
    return out_table, out_refs, live_given


__all__ = ["MAX_ROWS", "copy_pages", "fork_rows", "resize_rows", "compact_pages"]
