"""16-bit paged KV cache: fp16 and bf16 page pools, their append and their decode.

The unquantized counterpart of :mod:`tritonkv_amd.paged`.  A pool is a plain
tensor ``(num_pages, HKV, page_size, D)`` of ``torch.float16`` or
``torch.bfloat16``; logical token t of batch row b lives in page
``block_table[b, t // page_size]`` at slot ``t % page_size``.  Pools are used
as they are strided, as long as a token's D values are dense and rows start on
16 bytes: a token-major pool seen as ``(num_pages, page_size, HKV,
D).transpose(1, 2)`` or the K half of a ``(num_pages, 2, HKV, page_size, D)``
pool is one.  ``page_size`` is a multiple of 16.

The decode cuts the rows' tokens on the device, from ``seq_lens`` itself:
tables may be as wide as the longest request can get, and a captured step
keeps a balanced split as the rows grow.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .kernels.fused_decode_attn import _backend, _check_out, _PreparedCall, _prepared, compute_units
from .paged import _check_table
from .quantize import _require_gpu

PAGE_MULTIPLE = 16
HEAD_DIMS = (64, 128, 256)
DTYPES = (torch.float16, torch.bfloat16)


def empty_paged16_pool(num_pages: int, HKV: int, page_size: int, D: int,
                       dtype: torch.dtype = torch.float16, device="cuda") -> torch.Tensor:
    """An uninitialised 16-bit page pool of ``num_pages`` pages of ``page_size`` tokens."""
    if page_size <= 0 or page_size % PAGE_MULTIPLE:
        raise ValueError(f"page_size must be a positive multiple of {PAGE_MULTIPLE}, got {page_size}")
    if num_pages <= 0 or HKV <= 0:
        raise ValueError(f"num_pages and HKV must be positive, got {num_pages} and {HKV}")
    if D not in HEAD_DIMS:
        raise ValueError(f"D must be one of {HEAD_DIMS}, got {D}")
    if dtype not in DTYPES:
        raise TypeError(f"dtype must be float16 or bfloat16, got {dtype}")
    return torch.empty(num_pages, HKV, page_size, D, dtype=dtype, device=device)


def _dense_rows(t: torch.Tensor, align: int) -> bool:
    """Whether t's last axis is dense and every row starts on 16 bytes (``align`` elements)."""
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and \
        all(s % align == 0 for s, n in zip(t.stride()[:-1], t.shape) if n > 1)


def _strides(t: torch.Tensor, align: int) -> tuple:
    """t's strides without the last axis; those of axes of one entry, which nothing
    multiplies, as ``align``."""
    return tuple(s if n > 1 else align for s, n in zip(t.stride()[:-1], t.shape))


def _check_pools16(k_pool, v_pool) -> tuple:
    for name, pool in (("k_pool", k_pool), ("v_pool", v_pool)):
        if not isinstance(pool, torch.Tensor) or pool.dim() != 4:
            raise ValueError(f"{name} must be a (num_pages, HKV, page_size, D) tensor")
        if pool.dtype not in DTYPES:
            raise TypeError(f"{name} must be float16 or bfloat16, got {pool.dtype}")
        if pool.numel() == 0:
            raise ValueError(f"{name} is empty")
        if not _dense_rows(pool, 8) or any(s == 0 for s in _strides(pool, 8)):
            raise ValueError(f"{name} must hold each token's D values densely, on 16-byte boundaries")
    if v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype or v_pool.device != k_pool.device:
        raise ValueError("K and V pools must have the same shape, dtype and device")
    num_pages, HKV, page_size, D = k_pool.shape
    if page_size % PAGE_MULTIPLE:
        raise ValueError(f"page_size must be a multiple of {PAGE_MULTIPLE}, got {page_size}")
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {D}")
    return num_pages, HKV, page_size, D


def _int32_arg(t, n: int, device, name: str, what: str):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n \
            or t.device != device:
        raise ValueError(f"{name} must be an int32 tensor of {what} on the pools' device")
    return t.contiguous()


MAX_ROWS = MAX_WORKGROUPS = 65535  # grid y-dimension limit


def plan_shares(B: int, HKV: int, G: int, S: int, D: int = 128, device=None,
                piece_tokens: int | None = None) -> tuple[int, int, int, int]:
    """``(least_chunks, workgroups, long_workgroups, long_chunks)`` of a decode (``include/tkv.h``).

    ``S`` is the tables' capacity, all that the host knows of the lengths: it decides whether
    rows stay whole, the least share and the number of workgroups; the cut itself follows the
    lengths, on the device.
    ``piece_tokens`` fixes a workgroup's tokens instead.  The rules, with
    what was measured on MI355X (us of a captured step; U = HKV times the
    blocks of query heads, 16 or for more 32, the workgroups that attend to the same tokens):

    * Rows stay whole, in one launch, where that was faster than cutting them
      and joining (a second launch, 2.4 us and more): one CU reads at most
      38 GB/s, so only in narrow tables, or with many rows.  Up to 256 tokens of 128 dims
      (250 tokens, D 128: B * U = 2 5.8 whole, 6.8 cut; 32 6.3, 7.1; D 256 10.7,
      7.9).  Twice that where B * U * D is 16384 or more (whole / cut, 505 tokens of 128
      dims: B * U = 32 10.3 / 7.6, 64 10.7 / 8.9, 128 11.2 / 11.1, 256 12.9 / 15.8, 504 22.6 /
      26.5; 1-505 tokens: 64 10.2 / 9.9, 128 10.6 / 11.6; 1000 of 64 dims: 64 11.5 / 9.1, 128
      12.0 / 10.8, 256 13.2 / 15.8; 250 of 256 dims: 32 11.7 / 8.5, 64 12.3 / 13.7).  Four times
      from 512 units on (up to 512 of 1024: 512 units 19.9 / 23.7; all 1000: 512 44.0 / 46.0,
      1024 85 / 87; but 1-1000: 512 32.3 / 28.8, 1024 54.8 / 51.5: long and short rows mixed lose
      by whole rows, equal ones gain).
    * Otherwise two workgroups per CU (four at head dim 64, whose chunks are half
      as large: 8 rows of up to 2999, 16 KV heads, w = 1 / 2 / 4 16.9 / 15.7 /
      15.5), of at least 128 tokens of 128 dims, half of that in tables of
      at most 512 tokens.  The better one hangs on the lengths, which the table only bounds (64 /
      128 tokens, 2 KV heads: one row of 505 6.9 / 7.4, of 1000 7.3 / 7.5, of 2000 7.3 / 8.0, of
      4000 8.8 / 8.0; 8 KV heads: one row of 4000 10.6 / 8.7, 4 rows of 505 7.6 / 8.2, of 1000 9.4 /
      8.7, 8 rows of 505 9.1 / 8.7): a short row in a wide table takes 0.5 us more.
    * One per CU where the batch has no more rows than that and every workgroup
      gets a long stream, 16 chunks (2 per CU, 1, in turn: 32 rows of 32768 648, 637; of
      8192 169, 165; one of 32768 26.8, 25.9; 16 of 8000-16384 at D 256 143, 138;
      but 16 of up to 1024, 9 chunks each, 14.0, 14.4, and 64 of up to 2048, two rows
      each, 55.5, 58.4); 128 chunks at head dim 64 (32 rows of 30000-32768 323, 319; of
      8000-16384 131, 130).
    """
    units = HKV * -(-G // (16 if G <= 16 else 32))
    if B > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows, got {B}")
    if piece_tokens is not None:
        if piece_tokens <= 0:
            raise ValueError(f"piece_tokens must be positive, got {piece_tokens}")
        least = min(-(-piece_tokens // 32), 1 << 26)  # more than any table holds
        if S <= 32 * least:
            return least, 0, 0, 0
        most = -(-B * -(-S // 32) // least)  # where every row fills its table
        if most > MAX_WORKGROUPS:
            raise ValueError(f"piece_tokens={piece_tokens} cuts {B} rows of up to {S} tokens into "
                             f"more than {MAX_WORKGROUPS} pieces")
        return least, most, 0, 0
    row = S * D
    if row <= 32768 * (4 if B * units >= 512 else 2 if B * units * D >= 16384 else 1):
        return 1, 0, 0, 0
    least = (256 if S <= 512 else 512) // D or 1
    cu = compute_units(device) or 256
    groups = min(max(1, (4 if D == 64 else 2) * cu // units), -(-B * -(-S // 32) // least), MAX_WORKGROUPS)
    return least, groups, min(groups, max(1, cu // units)), 128 if D == 64 else 16


def _buffer(ws: dict, name: str, n: int, dtype, device) -> torch.Tensor:
    """A workspace buffer of at least n entries.  One that was handed out is never
    dropped, since a captured graph may hold its address; sizes are powers of two, so
    that those of a varying batch come to twice the largest at most."""
    n = 1 << max(0, n - 1).bit_length()
    key = (name, n, device)
    t = ws.get(key)
    if t is None:
        t = ws[key] = torch.empty(n, dtype=dtype, device=device)
    return t


class _Prepared16(_PreparedCall):
    """A checked call of this module or of ``pages``, kept as a decode's is.  Here
    every tensor may be another one of the same form, so that one workspace serves
    all layers of a model."""

    __slots__ = ()

    def run(self, *tensors) -> bool:
        rc = _lib.host().run(self.call, *tensors)
        if rc is None:
            return False
        if rc:
            _lib.check(rc, self.what)
        return True


def _keep16(ws, key, args, entry, what, device, buffers, slots):
    if ws is None or _lib.host() is None:
        return
    call = _lib.host().prepare(bytes(args), _lib.address(entry), device.index, slots, None)
    if call is not None:
        ws["call"] = _Prepared16(key, call, what, None, device, buffers)


def _offset(struct, field: str) -> int:
    return getattr(struct, field).offset


_D = {f: _offset(_lib.Paged16Args, f) for f in ("q", "k", "v", "block_table", "seq_lens", "out", "lse", "k_new",
                                                "v_new")}
_A = {f: _offset(_lib.Paged16AppendArgs, f) for f in ("k", "v", "k_new", "v_new", "block_table", "positions",
                                                      "counts")}


def _new_rows(x: torch.Tensor) -> torch.Tensor:
    """New tokens as the kernel reads them: rows on 16 bytes."""
    return x if _dense_rows(x, 16 // x.element_size()) else x.contiguous().clone()


def paged16_append(k_pool: torch.Tensor, v_pool: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                   block_table: torch.Tensor, positions: torch.Tensor,
                   counts: torch.Tensor | None = None, _workspace: dict | None = None) -> None:
    """K and V of new tokens ``(B, HKV, N, D)`` into 16-bit page pools, in one launch.

    Row b's first ``counts[b]`` tokens (None: all N) take logical positions
    ``positions[b]``, ``positions[b] + 1``, ... and land in the pages the block
    table names, rounded to the pools' type (nearest even).  ``k_new`` and
    ``v_new`` are float16, bfloat16 or float32 in any strides; a token-major
    ``(B, N, HKV, D).transpose(1, 2)`` is read as it lies.  Positions outside
    ``[0, block_table.shape[1] * page_size)`` and table entries outside ``[0,
    num_pages)`` are not written.  Two tokens for one place leave either.
    Allocates nothing where the tensors are used as they lie, and does not
    synchronise.
    """
    key = None
    if _workspace is not None:
        key = ("append16",)
        prep = _prepared(_workspace, key)
        if prep is not None and prep.run(k_pool, v_pool, k_new, v_new, block_table, positions, counts):
            return
    num_pages, HKV, page_size, D = _check_pools16(k_pool, v_pool)
    device = k_pool.device
    for name, x in (("k_new", k_new), ("v_new", v_new)):
        if not isinstance(x, torch.Tensor) or x.dim() != 4 or (x.shape[1], x.shape[3]) != (HKV, D):
            raise ValueError(f"{name} must be a (B, {HKV}, N, {D}) tensor")
        if x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise TypeError(f"{name} must be float16, bfloat16 or float32, got {x.dtype}")
        if x.device != device:
            raise ValueError(f"{name} is on {x.device}, the pools on {device}")
    if k_new.shape != v_new.shape or k_new.dtype != v_new.dtype:
        raise ValueError("k_new and v_new must have the same shape and dtype")
    B, _, N, _ = k_new.shape
    if B > MAX_ROWS or N * HKV * D // 8 > 2 ** 31 - 1:
        raise ValueError(f"k_new and v_new: at most {MAX_ROWS} rows of 2**34 values, got {tuple(k_new.shape)}")
    table = _check_table(block_table, B, device)
    pos = _int32_arg(positions, B, device, "positions", "B start positions")
    num = None if counts is None else _int32_arg(counts, B, device, "counts", "B token counts")
    _require_gpu(k_pool, "paged16_append")
    if B == 0 or N == 0:
        return
    kn, vn = _new_rows(k_new), _new_rows(v_new)
    align = 16 // kn.element_size()
    kind = 0 if kn.dtype == k_pool.dtype else 1 if kn.dtype == torch.float32 else 2
    args = _lib.Paged16AppendArgs(
        k_new=kn.data_ptr(), v_new=vn.data_ptr(), k_new_strides=_strides(kn, align),
        v_new_strides=_strides(vn, align), k=k_pool.data_ptr(), v=v_pool.data_ptr(),
        k_strides=_strides(k_pool, 8), v_strides=_strides(v_pool, 8), block_table=table.data_ptr(),
        positions=pos.data_ptr(), counts=_lib.ptr(num), new_is_fp32=kind,
        is_bf16=int(k_pool.dtype == torch.bfloat16), B=B, HKV=HKV, N=N, D=D,
        block_table_stride=table.shape[1], max_pages=table.shape[1], page_size=page_size,
        num_pages=num_pages)
    _lib.check(_lib.launch(device, "tkv_paged16_append", args), "paged16_append")
    if key is not None and kn is k_new and vn is v_new:
        _keep16(_workspace, key, args, "tkv_paged16_append", "paged16_append", device, (),
                ((k_pool, _A["k"], 16, 1), (v_pool, _A["v"], 16, 1), (k_new, _A["k_new"], 16, 1),
                 (v_new, _A["v_new"], 16, 1), (block_table, _A["block_table"], 4), (positions, _A["positions"], 4),
                 (counts, _A["counts"], 4)))


def paged16_decode_attention(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor | None = None,
    sm_scale: float | None = None,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    _workspace: dict | None = None,
    *,
    k_new: torch.Tensor | None = None,
    v_new: torch.Tensor | None = None,
    piece_tokens: int | None = None,
) -> torch.Tensor:
    """One decode step of attention over 16-bit page pools.

    q: ``(B, HQ, D)`` in the pools' type, D 64, 128 or 256; pools as
    :func:`empty_paged16_pool`; block_table: ``(B, max_pages)`` int32;
    seq_lens: ``(B,)`` int32 (None: every row holds ``max_pages * page_size``
    tokens; lengths past that are clamped to it).  Returns ``(B, HQ, D)`` float32, in
    ``out`` if it is given.  A row of no tokens gives zeros.  ``lse``: a contiguous ``(B, HQ)`` float32 tensor
    that receives the natural logarithm of each row's sum of exp(score), -inf
    for a row of no tokens, so that the results over two caches can be joined.
    Nothing past a row's length reaches them, NaN and infinities included; those
    of live tokens show as in softmax (a weight below 2**-126 of the largest counts as 0,
    and 0 times infinity is NaN).

    ``k_new`` / ``v_new``, ``(B, HKV, D)`` or ``(B, HKV, 1, D)`` in the pools'
    type, fuse the step's append into the call: the token takes position
    ``seq_lens[b] - 1`` of its row, in the page (unless the table entry lies
    outside the pool) and in the attention.  A row of no tokens takes none, nor does one
    whose length is past its table, as in :func:`paged16_append`.

    ``piece_tokens`` fixes how many tokens a workgroup takes of a row; by
    default the device chooses, from the lengths.  With ``_workspace`` the
    call allocates nothing but a missing ``out`` and keeps its checked form: a
    call like the previous one, on any tensors of the same shapes, strides and
    dtypes (every layer's pools), is checked and launched natively.  Calls that
    may overlap in time must not share a workspace.
    """
    key = None
    if _workspace is not None:
        key = ("paged16", sm_scale, piece_tokens)
        prep = _prepared(_workspace, key)
        if prep is not None:
            res = out if out is not None or not isinstance(q, torch.Tensor) else \
                torch.empty(q.shape, dtype=torch.float32, device=q.device)
            if prep.run(q, k_pool, v_pool, block_table, seq_lens, res, lse, k_new, v_new):
                return res
    num_pages, HKV, page_size, D = _check_pools16(k_pool, v_pool)
    device = k_pool.device
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.shape[2] != D:
        raise ValueError(f"q must be a (B, HQ, {D}) tensor")
    if q.dtype != k_pool.dtype:
        raise TypeError(f"q must have the pools' dtype {k_pool.dtype}, got {q.dtype}")
    if q.device != device:
        raise ValueError("q and the pools must be on the same device")
    B, HQ, _ = q.shape
    if B == 0 or HQ == 0 or HQ % HKV:
        raise ValueError(f"q of {B} rows and HQ={HQ}: HQ must be a multiple of HKV={HKV}, and neither zero")
    table = _check_table(block_table, B, device)
    S = table.shape[1] * page_size
    lens = None if seq_lens is None else _int32_arg(seq_lens, B, device, "seq_lens", "B lengths")
    if lse is not None and (not isinstance(lse, torch.Tensor) or lse.shape != (B, HQ) or lse.dtype != torch.float32
                            or not lse.is_contiguous() or lse.device != device):
        raise ValueError(f"lse must be a contiguous float32 ({B}, {HQ}) tensor on {device}")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new must be given together")
    new = [None, None]
    if k_new is not None:
        for i, (name, x) in enumerate((("k_new", k_new), ("v_new", v_new))):
            x = x[:, :, 0] if x.dim() == 4 and x.shape[2] == 1 else x
            if tuple(x.shape) != (B, HKV, D):
                raise ValueError(f"{name} must have shape ({B}, {HKV}, {D}) or ({B}, {HKV}, 1, {D}), "
                                 f"got {tuple(x.shape)}")
            if x.dtype != k_pool.dtype:
                raise TypeError(f"{name} must have the pools' dtype {k_pool.dtype}, got {x.dtype}")
            if x.device != device:
                raise ValueError(f"{name} must be on the pools' device")
            new[i] = x if _dense_rows(x, 8) else x.contiguous().clone()
    out = _check_out(out, B, HQ, D, device)
    if out.data_ptr() % 16:
        raise ValueError("out must start on a 16-byte boundary")
    G = HQ // HKV
    least, groups, few, long = plan_shares(B, HKV, G, S, D, device, piece_tokens)
    ok, why = _backend(q)
    if not ok:
        raise RuntimeError(f"paged16_decode_attention requires the tritonkv_amd HIP backend: {why}")
    qk = q if _dense_rows(q, 8) else q.contiguous().clone()
    partials = rows = None
    if groups:
        ws = {} if _workspace is None else _workspace
        partials = _buffer(ws, "partials16", 2 * groups * HQ * (D + 2), torch.float32, device)
        rows = _buffer(ws, "row_pieces16", 2 * B, torch.int32, device)
    kn, vn = new
    args = _lib.Paged16Args(
        q=qk.data_ptr(), q_strides=_strides(qk, 8), k=k_pool.data_ptr(), v=v_pool.data_ptr(),
        k_strides=_strides(k_pool, 8), v_strides=_strides(v_pool, 8), block_table=table.data_ptr(),
        seq_lens=_lib.ptr(lens), out=out.data_ptr(), lse=_lib.ptr(lse), partials=_lib.ptr(partials),
        row_pieces=_lib.ptr(rows), k_new=_lib.ptr(kn), v_new=_lib.ptr(vn),
        k_new_strides=_strides(kn, 8) if kn is not None else (0, 0),
        v_new_strides=_strides(vn, 8) if vn is not None else (0, 0),
        is_bf16=int(k_pool.dtype == torch.bfloat16), B=B, HQ=HQ, HKV=HKV, D=D,
        block_table_stride=table.shape[1], max_pages=table.shape[1], page_size=page_size,
        num_pages=num_pages,
        sm_scale=1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale),
        least_chunks=least, workgroups=groups, long_workgroups=few, long_chunks=long)
    _lib.check(_lib.launch(device, "tkv_paged16_decode_attention", args), "paged16_decode_attention")
    if key is not None and qk is q:
        strided = (k_new is None or kn.data_ptr() == k_new.data_ptr()) and \
            (v_new is None or vn.data_ptr() == v_new.data_ptr())
        if strided:  # nothing was copied: every tensor is read where it lies
            _keep16(_workspace, key, args, "tkv_paged16_decode_attention", "paged16_decode_attention",
                    device, (partials, rows),
                    ((q, _D["q"], 16, 1), (k_pool, _D["k"], 16, 1), (v_pool, _D["v"], 16, 1),
                     (block_table, _D["block_table"], 4), (seq_lens, _D["seq_lens"], 4), (out, _D["out"], 16), (lse, _D["lse"], 4),
                     (k_new, _D["k_new"], 16, 1), (v_new, _D["v_new"], 16, 1)))
    return out


__all__ = ["PAGE_MULTIPLE", "HEAD_DIMS", "empty_paged16_pool", "paged16_append",
           "paged16_decode_attention", "plan_shares"]
