"""8-bit paged KV cache: a scale for each block of tokens and head.

Between the 2- and 4-bit pages of :mod:`tritonkv_amd.paged` and the 16-bit ones of
:mod:`tritonkv_amd.paged16`.  A :class:`Paged8Pool` is

    codes  (num_pages, HKV, page_size, D)          float8_e4m3fn or int8
    scale  (num_pages, HKV, page_size // block)    float32

and slot t of a page stands for ``codes[..., t, :] * scale[..., t // block]``.  A block
is 32, 64 or 128 tokens; ``page_size`` is a multiple of it.  Logical token t of batch
row b lives in page ``block_table[b, t // page_size]`` at slot ``t % page_size``, as in the
other paged caches, and :mod:`tritonkv_amd.pages` forks, truncates, frees and compacts
these pools too.

:func:`paged8_append` quantizes tokens as they are written (with rotary positions on the
way, if asked), :func:`paged8_decode_attention` attends to them, for one new token
of every row or for its last few (the tokens of a draft), :func:`paged8_read` gives them back as
values.

How a block gets its scale: the append gives it the least power of two under which its new
values fit the codes (448, or 127), 2**-64 at least.  Tokens that come later keep the block's
scale while they fit; where one does not, the scale rises and the codes of the block's earlier
tokens are rounded again under it -- by a power of two, which leaves e4m3 codes exact unless they
fall among its smallest.  An append that writes a block's first slot starts the block anew.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib
from .kernels.fused_decode_attn import _backend, _prepared, compute_units
from .paged import _check_table
from .paged16 import (HEAD_DIMS, MAX_ROWS, MAX_WORKGROUPS, _buffer, _dense_rows, _int32_arg, _keep16, _new_rows, _offset, _strides,
                      plan_shares)
from .quantize import _require_gpu
from .rotary import _APART, _WRITTEN, DTYPES, MAX_TOKENS, Rotary, _apart, _check_rotary, _no_grad, _same_place

CODES = (torch.float8_e4m3fn, torch.int8)
BLOCKS = (32, 64, 128)
MAX_QUERIES = 32
ROTARY_MULTIPLE = 16
MAX_PAGE_SIZE = 2 ** 24


def plan_shares8(B: int, HKV: int, columns: int, S: int, D: int, device=None,
                 piece_tokens: int | None = None) -> tuple[int, int, int, int]:
    """:func:`~tritonkv_amd.paged16.plan_shares` for 8-bit pages, whose chunks hold half the bytes;
    ``columns`` are a KV head's queries.  Measured on MI355X (us, each pair in one session; U = HKV times the
    blocks of 16 or 32 columns):

    * Rows stay whole up to 512 tokens of 128 dims, 256 of 256 and 512 of 64 (whole / cut, one row, steps of
      a graph: 507 of 128 7.8 / 8.0, 1019 10.9 / 8.1; 251 of 256 8.9 / 9.9, 507 11.8 / 9.8; 1019 of 64 8.3 /
      8.1; 16 rows of 1-507, 8 KV heads, 9.4 / 12.8), and where B * U is 512 or more, twice or four times that
      (64 rows of 1-1019, 8 KV heads, 21.9 / 24.1, all 1019 27.8 / 32.1; of 64 dims 13.6 / 16.5 and 15.7 /
      19.0; 507 of 256 29.1 / 33.0; but 1-2043 of 128 38.6 / 36.9).
    * Otherwise two workgroups per CU, four of 64 dims and one of 256 with more than 16 columns (1 / 2 /
      3 / 4: 32 rows of 32768 422 / 353 / 362 / 361, of 8000-16384 with 64 dims 105 / 71 / 71 / 71, 8 of 1-2999
      with 64 dims, 16 KV heads, 16.7 / 15.4 / 14.9 / 15.1; 16 rows of 4 queries and 64 heads 58 / 49 / 63 / 60;
      one row of 32768 21.4 / 19.5 / 20.9 / 22.6; 32 of 16384 with 256 dims 372 / 349 / 360, one with 24
      columns 29 / 41 / 55), of at least 128 tokens of 128 dims, half of that in tables of at most 512
      tokens (64 / 128 / 256: 16 rows of 1-1000 13.6 / 13.9 / 15.0).
    """
    if piece_tokens is not None:
        return plan_shares(B, HKV, columns, S, D, device, piece_tokens)
    if B > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows, got {B}")
    units = HKV * -(-columns // (16 if columns <= 16 else 32))
    if S * D <= (131072 if B * units >= 512 else 32768 if D == 64 else 65536):
        return 1, 0, 0, 0
    least = (256 if S <= 512 else 512) // D or 1
    per_cu = 4 if D == 64 else 1 if D == 256 and columns > 16 else 2
    cu = compute_units(device) or 256
    return least, min(max(1, per_cu * cu // units), -(-B * -(-S // 32) // least), MAX_WORKGROUPS), 0, 0


@dataclass(frozen=True, eq=False)
class Paged8Pool:
    """Codes of a page pool and their scales (see the module).

    Both are used as they are strided, as long as a token's D codes are dense and start on 16
    bytes.  For :mod:`tritonkv_amd.pages`, scales of a page must start on 16 bytes too, with room up to
    the next 16, as :func:`empty_paged8_pool` lays them out."""

    codes: torch.Tensor
    scale: torch.Tensor

    @property
    def block(self) -> int:
        """Tokens that share a scale."""
        return self.codes.shape[2] // self.scale.shape[2]

    @property
    def page_size(self) -> int:
        return self.codes.shape[2]

    def page_tensors(self) -> list:
        """The pool as tensors of whole pages, ``(num_pages, ...)`` of 16-byte multiples: the
        codes, and the scales with the room after them."""
        pages, n = self.scale.shape[0], self.scale[0].numel()
        room = -(-n // 4) * 4
        if not self.scale[0].is_contiguous() or (pages > 1 and self.scale.stride(0) < room):
            raise ValueError("the pages of a pool's scales must be dense, with room up to a multiple of 16 bytes "
                             "(empty_paged8_pool makes them so)")
        stride = self.scale.stride(0) if pages > 1 else room
        try:
            return [self.codes, self.scale.as_strided((pages, 1, 1, room), (stride, room, room, 1))]
        except RuntimeError as exc:  # no room after the last page
            raise ValueError("the pages of a pool's scales must have room up to a multiple of 16 bytes "
                             "(empty_paged8_pool makes them so)") from exc


def empty_paged8_pool(num_pages: int, HKV: int, page_size: int, D: int, dtype: torch.dtype = torch.float8_e4m3fn,
                      block: int = 32, device="cuda") -> Paged8Pool:
    """A pool of ``num_pages`` pages of ``page_size`` tokens; its codes are uninitialised, its scales 0."""
    if block not in BLOCKS:
        raise ValueError(f"block must be one of {BLOCKS}, got {block}")
    if page_size <= 0 or page_size % block or page_size > MAX_PAGE_SIZE:
        raise ValueError(f"page_size must be a positive multiple of block={block}, at most {MAX_PAGE_SIZE}, got {page_size}")
    if num_pages <= 0 or HKV <= 0:
        raise ValueError(f"num_pages and HKV must be positive, got {num_pages} and {HKV}")
    if D not in HEAD_DIMS:
        raise ValueError(f"D must be one of {HEAD_DIMS}, got {D}")
    if dtype not in CODES:
        raise TypeError(f"dtype must be float8_e4m3fn or int8, got {dtype}")
    n = HKV * (page_size // block)
    scale = torch.zeros(num_pages, -(-n // 4) * 4, dtype=torch.float32, device=device)
    return Paged8Pool(torch.empty(num_pages, HKV, page_size, D, dtype=dtype, device=device),
                      scale[:, :n].view(num_pages, HKV, page_size // block))


def _check_pools8(k_pool, v_pool) -> tuple:
    for name, pool in (("k_pool", k_pool), ("v_pool", v_pool)):
        if not isinstance(pool, Paged8Pool):
            raise TypeError(f"{name} must be a Paged8Pool, got {type(pool).__name__}")
        codes, scale = pool.codes, pool.scale
        if not isinstance(codes, torch.Tensor) or codes.dim() != 4 or codes.numel() == 0:
            raise ValueError(f"{name}.codes must be a (num_pages, HKV, page_size, D) tensor")
        if codes.dtype not in CODES:
            raise TypeError(f"{name}.codes must be float8_e4m3fn or int8, got {codes.dtype}")
        if not _dense_rows(codes, 16) or any(s <= 0 for s in _strides(codes, 16)):
            raise ValueError(f"{name}.codes must hold each token's D codes densely, on 16-byte boundaries")
        if not isinstance(scale, torch.Tensor) or scale.dim() != 3 or scale.dtype != torch.float32 \
                or scale.shape[:2] != codes.shape[:2] or scale.numel() == 0 or scale.device != codes.device:
            raise ValueError(f"{name}.scale must be a float32 (num_pages, HKV, page_size // block) tensor on the "
                             "codes' device")
        if codes.shape[2] % scale.shape[2] or pool.block not in BLOCKS:
            raise ValueError(f"{name}: a page of {codes.shape[2]} tokens and {scale.shape[2]} scales: a block must be one "
                             f"of {BLOCKS} tokens")
        if any(s <= 0 for s, n in zip(scale.stride(), scale.shape) if n > 1):
            raise ValueError(f"{name}.scale must hold a value of its own for every block")
    if v_pool.codes.shape != k_pool.codes.shape or v_pool.codes.dtype != k_pool.codes.dtype \
            or v_pool.codes.device != k_pool.codes.device or v_pool.scale.shape != k_pool.scale.shape:
        raise ValueError("K and V pools must have the same shapes, dtype and device")
    num_pages, HKV, page_size, D = k_pool.codes.shape
    if D not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {D}")
    if page_size > MAX_PAGE_SIZE or num_pages > 2 ** 31 - 1:
        raise ValueError(f"pages of at most {MAX_PAGE_SIZE} tokens, at most 2**31 - 1 of them")
    return num_pages, HKV, page_size, D


def _pool_fields(k_pool: Paged8Pool, v_pool: Paged8Pool) -> dict:
    """A call's fields that describe the pools."""
    return dict(k=k_pool.codes.data_ptr(), v=v_pool.codes.data_ptr(), k_strides=_strides(k_pool.codes, 16),
                v_strides=_strides(v_pool.codes, 16), k_scale=k_pool.scale.data_ptr(),
                v_scale=v_pool.scale.data_ptr(), k_scale_strides=k_pool.scale.stride(),
                v_scale_strides=v_pool.scale.stride(), is_int8=int(k_pool.codes.dtype == torch.int8),
                block=k_pool.block, page_size=k_pool.page_size, num_pages=k_pool.codes.shape[0])


def _pool_slots(offsets: dict, k_pool: Paged8Pool, v_pool: Paged8Pool, flags: int = 0) -> tuple:
    return ((k_pool.codes, offsets["k"], 16, 1 | flags), (k_pool.scale, offsets["k_scale"], 4, 1 | flags),
            (v_pool.codes, offsets["v"], 16, 1 | flags), (v_pool.scale, offsets["v_scale"], 4, 1 | flags))


def _pool_tensors(k_pool, v_pool) -> tuple:
    return k_pool.codes, k_pool.scale, v_pool.codes, v_pool.scale


_POOL = ("k", "k_scale", "v", "v_scale")
_D = {f: _offset(_lib.Paged8Args, f) for f in (*_POOL, "q", "block_table", "seq_lens", "counts", "out", "lse")}
_A = {f: _offset(_lib.Paged8AppendArgs, f) for f in (*_POOL, "k_new", "v_new", "block_table", "positions", "counts",
                                                     "turns", "q", "q_out")}
_R = {f: _offset(_lib.Paged8ReadArgs, f) for f in (*_POOL, "k_out", "v_out", "block_table", "positions", "counts")}


def _both_pools(k_pool, v_pool) -> bool:
    return isinstance(k_pool, Paged8Pool) and isinstance(v_pool, Paged8Pool)


def paged8_append(k_pool: Paged8Pool, v_pool: Paged8Pool, k_new: torch.Tensor, v_new: torch.Tensor,
                  block_table: torch.Tensor, positions: torch.Tensor, counts: torch.Tensor | None = None,
                  _workspace: dict | None = None, *, rotary: Rotary | None = None, q: torch.Tensor | None = None,
                  q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Quantize K and V of new tokens ``(B, HKV, N, D)`` into 8-bit page pools.

    Row b's first ``counts[b]`` tokens (None: all N) take logical positions ``positions[b]``,
    ``positions[b] + 1``, ... in the pages the block table names.  ``k_new`` and ``v_new``
    are float16, bfloat16 or float32 in any strides; a token-major ``(B, N, HKV,
    D).transpose(1, 2)`` is read as it lies.  Positions outside ``[0, block_table.shape[1] *
    page_size)`` and table entries outside ``[0, num_pages)`` are not written.  Two tokens for
    one place leave either, and rows that write into one block leave it with the codes of
    both under the scale of either: give every row pages of its own to write into, as
    :mod:`tritonkv_amd.pages` does.

    How blocks get their scales stands in the module's documentation.  Codes behind the new tokens in
    their last block are left as they are, under the scale that it then has: what is written over is written
    over up to the row's end.  Magnitudes above 2**64,
    infinities among them, count as 2**64.  NaN does not count for a scale; e4m3 keeps it, int8
    stores 0.

    ``rotary`` turns the keys to their positions on the way (in 32 bits: they are rounded
    once, to codes); it must turn a multiple of 16 values of a head.  With it, ``q`` ``(B, HQ, N, D)``
    in k_new's type, the same tokens' queries, are turned too, into ``q_out`` (None: a new
    tensor; it may be q), which is returned.  Rows of ``q_out`` past a row's count are left as they
    were (zero in a new one).

    Does not synchronise, and with ``q_out`` allocates nothing where the tensors are used as they lie.
    """
    _no_grad(k_new, v_new, q)
    key = None
    if _workspace is not None and (q is None or q_out is not None) and _both_pools(k_pool, v_pool) \
            and (rotary is None or isinstance(rotary, Rotary)):
        key = ("append8",) if rotary is None else ("append8", rotary.factor, rotary.interleaved, q_out is q)
        prep = _prepared(_workspace, key)
        if prep is not None and prep.run(*_pool_tensors(k_pool, v_pool), k_new, v_new, block_table, positions, counts,
                                         None if rotary is None else rotary.turns, q, q_out):
            return q_out
    num_pages, HKV, page_size, D = _check_pools8(k_pool, v_pool)
    device = k_pool.codes.device
    for name, x in (("k_new", k_new), ("v_new", v_new)):
        if not isinstance(x, torch.Tensor) or x.dim() != 4 or (x.shape[1], x.shape[3]) != (HKV, D):
            raise ValueError(f"{name} must be a (B, {HKV}, N, {D}) tensor")
        if x.dtype not in DTYPES:
            raise TypeError(f"{name} must be float16, bfloat16 or float32, got {x.dtype}")
        if x.device != device:
            raise ValueError(f"{name} is on {x.device}, the pools on {device}")
    if k_new.shape != v_new.shape or k_new.dtype != v_new.dtype:
        raise ValueError("k_new and v_new must have the same shape and dtype")
    B, _, N, _ = k_new.shape
    if B > MAX_ROWS or N * HKV * D > 2 ** 33:
        raise ValueError(f"k_new and v_new: at most {MAX_ROWS} rows of 2**33 values, got {tuple(k_new.shape)}")
    table = _check_table(block_table, B, device)
    if table.shape[1] * page_size > 2 ** 32 - 1:
        raise ValueError(f"{table.shape[1]} pages of {page_size} tokens a row: at most 2**32 - 1 tokens")
    pos = _int32_arg(positions, B, device, "positions", "B start positions")
    num = None if counts is None else _int32_arg(counts, B, device, "counts", "B token counts")
    align = 16 // k_new.element_size()
    if rotary is None:
        if q is not None or q_out is not None:
            raise ValueError("q and q_out are for rotary")
    else:
        _check_rotary(rotary, D, device)
        if rotary.dims % ROTARY_MULTIPLE:
            raise ValueError(f"rotary must turn a multiple of {ROTARY_MULTIPLE} values of a head here, got {rotary.dims}: "
                             "use apply_rotary")
        if q is None and q_out is not None:
            raise ValueError("q_out without q")
    if q is not None:
        if not isinstance(q, torch.Tensor) or q.dim() != 4 or (q.shape[0], q.shape[2], q.shape[3]) != (B, N, D) \
                or not 0 < q.shape[1] <= 65535 or N > MAX_TOKENS:
            raise ValueError(f"q must be a ({B}, HQ, {N}, {D}) tensor of at most {MAX_TOKENS} tokens a row")
        if q.dtype != k_new.dtype or q.device != device:
            raise ValueError(f"q must be {k_new.dtype} on {device}, got {q.dtype} on {q.device}")
        if q_out is not None:
            if not isinstance(q_out, torch.Tensor) or q_out.shape != q.shape or q_out.dtype != q.dtype \
                    or q_out.device != device or not _dense_rows(q_out, align) \
                    or any(s <= 0 for s in _strides(q_out, align)):
                raise ValueError("q_out must be a tensor of q's shape, dtype and device with dense rows on 16 bytes")
            others = [t for t in (k_new, v_new, table, pos, num, rotary.turns) if t is not None]
            if not (_same_place(q, q_out) or _apart(q, q_out)) or \
                    not all(_apart(q_out, t) for t in (*others, *_pool_tensors(k_pool, v_pool))):
                raise ValueError("q_out must be q itself or share no memory with the other tensors")
    _require_gpu(k_pool.codes, "paged8_append")
    if q is not None and q_out is None:
        fresh = torch.zeros if counts is not None else torch.empty
        q_out = fresh(q.shape, dtype=q.dtype, device=device)
    if B == 0 or N == 0:
        return q_out
    kn, vn, qn = _new_rows(k_new), _new_rows(v_new), None if q is None else _new_rows(q)
    args = _lib.Paged8AppendArgs(
        **_pool_fields(k_pool, v_pool), k_new=kn.data_ptr(), v_new=vn.data_ptr(), k_new_strides=_strides(kn, align),
        v_new_strides=_strides(vn, align), block_table=table.data_ptr(), positions=pos.data_ptr(), counts=_lib.ptr(num),
        turns=None if rotary is None else rotary.turns.data_ptr(), q=_lib.ptr(qn), q_out=_lib.ptr(q_out),
        q_strides=(0, 0, 0) if qn is None else _strides(qn, align),
        q_out_strides=(0, 0, 0) if q_out is None else _strides(q_out, align),
        factor=1.0 if rotary is None else rotary.factor, interleaved=int(rotary is not None and rotary.interleaved),
        dims=0 if rotary is None else rotary.dims, HQ=0 if q is None else q.shape[1], x_type=DTYPES.index(kn.dtype),
        B=B, HKV=HKV, N=N, D=D, block_table_stride=table.shape[1], max_pages=table.shape[1])
    _lib.check(_lib.launch(device, "tkv_paged8_append", args), "paged8_append")
    if key is not None and kn is k_new and vn is v_new and qn is q:
        # In place q is what is written, as q_out, the same tensor, which need not lie apart from it.
        read, written = (_WRITTEN, 0) if q_out is q else (_APART, _WRITTEN)
        _keep16(_workspace, key, args, "tkv_paged8_append", "paged8_append", device, (),
                (*_pool_slots(_A, k_pool, v_pool, _APART), (k_new, _A["k_new"], 16, 1 | _APART),
                 (v_new, _A["v_new"], 16, 1 | _APART), (block_table, _A["block_table"], 4, _APART),
                 (positions, _A["positions"], 4, _APART), (counts, _A["counts"], 4, _APART),
                 (None if rotary is None else rotary.turns, _A["turns"], 8, _APART), (q, _A["q"], 16, 1 | read),
                 (q_out, _A["q_out"], 16, 1 | written)))
    return q_out


def paged8_read(k_pool: Paged8Pool, v_pool: Paged8Pool, block_table: torch.Tensor,
                positions: torch.Tensor | None = None, counts: torch.Tensor | None = None, tokens: int | None = None,
                dtype: torch.dtype = torch.bfloat16, out=None, _workspace: dict | None = None) -> tuple:
    """Tokens of 8-bit pages as values: ``(k, v)``, each ``(B, HKV, tokens, D)``.

    Row b's are the ``counts[b]`` tokens (None: all of ``tokens``) from ``positions[b]`` on
    (None: 0), code times scale in 32 bits, rounded to ``dtype`` (float16, bfloat16 or float32): once, where
    the scale is a power of two, as the append's are.
    ``out``: a pair of tensors for them, in any strides with dense rows (``tokens`` and ``dtype``
    are then theirs).  Rows past a row's count, and tokens outside the table or in entries outside
    the pool, are left as they were; in new tensors they are zero.
    """
    key = None
    if _workspace is not None and isinstance(out, (tuple, list)) and len(out) == 2 and _both_pools(k_pool, v_pool):
        key = ("read8", tokens)
        prep = _prepared(_workspace, key)
        if prep is not None and prep.run(*_pool_tensors(k_pool, v_pool), block_table, positions, counts, *out):
            return out[0], out[1]
    num_pages, HKV, page_size, D = _check_pools8(k_pool, v_pool)
    device = k_pool.codes.device
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError("block_table must be an int32 (B, max_pages) tensor on the pool's device")
    B = block_table.shape[0]
    if out is None:
        if tokens is None or tokens < 0:
            raise ValueError(f"tokens must say how many to read, got {tokens}")
        if dtype not in DTYPES:
            raise TypeError(f"dtype must be float16, bfloat16 or float32, got {dtype}")
        N = tokens
    else:
        if not isinstance(out, (tuple, list)) or len(out) != 2:
            raise ValueError("out must be a pair of tensors")
        for x in out:
            if not isinstance(x, torch.Tensor) or x.dim() != 4 or (x.shape[0], x.shape[1], x.shape[3]) != (B, HKV, D) \
                    or x.shape != out[0].shape or x.dtype != out[0].dtype or x.device != device:
                raise ValueError(f"out must be two ({B}, {HKV}, tokens, {D}) tensors of one shape and dtype on {device}")
            if x.dtype not in DTYPES:
                raise TypeError(f"out must be float16, bfloat16 or float32, got {x.dtype}")
            if not _dense_rows(x, 16 // x.element_size()) or any(s <= 0 for s in _strides(x, 1)):
                raise ValueError("out must hold each token's values densely, on 16-byte boundaries")
        N, dtype = out[0].shape[2], out[0].dtype
        if tokens is not None and tokens != N:
            raise ValueError(f"out has {N} tokens, not {tokens}")
    if B > MAX_ROWS or N * HKV * D > 2 ** 33:
        raise ValueError(f"at most {MAX_ROWS} rows of 2**33 values, got {B} of {N} tokens")
    table = _check_table(block_table, B, device)
    if table.shape[1] * page_size > 2 ** 32 - 1:
        raise ValueError(f"{table.shape[1]} pages of {page_size} tokens a row: at most 2**32 - 1 tokens")
    pos = None if positions is None else _int32_arg(positions, B, device, "positions", "B start positions")
    num = None if counts is None else _int32_arg(counts, B, device, "counts", "B token counts")
    if out is not None:
        others = [t for t in (table, pos, num, *_pool_tensors(k_pool, v_pool)) if t is not None]
        if not _apart(out[0], out[1]) or not all(_apart(x, t) for x in out for t in others):
            raise ValueError("out must not share memory with itself or the other tensors")
    _require_gpu(k_pool.codes, "paged8_read")
    if out is None:
        out = tuple(torch.zeros(B, HKV, N, D, dtype=dtype, device=device) for _ in range(2))
    if B == 0 or N == 0:
        return out[0], out[1]
    align = 16 // out[0].element_size()
    args = _lib.Paged8ReadArgs(
        **_pool_fields(k_pool, v_pool), k_out=out[0].data_ptr(), v_out=out[1].data_ptr(),
        k_out_strides=_strides(out[0], align), v_out_strides=_strides(out[1], align), block_table=table.data_ptr(),
        positions=_lib.ptr(pos), counts=_lib.ptr(num), x_type=DTYPES.index(dtype), B=B, HKV=HKV, N=N, D=D,
        block_table_stride=table.shape[1], max_pages=table.shape[1])
    _lib.check(_lib.launch(device, "tkv_paged8_read", args), "paged8_read")
    if key is not None:
        _keep16(_workspace, key, args, "tkv_paged8_read", "paged8_read", device, (),
                (*_pool_slots(_R, k_pool, v_pool, _APART), (block_table, _R["block_table"], 4, _APART),
                 (positions, _R["positions"], 4, _APART), (counts, _R["counts"], 4, _APART),
                 (out[0], _R["k_out"], 16, 1 | _WRITTEN), (out[1], _R["v_out"], 16, 1 | _WRITTEN)))
    return out[0], out[1]


def paged8_decode_attention(
    q: torch.Tensor,
    k_pool: Paged8Pool,
    v_pool: Paged8Pool,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor | None = None,
    sm_scale: float | None = None,
    out: torch.Tensor | None = None,
    lse: torch.Tensor | None = None,
    _workspace: dict | None = None,
    *,
    counts: torch.Tensor | None = None,
    piece_tokens: int | None = None,
) -> torch.Tensor:
    """Attention of every row's last tokens over 8-bit page pools.

    q: ``(B, HQ, D)`` for one token, or ``(B, HQ, M, D)`` for up to 32, float16 or bfloat16, D 64,
    128 or 256, in any strides; the tokens themselves are in the cache (:func:`paged8_append`
    comes before).  block_table: ``(B, max_pages)`` int32; seq_lens: ``(B,)`` int32, the rows'
    tokens with the new ones (None: every row holds ``max_pages * page_size``; lengths
    past that are clamped to it).  counts: ``(B,)`` int32, how many of row b's M queries there
    are (None: all), the others being padding: query m is the row's token ``seq_lens[b] -
    counts[b] + m`` and attends to itself and the tokens before it.

    Returns ``out``, float32 of q's shape; ``lse``, a contiguous float32 tensor of its shape without D,
    receives the natural logarithm of each sum of exp(score).  A query that attends to nothing,
    or that there is not, gives zeros and -inf.  Nothing past a query's token reaches its
    result, NaN included; those of the tokens it sees show as in softmax in 32 bits (a query
    whose scores pass 2**128 gives NaN; scores below -2**128 count as -inf).  Records no gradient: a
    query that requires grad is refused.

    ``piece_tokens`` and ``_workspace`` as in
    :func:`~tritonkv_amd.paged16.paged16_decode_attention`.
    """
    _no_grad(q)
    key = None
    if _workspace is not None and _both_pools(k_pool, v_pool):
        key = ("paged8", sm_scale, piece_tokens)
        prep = _prepared(_workspace, key)
        if prep is not None:
            res = out if out is not None or not isinstance(q, torch.Tensor) else \
                torch.empty(q.shape, dtype=torch.float32, device=q.device)
            if prep.run(q, *_pool_tensors(k_pool, v_pool), block_table, seq_lens, counts, res, lse):
                return res
    num_pages, HKV, page_size, D = _check_pools8(k_pool, v_pool)
    device = k_pool.codes.device
    if not isinstance(q, torch.Tensor) or q.dim() not in (3, 4) or q.shape[-1] != D:
        raise ValueError(f"q must be a (B, HQ, {D}) or (B, HQ, M, {D}) tensor")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q must be float16 or bfloat16, got {q.dtype}")
    if q.device != device:
        raise ValueError("q and the pools must be on the same device")
    B, HQ = q.shape[:2]
    M = 1 if q.dim() == 3 else q.shape[2]
    if B == 0 or HQ == 0 or HQ % HKV:
        raise ValueError(f"q of {B} rows and HQ={HQ}: HQ must be a multiple of HKV={HKV}, and neither zero")
    if not 0 < M <= MAX_QUERIES:
        raise ValueError(f"q must hold 1 to {MAX_QUERIES} tokens of a row, got {M}")
    table = _check_table(block_table, B, device)
    S = table.shape[1] * page_size
    lens = None if seq_lens is None else _int32_arg(seq_lens, B, device, "seq_lens", "B lengths")
    num = None if counts is None else _int32_arg(counts, B, device, "counts", "B query counts")
    for name, t, shape in (("out", out, q.shape), ("lse", lse, q.shape[:-1])):
        if t is not None and (not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype != torch.float32
                              or not t.is_contiguous() or t.device != device):
            raise ValueError(f"{name} must be a contiguous float32 {tuple(shape)} tensor on {device}")
    if out is not None and out.data_ptr() % 16:
        raise ValueError("out must start on a 16-byte boundary")
    least, groups, few, long = plan_shares8(B, HKV, HQ // HKV * M, S, D, device, piece_tokens)
    ok, why = _backend(q)
    if not ok:
        raise RuntimeError(f"paged8_decode_attention requires the tritonkv_amd HIP backend: {why}")
    if out is None:
        out = torch.empty(q.shape, dtype=torch.float32, device=device)
    qk = q if _dense_rows(q, 8) else q.contiguous().clone()
    partials = rows = None
    if groups:
        ws = {} if _workspace is None else _workspace
        partials = _buffer(ws, "partials8", 2 * groups * HQ * M * (D + 2), torch.float32, device)
        rows = _buffer(ws, "row_pieces8", 2 * B, torch.int32, device)
    strides = _strides(qk, 8)
    args = _lib.Paged8Args(
        **_pool_fields(k_pool, v_pool), q=qk.data_ptr(), q_strides=(*strides, 8) if q.dim() == 3 else strides,
        block_table=table.data_ptr(), seq_lens=_lib.ptr(lens), counts=_lib.ptr(num), out=out.data_ptr(),
        lse=_lib.ptr(lse), partials=_lib.ptr(partials), row_pieces=_lib.ptr(rows),
        q_is_bf16=int(q.dtype == torch.bfloat16), B=B, HQ=HQ, HKV=HKV, M=M, D=D, block_table_stride=table.shape[1],
        max_pages=table.shape[1], sm_scale=1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale),
        least_chunks=least, workgroups=groups, long_workgroups=few, long_chunks=long)
    _lib.check(_lib.launch(device, "tkv_paged8_decode_attention", args), "paged8_decode_attention")
    if key is not None and qk is q:
        _keep16(_workspace, key, args, "tkv_paged8_decode_attention", "paged8_decode_attention", device,
                (partials, rows),
                ((q, _D["q"], 16, 1), *_pool_slots(_D, k_pool, v_pool), (block_table, _D["block_table"], 4),
                 (seq_lens, _D["seq_lens"], 4), (counts, _D["counts"], 4), (out, _D["out"], 16), (lse, _D["lse"], 4)))
    return out


__all__ = ["BLOCKS", "CODES", "MAX_QUERIES", "Paged8Pool", "empty_paged8_pool", "paged8_append", "paged8_read",
           "paged8_decode_attention"]
