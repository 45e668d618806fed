"""The operators of 16-bit page pools, as cases to time and to compare.

Five operators: ``paged16_decode_attention`` (one new token over a paged fp16
or bf16 cache), ``paged16_append`` (tokens into such a cache), ``copy_pages``,
``fork_rows`` (rows forked, reordered, truncated, grown or freed over shared,
reference-counted pages) and ``compact_pages`` (live pages moved to the low end
of the pools).

A case is a dict with ``kind`` and the sizes of that kind.  ``run`` takes the
operators' plain form, in elementary torch operations and 32 bits, or (``own``)
the package's entry points.  Lengths, page counts and numbers of copies follow
from the case alone; the seed decides values, which row has which length and
which page is which.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
OUTLIERS, OUTLIER_SCALE = 4, 8.0  # channels per KV head that stand out, as in the benchmark's caches


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def _decode(B, HQ, HKV, D, page, cap, lo, hi, dtype, append):
    return dict(kind="decode", B=B, HQ=HQ, HKV=HKV, D=D, page=page, cap=cap, lo=lo, hi=hi, dtype=dtype,
                append=append)


def _append(B, N, HKV, D, page, dtype, x, counts, token_major):
    return dict(kind="append", B=B, N=N, HKV=HKV, D=D, page=page, dtype=dtype, x=x, counts=counts,
                token_major=token_major)


def _fork(groups, width, survivors, length, room, page, cap, layers, HKV, D):
    return dict(kind="fork", groups=groups, width=width, survivors=survivors, length=length, room=room,
                page=page, cap=cap, layers=layers, HKV=HKV, D=D)


def _compact(pages, live, moves, rows, page, layers, HKV, D):
    return dict(kind="compact", pages=pages, live=live, moves=moves, rows=rows, page=page, layers=layers,
                HKV=HKV, D=D)


def _copy(pages, pairs, other, page, layers, HKV, D):
    return dict(kind="copy", pages=pages, pairs=pairs, other=other, page=page, layers=layers, HKV=HKV, D=D)


def listed():
    return [
        # One sequence of the Qwen2.5-1.5B shape, a short chat: latency counts.
        dict(_decode(1, 12, 2, 128, 64, 512, 505, 505, "float16", False), name="decode_b1_short"),
        # A small batch of a model without shared KV heads, head dim 64, the
        # smallest pages, rows from a single token to 2999.
        dict(_decode(8, 16, 16, 64, 16, 4096, 1, 2999, "bfloat16", False), name="decode_mha_d64"),
        # A 70B-style continuous batch: lengths 1k to 16k in tables made for
        # twice that, every row's new token appended by the call.
        dict(_decode(32, 64, 8, 128, 64, 32768, 1000, 16384, "bfloat16", True), name="decode_70b_ragged"),
        # The benchmark's Llama-3-8B batch, 32 rows at 32k, as 16-bit pages.
        dict(_decode(32, 32, 8, 128, 256, 32768, 32768, 32768, "float16", False), name="decode_8b_large"),
        # The append of one decode step of a serving batch.
        dict(_append(64, 1, 8, 128, 64, "bfloat16", "bfloat16", False, False), name="append_step"),
        # Prompts as the projections leave them (token-major), padded to the
        # longest, each row's own count of tokens.
        dict(_append(4, 8213, 8, 128, 64, "float16", "float16", True, True), name="append_prompt"),
        # A beam-search step: 8 requests of 4 beams, half of the beams go on.
        dict(_fork(8, 4, 2, 1000, 0, 64, 2048, 2, 8, 128), name="fork_beams"),
        # Parallel sampling: 16 requests, 16 samples of each from one prompt,
        # with room for the next tokens.
        dict(_fork(16, 16, 1, 4003, 40, 16, 8192, 8, 8, 128), name="fork_samples"),
        # A small pool with a few stray pages.
        dict(_compact(1024, 700, 24, 64, 64, 1, 2, 128), name="compact_small"),
        # A large pool, a fifth of its live pages out of place.
        dict(_compact(16384, 10000, 2000, 64, 64, 1, 8, 128), name="compact_large"),
        # A handful of pages of one model.
        dict(_copy(512, 8, False, 64, 2, 8, 128), name="copy_few"),
        # Rows moved into another pool of pages (another server's share).
        dict(_copy(4096, 2000, True, 32, 2, 8, 128), name="copy_to_pool"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "append", "fork", "compact", "copy"])
    HKV, D = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 128, 128, 256])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    dtype = rng.choice(["float16", "bfloat16"])
    if kind == "decode":
        B = _log(rng, 1, 128)
        G = rng.choice([1, 2, 4, 5, 6, 8, 16, 24])
        hi = _log(rng, 1, min(65536, 200_000_000 // (B * HKV * D)))
        lo = rng.choice([0, 1, hi // 2, hi])
        cap = -(-rng.choice([hi, hi, 2 * hi]) // page) * page
        return _decode(B, HKV * G, HKV, D, page, cap, lo, hi, dtype, rng.random() < 0.5)
    if kind == "append":
        B = _log(rng, 1, 128)
        N = rng.choice([1, _log(rng, 2, max(2, min(16384, 60_000_000 // (B * HKV * D))))])
        return _append(B, N, HKV, D, page, dtype, rng.choice([dtype, dtype, "float32"]), rng.random() < 0.5,
                       rng.random() < 0.5)
    D, HKV = min(D, 128), min(HKV, 8)
    layers = rng.choice([1, 2, 4])
    if kind == "fork":
        width = _log(rng, 1, 16)
        groups = _log(rng, 1, 16)
        length = _log(rng, 1, min(6000, 5_000_000 // (groups * width * HKV * layers)))
        room = rng.choice([0, 0, _log(rng, 1, 300)])
        cap = -(-2 * (length + room) // page) * page
        return _fork(groups, width, rng.randint(1, width), length, room, page, cap, layers, HKV, D)
    pages = _log(rng, 64, min(20000, 600_000_000 // (page * HKV * D * layers)))
    if kind == "compact":
        live = rng.randint(pages // 8, 7 * pages // 8)
        moves = min(_log(rng, 1, live), pages - live)
        return _compact(pages, live, moves, rng.randint(1, 128), page, layers, HKV, D)
    return _copy(pages, _log(rng, 1, pages // 2), rng.random() < 0.5, page, layers, HKV, D)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _gen(seed, what):
    return torch.Generator(device=DEV).manual_seed(seed * 1_000_003 + 7919 * (what + 2))


def _lengths(c):
    """The rows' lengths in rising order: evenly spread over [lo, hi]."""
    return [c["hi"] if c["B"] == 1 else c["lo"] + (c["hi"] - c["lo"]) * b // (c["B"] - 1)
            for b in range(c["B"])]


def _pages(lens, page):
    return [-(-n // page) for n in lens]


def _table(lens, page, width, num_pages, g):
    """A block table whose rows hold distinct pages in no order, -1 past a row's pages."""
    B = lens.numel()
    need = (lens + page - 1) // page
    first = need.cumsum(0) - need
    slot = torch.arange(width, device=DEV)[None, :].expand(B, width)
    order = torch.randperm(num_pages, device=DEV, generator=g)
    at = (first[:, None] + slot).clamp(max=num_pages - 1)
    return torch.where(slot < need[:, None], order[at], -1).to(torch.int32)


def _pool(num_pages, HKV, page, D, dtype, g, mult=None):
    x = torch.randn(num_pages, HKV, page, D, device=DEV, generator=g, dtype=dtype)
    return x if mult is None else x.mul_(mult[:, None, :].to(dtype))


def _prepare_decode(c, seed):
    g = _gen(seed, 0)
    dtype = DTYPES[c["dtype"]]
    lens = torch.tensor(_lengths(c), device=DEV)[torch.randperm(c["B"], device=DEV, generator=g)]
    num_pages = max(1, sum(_pages(_lengths(c), c["page"])))
    s = dict(table=_table(lens, c["page"], max(1, c["cap"] // c["page"]), num_pages, g),
             lens=lens.to(torch.int32), ws={})
    mult = torch.ones(c["HKV"], c["D"], device=DEV)
    mult[:, torch.randperm(c["D"], device=DEV, generator=g)[:OUTLIERS]] = OUTLIER_SCALE
    s["k"] = _pool(num_pages, c["HKV"], c["page"], c["D"], dtype, g, mult)
    s["v"] = _pool(num_pages, c["HKV"], c["page"], c["D"], dtype, g)
    s["q"] = torch.randn(c["B"], c["HQ"], c["D"], device=DEV, generator=g, dtype=dtype)
    s["kn"] = s["vn"] = None
    if c["append"]:
        s["kn"] = torch.randn(c["B"], c["HKV"], c["D"], device=DEV, generator=g, dtype=dtype).mul_(mult.to(dtype))
        s["vn"] = torch.randn(c["B"], c["HKV"], c["D"], device=DEV, generator=g, dtype=dtype)
    s["out"] = torch.empty(c["B"], c["HQ"], c["D"], device=DEV)
    s["lse"] = torch.empty(c["B"], c["HQ"], device=DEV)
    return s


def _append_counts(c):
    """Tokens of each row, in rising order."""
    return [c["N"] - (c["N"] // 2) * (c["B"] - 1 - b) // max(1, c["B"] - 1) if c["counts"] else c["N"]
            for b in range(c["B"])]


def _prepare_append(c, seed):
    g = _gen(seed, 1)
    counts = torch.tensor(_append_counts(c), device=DEV)[torch.randperm(c["B"], device=DEV, generator=g)]
    before = torch.randint(0, 4 * c["page"], (c["B"],), device=DEV, generator=g)
    width = -(-(c["N"] + 4 * c["page"]) // c["page"])
    num_pages = c["B"] * width
    s = dict(table=_table(torch.full((c["B"],), width * c["page"], device=DEV), c["page"], width, num_pages, g),
             pos=before.to(torch.int32), counts=counts.to(torch.int32) if c["counts"] else None, ws={})
    s["k"], s["v"] = (_pool(num_pages, c["HKV"], c["page"], c["D"], DTYPES[c["dtype"]], g) for _ in range(2))
    if c["token_major"]:
        s["kn"], s["vn"] = (torch.randn(c["B"], c["N"], c["HKV"], c["D"], device=DEV, generator=g,
                                        dtype=DTYPES[c["x"]]).transpose(1, 2) for _ in range(2))
    else:
        s["kn"], s["vn"] = (torch.randn(c["B"], c["HKV"], c["N"], c["D"], device=DEV, generator=g,
                                        dtype=DTYPES[c["x"]]) for _ in range(2))
    return s


def _store(c, num_pages, g):
    """K and V pools of every layer: (2 * layers, num_pages, HKV, page, D)."""
    return torch.randn(2 * c["layers"], num_pages, c["HKV"], c["page"], c["D"], device=DEV, generator=g,
                       dtype=torch.float16)


def _fork_pages(c):
    """Pages of the pools: the parents' own, and twice what one call can ask for."""
    return c["groups"] * (c["survivors"] * -(-c["length"] // c["page"])
                          + c["width"] * 2 * (-(-c["room"] // c["page"]) + 2))


def _prepare_fork(c, seed):
    """Groups of ``width`` rows; in each, ``survivors`` rows of one length are in
    turn the parents of all the group's rows, and the others are empty at first.
    Run again and again the step stays the same: as many pages are copied,
    released and handed out."""
    g = _gen(seed, 2)
    rows, num_pages = c["groups"] * c["width"], _fork_pages(c)
    order = torch.rand(c["groups"], c["width"], device=DEV, generator=g).argsort(1)
    turn = torch.arange(c["width"], device=DEV) % c["survivors"]
    pick = turn[torch.rand(c["groups"], c["width"], device=DEV, generator=g).argsort(1)]
    parents = (torch.arange(c["groups"], device=DEV)[:, None] * c["width"] + order.gather(1, pick)).flatten()
    lens = torch.zeros(rows, dtype=torch.long, device=DEV)
    lens[parents] = c["length"]
    table = _table(lens, c["page"], c["cap"] // c["page"], num_pages, g)
    refs = torch.zeros(num_pages + 1, dtype=torch.int32, device=DEV)
    refs[table.long().flatten()] = 1  # -1 names the entry past the pages
    store = _store(c, num_pages, g)
    return dict(store=store, pools=list(store.unbind(0)), table=table, lens=lens.to(torch.int32),
                refs=refs[:-1].clone(), parents=parents.to(torch.int32),
                new=torch.full((rows,), c["length"] + c["room"], dtype=torch.int32, device=DEV) if c["room"] else None,
                page=c["page"], status=torch.zeros(1, dtype=torch.int32, device=DEV), ws={})


def _prepare_compact(c, seed):
    g = _gen(seed, 3)
    low = torch.randperm(c["live"], device=DEV, generator=g)[:c["live"] - c["moves"]]
    high = c["live"] + torch.randperm(c["pages"] - c["live"], device=DEV, generator=g)[:c["moves"]]
    used = torch.cat([low, high])[torch.randperm(c["live"], device=DEV, generator=g)]
    refs = torch.zeros(c["pages"], dtype=torch.int32, device=DEV)
    refs[used] = 1
    width = -(-c["live"] // c["rows"])
    table = torch.full((c["rows"] * width,), -1, dtype=torch.int32, device=DEV)
    table[:c["live"]] = used.to(torch.int32)
    table = table.view(c["rows"], width)
    store = _store(c, c["pages"], g)
    return dict(store=store, pools=list(store.unbind(0)), table=table, refs=refs,
                out=(torch.empty_like(table), torch.empty_like(refs)),
                live=torch.empty(1, dtype=torch.int32, device=DEV), ws={})


def _prepare_copy(c, seed):
    g = _gen(seed, 4)
    order = torch.randperm(c["pages"], device=DEV, generator=g).to(torch.int32)
    s = dict(store=_store(c, c["pages"], g), src=order[:c["pairs"]].clone(),
             dst=order[c["pages"] - c["pairs"]:].clone(), ws={})
    s["pools"] = list(s["store"].unbind(0))
    s["to"] = torch.zeros_like(s["store"]) if c["other"] else s["store"]
    s["to_pools"] = list(s["to"].unbind(0)) if c["other"] else None
    return s


def prepare(case, seed):
    make = {"decode": _prepare_decode, "append": _prepare_append, "fork": _prepare_fork,
            "compact": _prepare_compact, "copy": _prepare_copy}[case["kind"]]
    return dict(make(case, seed), kind=case["kind"])


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _scatter(pool, x, table, pos, counts):
    """x (B, HKV, N, D) into the pages of positions pos .. pos + counts - 1 (of all N without counts)."""
    B, HKV, N, D = x.shape
    page = pool.shape[2]
    n = torch.arange(N, device=x.device)
    t = pos.long()[:, None] + n
    entry = table.long().gather(1, (t // page).clamp(0, table.shape[1] - 1))
    ok = (t >= 0) & (t < table.shape[1] * page) & (entry >= 0) & (entry < pool.shape[0])
    if counts is not None:
        ok &= n < counts.long()[:, None]
    b, i = ok.nonzero(as_tuple=True)
    pool[entry[b, i], :, (t % page)[b, i]] = x[b, :, i].float().to(pool.dtype)


def _plain_decode(s):
    q, table, lens = s["q"].float(), s["table"], s["lens"].long()
    B, HQ, D = q.shape
    num_pages, HKV, page, _ = s["k"].shape
    if s["kn"] is not None:
        _scatter(s["k"], s["kn"][:, :, None], table, lens - 1, None)
        _scatter(s["v"], s["vn"][:, :, None], table, lens - 1, None)
    pages = table.long().clamp(0, num_pages - 1)
    k, v = (x[pages].permute(0, 2, 1, 3, 4).reshape(B, HKV, -1, D).float() for x in (s["k"], s["v"]))
    scores = torch.matmul(q.view(B, HKV, HQ // HKV, D), k.transpose(2, 3)) / math.sqrt(D)
    hidden = torch.arange(k.shape[2], device=q.device) >= lens[:, None]
    scores = scores.masked_fill(hidden[:, None, None], -math.inf)
    v = v.masked_fill(hidden[:, None, :, None], 0.0)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, torch.matmul(p, v) / total.clamp(min=1e-38), 0.0)
    return out.view(B, HQ, D), (top + total.log()).view(B, HQ)


def _plain_fork(s):
    table, lens, refs, page = s["table"], s["lens"].long(), s["refs"], s["page"]
    (B, P), N = table.shape, refs.numel()
    row, old = torch.arange(B, device=table.device), table.long()
    known = (s["parents"] >= 0) & (s["parents"] < B)
    a = s["parents"].long().clamp(0, B - 1)
    lens = lens.clamp(0, P * page)
    have = torch.where(known, lens[a], 0)
    want = torch.where(known, have if s["new"] is None else s["new"].long().clamp(min=0), 0)
    keep = torch.minimum(have, want)
    full, rest = keep // page, keep % page != 0
    # the partial page stays with one row, if nobody else keeps it: the parent itself, or its first child
    most = torch.full_like(row, -1).scatter_reduce(0, a, torch.where(known, full, -1), "amax")
    last = old[a, full.clamp(max=P - 1)].clamp(0, N - 1)
    heir = rest & (full == most[a]) & (refs[last] == 1)
    rank = torch.where(row == a, -1, row)
    best = torch.full_like(row, B).scatter_reduce(0, a, torch.where(heir, rank, B), "amin")
    heir &= rank == best[a]
    need = (want + page - 1) // page - full - heir.long()
    first = need.cumsum(0) - need
    free = refs == 0
    order = torch.zeros(N + 1, dtype=torch.long, device=table.device)
    order[torch.where(free, free.cumsum(0) - 1, N)] = torch.arange(N, device=table.device)
    long_rows = (want > P * page).any()
    short = need.sum() > free.sum()
    status = torch.where(long_rows, 2, torch.where(short, 1, 0)).to(torch.int32).view(1)
    done = status == 0
    slot = torch.arange(P, device=table.device)
    kept = (full + heir.long())[:, None]
    fresh = order[(first[:, None] + slot - kept).clamp(0, N - 1)]
    new = torch.where(slot < kept, old[a], torch.where(slot < ((want + page - 1) // page)[:, None], fresh, -1))
    was = (slot < ((lens + page - 1) // page)[:, None]) & (old >= 0) & (old < N)
    now = (slot < ((want + page - 1) // page)[:, None]) & (new >= 0) & (new < N)
    change = torch.zeros(N, dtype=torch.int32, device=table.device)
    change.index_add_(0, new.clamp(0, N - 1).flatten(), now.to(torch.int32).flatten())
    change.index_add_(0, old.clamp(0, N - 1).flatten(), -was.to(torch.int32).flatten())
    copied = (rest & ~heir & done).nonzero().flatten()
    s["store"][:, order[first[copied].clamp(max=N - 1)]] = s["store"][:, last[copied]]
    s["table"].copy_(torch.where(done, new, old))
    s["lens"].copy_(torch.where(done, want, s["lens"].long()))
    s["refs"].add_(torch.where(done, change, 0))
    s["status"].copy_(status)


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    N = refs.numel()
    page = torch.arange(N, device=refs.device)
    used = refs > 0
    live = used.sum()
    src, dst = used & (page >= live), ~used & (page < live)
    src_at, dst_at = src.nonzero().flatten(), dst.nonzero().flatten()
    s["store"][:, dst_at] = s["store"][:, src_at]
    to = page.clone()
    to[src_at] = dst_at
    known = (table >= 0) & (table < N)
    s["out"][0].copy_(torch.where(known, to[table.long().clamp(0, N - 1)], table.long()))
    moved = torch.zeros_like(refs)
    moved[to[used]] = refs[used]
    s["out"][1].copy_(moved)
    s["live"].copy_(live.view(1))


def run(state):
    s = state
    if s["kind"] == "decode":
        if own:
            from tritonkv_amd.paged16 import paged16_decode_attention

            out = paged16_decode_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], out=s["out"],
                                           lse=s["lse"], _workspace=s["ws"], k_new=s["kn"], v_new=s["vn"])
            lse = s["lse"]
        else:
            out, lse = _plain_decode(s)
        return (out, lse) if s["kn"] is None else (out, lse, s["k"], s["v"])
    if s["kind"] == "append":
        if own:
            from tritonkv_amd.paged16 import paged16_append

            paged16_append(s["k"], s["v"], s["kn"], s["vn"], s["table"], s["pos"], s["counts"],
                           _workspace=s["ws"])
        else:
            _scatter(s["k"], s["kn"], s["table"], s["pos"], s["counts"])
            _scatter(s["v"], s["vn"], s["table"], s["pos"], s["counts"])
        return s["k"], s["v"]
    if s["kind"] == "fork":
        if own:
            from tritonkv_amd.pages import fork_rows

            fork_rows(s["pools"], s["table"], s["lens"], s["refs"], s["parents"], s["new"],
                      status=s["status"], _workspace=s["ws"])
        else:
            _plain_fork(s)
        return s["table"], s["lens"], s["refs"], s["status"], s["store"]
    if s["kind"] == "compact":
        if own:
            from tritonkv_amd.pages import compact_pages

            compact_pages(s["pools"], s["table"], s["refs"], out=s["out"], live=s["live"], _workspace=s["ws"])
        else:
            _plain_compact(s)
        return s["out"][0], s["out"][1], s["live"], s["store"]
    if own:
        from tritonkv_amd.pages import copy_pages

        copy_pages(s["pools"], s["src"], s["dst"], s["to_pools"], _workspace=s["ws"])
    else:
        s["to"][:, s["dst"].long()] = s["store"][:, s["src"].long()]
    return s["to"]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    c = case
    size = {"float16": 2, "bfloat16": 2, "float32": 4}
    if c["kind"] == "decode":
        lens = _lengths(c)
        row = c["HKV"] * c["D"] * 2  # one token's keys, or its values
        io = c["B"] * c["HQ"] * (c["D"] * (2 + 4) + 4) + 4 * (c["B"] + sum(_pages(lens, c["page"])))
        return {"bytes": 2 * row * sum(lens) + io + (4 * row * c["B"] if c["append"] else 0),
                "flops": 4.0 * c["HQ"] * c["D"] * sum(lens)}
    if c["kind"] == "append":
        tokens = sum(_append_counts(c))
        return {"bytes": 2 * c["HKV"] * c["D"] * tokens * (size[c["x"]] + 2), "flops": 0.0}
    page_bytes = 2 * c["layers"] * c["HKV"] * c["page"] * c["D"] * 2
    if c["kind"] == "fork":
        rows, end = c["groups"] * c["width"], c["length"] + c["room"]
        copies = c["groups"] * (c["width"] - c["survivors"]) if end % c["page"] else 0
        return {"bytes": 2 * page_bytes * copies + 8 * rows * -(-end // c["page"]) + 12 * rows
                + 4 * _fork_pages(c), "flops": 0.0}
    if c["kind"] == "compact":
        return {"bytes": 2 * page_bytes * c["moves"] + 8 * c["live"] + 8 * c["pages"], "flops": 0.0}
    return {"bytes": 2 * page_bytes * c["pairs"] + 8 * c["pairs"], "flops": 0.0}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits, one row or page at a time
# ---------------------------------------------------------------------------


def _exact_decode(c, s):
    lens, table, page = s["lens"].tolist(), s["table"].tolist(), c["page"]
    G = c["HQ"] // c["HKV"]
    out = torch.zeros(c["B"], c["HQ"], c["D"], dtype=torch.float64, device=DEV)
    lse = torch.full((c["B"], c["HQ"]), -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        at = torch.tensor(table[b][:-(-n // page)], device=DEV)
        k, v = (s[x][at].double().transpose(0, 1).reshape(c["HKV"], -1, c["D"])[:, :n] for x in "kv")
        if c["append"]:
            k, v = torch.cat([k[:, :-1], s["kn"][b].double()[:, None]], 1), torch.cat(
                [v[:, :-1], s["vn"][b].double()[:, None]], 1)
        for h in range(c["HKV"]):
            x = (k[h] @ s["q"][b, h * G:(h + 1) * G].double().T).T * c["D"] ** -0.5
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(x, -1)
            out[b, h * G:(h + 1) * G] = torch.softmax(x, -1) @ v[h]
    return (out, lse, None, None) if c["append"] else (out, lse)


def _exact_append(c, s):
    table, pos = s["table"].tolist(), s["pos"].tolist()
    counts = s["counts"].tolist() if c["counts"] else [c["N"]] * c["B"]
    got = []
    for pool, x in ((s["k"], s["kn"]), (s["v"], s["vn"])):
        out = pool.double()
        for b in range(c["B"]):
            n = 0
            while n < counts[b]:
                at, first = divmod(pos[b] + n, c["page"])
                m = min(c["page"] - first, counts[b] - n)
                out[table[b][at], :, first:first + m] = x[b, :, n:n + m].double()
                n += m
        got.append(out)
    return tuple(got)


def _exact_fork(c, s):
    page, refs = c["page"], s["refs"].tolist()
    table, lens, parents = s["table"].tolist(), s["lens"].tolist(), s["parents"].tolist()
    rows = range(len(parents))
    ends = s["new"].tolist() if c["room"] else [lens[a] for a in parents]
    free = [p for p, n in enumerate(refs) if n == 0]
    src, dst = [], []
    for b in rows:
        a = parents[b]
        keep = min(lens[a], ends[b])
        pages = -(-ends[b] // page) - keep // page
        if keep % page:
            children = [r for r in rows if parents[r] == a]
            if (a if a in children else children[0]) == b:
                pages -= 1
            else:
                src.append(table[a][keep // page])
                dst.append(free[0])
        free = free[pages:]
    store = s["store"].double()
    store[:, dst] = s["store"][:, src].double()
    return None, None, None, None, store


def _exact_compact(c, s):
    refs = s["refs"].tolist()
    live = sum(n > 0 for n in refs)
    src = [p for p in range(live, len(refs)) if refs[p] > 0]
    dst = [p for p in range(live) if refs[p] == 0]
    store = s["store"].double()
    store[:, dst] = s["store"][:, src].double()
    return None, None, None, store


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        to = s["to"].double()
        to[:, s["dst"].tolist()] = s["store"][:, s["src"].tolist()].double()
        return to
    return {"decode": _exact_decode, "append": _exact_append, "fork": _exact_fork,
            "compact": _exact_compact}[case["kind"]](case, s)
