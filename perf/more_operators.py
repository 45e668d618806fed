"""The operators of an 8-bit paged cache, as cases to time and to compare.

Four operators: ``paged8_decode_attention`` (attention of the last tokens of
every row over pages of e4m3 or int8 codes with a scale for each block of tokens
and KV head), ``paged8_append`` (tokens quantized into such pages as they are
written, with rotary positions on the way where a case says so), ``paged8_read``
(tokens of such pages back as 16- or 32-bit values) and ``apply_rotary`` (rotary
positions of queries and keys).

A case is a dict with ``kind`` and the sizes of that kind.  ``run`` takes the
operators' plain form, in elementary torch operations and 32 bits (angles in 64),
or (``own``) the package's entry points.  Lengths and counts of tokens follow from
the case alone; the seed decides values, which row has which length and which page
is which.

The format: a block is ``block`` consecutive slots of a page; a value is its code
times its block's scale.  Codes are e4m3 (largest 448) or int8 (largest 127).  An
append gives a block the least power of two, 2^-64 or more, under which its new
values fit the codes (magnitudes above 2^64 count as 2^64), or keeps the scale that
is there if that is larger; where it grows, the codes of the block's earlier tokens
are rounded again under the new one.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32,
          "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
CODE_MAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
OUTLIERS, OUTLIER_SCALE = 4, 8.0  # channels per KV head that stand out, as in the benchmark's caches
LARGEST, LEAST_SCALE = 2.0 ** 64, 2.0 ** -64


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def _decode(B, HQ, HKV, D, M, page, block, cap, lo, hi, codes, dtype, counts):
    return dict(kind="decode", B=B, HQ=HQ, HKV=HKV, D=D, M=M, page=page, block=block, cap=cap, lo=lo, hi=hi,
                codes=codes, dtype=dtype, counts=counts)


def _append(B, N, HQ, HKV, D, page, block, codes, x, counts, token_major, rot):
    """rot: the dims of a head that turn, 0: no rotary positions (and no queries)."""
    return dict(kind="append", B=B, N=N, HQ=HQ, HKV=HKV, D=D, page=page, block=block, codes=codes, x=x,
                counts=counts, token_major=token_major, rot=rot)


def _read(B, HKV, D, page, block, lo, hi, codes, x):
    return dict(kind="read", B=B, HKV=HKV, D=D, page=page, block=block, lo=lo, hi=hi, codes=codes, x=x)


def _rotary(B, N, HQ, HKV, D, rot, far, x, interleaved, token_major, stretch, factor, adjoint):
    return dict(kind="rotary", B=B, N=N, HQ=HQ, HKV=HKV, D=D, rot=rot, far=far, x=x, interleaved=interleaved,
                token_major=token_major, stretch=stretch, factor=factor, adjoint=adjoint)


def listed():
    return [
        # One sequence of the Qwen2.5-1.5B shape, a short chat: latency counts.
        dict(_decode(1, 12, 2, 128, 1, 64, 32, 512, 505, 505, "e4m3", "float16", False), name="decode_b1_short"),
        # A small batch of a model without shared KV heads, head dim 64, int8
        # codes, rows from a single token to 2999.
        dict(_decode(8, 16, 16, 64, 1, 32, 32, 4096, 1, 2999, "int8", "bfloat16", False), name="decode_mha_d64"),
        # Verifying four drafted tokens of 16 requests at once; some drafted fewer.
        dict(_decode(16, 64, 8, 128, 4, 64, 32, 8192, 500, 8000, "int8", "bfloat16", True), name="decode_drafts"),
        # A 70B-style continuous batch: lengths 1k to 16k in tables made for twice that.
        dict(_decode(32, 64, 8, 128, 1, 64, 64, 32768, 1000, 16384, "e4m3", "bfloat16", False),
             name="decode_70b_ragged"),
        # The benchmark's Llama-3-8B batch, 32 rows at 32k.
        dict(_decode(32, 32, 8, 128, 1, 256, 128, 32768, 32768, 32768, "e4m3", "float16", False),
             name="decode_8b_large"),
        # One decode step of a serving batch: q and k turned, k and v quantized.
        dict(_append(64, 1, 64, 8, 128, 64, 32, "e4m3", "bfloat16", False, False, 128), name="append_step_rotary"),
        # Prompts as the projections leave them (token-major), padded to the
        # longest, each row's own count of tokens.
        dict(_append(4, 8213, 32, 8, 128, 64, 32, "e4m3", "float16", True, True, 0), name="append_prompt"),
        # The same with rotary positions on the way, 64 tokens to a scale.
        dict(_append(4, 2049, 32, 8, 128, 64, 64, "e4m3", "bfloat16", True, True, 128),
             name="append_prompt_rotary"),
        # A short prefix read back for the prefill of what follows it.
        dict(_read(1, 2, 128, 64, 32, 505, 505, "e4m3", "float16"), name="read_prefix"),
        # Rows of a large batch handed to another cache.
        dict(_read(8, 8, 128, 64, 32, 2000, 16384, "int8", "bfloat16"), name="read_rows"),
        # One decode step's q and k.
        dict(_rotary(64, 1, 32, 8, 128, 128, 131072, "bfloat16", False, False, 1.0, 1.0, False),
             name="rotary_step"),
        # Prompts of a model that turns a part of each head in neighbouring
        # pairs, its context stretched four times.
        dict(_rotary(4, 8213, 32, 8, 128, 64, 131072, "bfloat16", True, True, 4.0, 1.1386, False),
             name="rotary_prompt"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "append", "append", "read", "rotary"])
    HKV, D = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 128, 128, 256])
    block = rng.choice([32, 32, 64, 128])
    page = block * rng.choice([1, 2, 3, 4])
    codes = rng.choice(["e4m3", "int8"])
    x = rng.choice(["float16", "bfloat16"])
    G = rng.choice([1, 2, 4, 5, 6, 8, 16, 24])
    if kind == "decode":
        B, M = _log(rng, 1, 128), rng.choice([1, 1, 1, 2, 3, 4, 8])
        hi = _log(rng, 1, min(65536, 100_000_000 // (B * HKV * D * M)))
        lo = rng.choice([0, 1, hi // 2, hi])
        cap = -(-rng.choice([hi, hi, 2 * hi]) // page) * page
        return _decode(B, HKV * G, HKV, D, M, page, block, cap, lo, hi, codes, x, M > 1 and rng.random() < 0.5)
    if kind == "append":
        B = _log(rng, 1, 128)
        rot = rng.choice([0, 0, D, D // 2])
        N = rng.choice([1, _log(rng, 2, max(2, min(16384, 30_000_000 // (B * HKV * D * (1 + (G if rot else 0))))))])
        return _append(B, N, HKV * G, HKV, D, page, block, codes, rng.choice([x, x, "float32"]),
                       rng.random() < 0.5, rng.random() < 0.5, rot)
    if kind == "read":
        B = _log(rng, 1, 64)
        hi = _log(rng, 1, min(32768, 60_000_000 // (B * HKV * D)))
        return _read(B, HKV, D, page, block, rng.choice([0, 1, hi // 2, hi]), hi, codes,
                     rng.choice([x, x, "float32"]))
    B = _log(rng, 1, 128)
    N = rng.choice([1, _log(rng, 2, max(2, min(16384, 60_000_000 // (B * HKV * D * (1 + G)))))])
    rot = rng.choice([D, D, D // 2, D // 4, 20])
    return _rotary(B, N, HKV * G, HKV, D, rot, _log(rng, 1000, 1_000_000), rng.choice([x, x, "float32"]),
                   rng.random() < 0.5, rng.random() < 0.5, rng.choice([1.0, 4.0, 32.0]),
                   rng.choice([1.0, 1.0, 1.1386]), rng.random() < 0.3)


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


def _outliers(c, g):
    mult = torch.ones(c["HKV"], c["D"], device=DEV)
    mult[:, torch.randperm(c["D"], device=DEV, generator=g)[:OUTLIERS]] = OUTLIER_SCALE
    return mult


def _need(top, code):
    """The least scale under which magnitudes up to ``top`` fit the codes."""
    m, e = torch.frexp(top)
    whole, bits = (0.875, 9) if code is torch.float8_e4m3fn else (127 / 128, 7)
    s = torch.ldexp(torch.ones_like(m), (e - bits + (m > whole)).to(torch.int32))
    return torch.where(top > 0, s, 0.0).clamp(min=LEAST_SCALE)


def _round(y, code):
    """Values over their scale to codes, nearest even."""
    if code is torch.int8:
        return y.nan_to_num(0.0).round().clamp(-127.0, 127.0).to(torch.int8)
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _pool(c, num_pages, g, mult):
    """Codes and scales of a pool filled with normal values, ``mult`` standing out."""
    code, n = DTYPES[c["codes"]], c["page"] // c["block"]
    x = torch.randn(num_pages, c["HKV"], n, c["block"], c["D"], device=DEV, generator=g, dtype=torch.float16)
    if mult is not None:
        x.mul_(mult[:, None, None, :].to(x.dtype))
    scale = _need(x.abs().amax((3, 4)).float(), code)
    codes = _round(x.float().div_(scale[..., None, None]), code)
    return codes.view(num_pages, c["HKV"], c["page"], c["D"]), scale


def _rows(c, H, N, g, dtype, mult=None):
    """(B, H, N, D) values, token-major in memory where the case says so."""
    shape = (c["B"], N, H, c["D"]) if c.get("token_major") else (c["B"], H, N, c["D"])
    x = torch.randn(*shape, device=DEV, generator=g, dtype=dtype)
    x = x.transpose(1, 2) if c.get("token_major") else x
    return x if mult is None else x.mul_(mult[:, None, :].to(dtype))


def _frequencies(c):
    """Radians per position of the pairs of a head, in 64 bits: base 500000 over the dims
    that turn, stretched as a whole for a longer context."""
    i = torch.arange(c["rot"] // 2, dtype=torch.float64, device=DEV)
    return torch.exp(-2.0 * i / c["rot"] * math.log(500000.0)) / c.get("stretch", 1.0)


def _prepare_decode(c, seed):
    g = _gen(seed, 0)
    order = torch.randperm(c["B"], device=DEV, generator=g)
    lens = torch.tensor(_lengths(c), device=DEV)[order]
    num_pages = max(1, sum(_pages(_lengths(c), c["page"])))
    s = dict(table=_table(lens, c["page"], max(1, c["cap"] // c["page"]), num_pages, g),
             lens=lens.to(torch.int32), counts=None, ws={})
    if c["counts"]:  # 1 to M of the row's tokens ask
        s["counts"] = (1 + order % c["M"]).to(torch.int32)
    s["k"], s["ks"] = _pool(c, num_pages, g, _outliers(c, g))
    s["v"], s["vs"] = _pool(c, num_pages, g, None)
    s["q"] = torch.randn(c["B"], c["M"], c["HQ"], c["D"], device=DEV, generator=g,
                         dtype=DTYPES[c["dtype"]]).transpose(1, 2)
    s["out"] = torch.empty(c["B"], c["HQ"], c["M"], c["D"], device=DEV)
    s["lse"] = torch.empty(c["B"], c["HQ"], c["M"], device=DEV)
    return s


def _append_counts(c):
    """Tokens of each row, in rising order."""
    return [c["N"] - (c["N"] // 2) * (c["B"] - 1 - b) // max(1, c["B"] - 1) if c["counts"] else c["N"]
            for b in range(c["B"])]


def _prepare_append(c, seed):
    g = _gen(seed, 1)
    counts = torch.tensor(_append_counts(c), device=DEV)[torch.randperm(c["B"], device=DEV, generator=g)]
    before = torch.randint(0, c["page"], (c["B"],), device=DEV, generator=g)
    width = -(-(c["N"] + c["page"]) // c["page"])
    num_pages = c["B"] * width
    s = dict(table=_table(torch.full((c["B"],), width * c["page"], device=DEV), c["page"], width, num_pages, g),
             pos=before.to(torch.int32), counts=counts.to(torch.int32) if c["counts"] else None, q=None, q_out=None,
             ws={})
    mult = _outliers(c, g)
    s["k"], s["ks"] = _pool(c, num_pages, g, mult)
    s["v"], s["vs"] = _pool(c, num_pages, g, None)
    s["kn"], s["vn"] = (_rows(c, c["HKV"], c["N"], g, DTYPES[c["x"]], m) for m in (mult, None))
    if c["rot"]:
        s["w"] = _frequencies(c)
        s["q"] = _rows(c, c["HQ"], c["N"], g, DTYPES[c["x"]])
        s["q_out"] = torch.zeros_like(s["q"])
    return s


def _prepare_read(c, seed):
    g = _gen(seed, 2)
    lens = torch.tensor(_lengths(c), device=DEV)[torch.randperm(c["B"], device=DEV, generator=g)]
    before = torch.randint(0, 2 * c["page"], (c["B"],), device=DEV, generator=g)
    num_pages = sum(_pages(_lengths(c), c["page"])) + 2 * c["B"]
    s = dict(table=_table(lens + before, c["page"], c["hi"] // c["page"] + 3, num_pages, g),
             pos=before.to(torch.int32), counts=lens.to(torch.int32), ws={})
    s["k"], s["ks"] = _pool(c, num_pages, g, _outliers(c, g))
    s["v"], s["vs"] = _pool(c, num_pages, g, None)
    s["out"] = tuple(torch.zeros(c["B"], c["HKV"], c["hi"], c["D"], device=DEV, dtype=DTYPES[c["x"]])
                     for _ in range(2))
    return s


def _prepare_rotary(c, seed):
    g = _gen(seed, 3)
    s = dict(pos=torch.randint(0, c["far"], (c["B"],), device=DEV, generator=g).to(torch.int32),
             w=_frequencies(c), q=_rows(c, c["HQ"], c["N"], g, DTYPES[c["x"]]),
             k=_rows(c, c["HKV"], c["N"], g, DTYPES[c["x"]]), ws={})
    s["out"] = (torch.zeros_like(s["q"]), torch.zeros_like(s["k"]))
    return s


def prepare(case, seed):
    make = {"decode": _prepare_decode, "append": _prepare_append, "read": _prepare_read, "rotary": _prepare_rotary}
    return dict(make[case["kind"]](case, seed), kind=case["kind"], c=dict(case))


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _turn(x, t, w, interleaved=False, factor=1.0, adjoint=False):
    """x (B, H, N, D) in 32 bits, its first 2 * len(w) dims turned by t (B, N) times w."""
    n = w.numel()
    angle = t.double()[:, None, :, None] * w
    cos, sin = (factor * angle.cos()).float(), (factor * angle.sin()).float()
    sin = -sin if adjoint else sin
    y = x.float()
    a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else (y[..., :n], y[..., n:2 * n])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1),
                      y[..., 2 * n:]], -1)


def _put(codes, scale, x, table, pos, counts):
    """x (B, HKV, N, D), in 32 bits, quantized into the pages of positions pos .. pos + counts - 1."""
    code, N = codes.dtype, x.shape[2]
    P, HKV, page, D = codes.shape
    blocks = scale.shape[2]
    block = page // blocks
    n = torch.arange(N, device=x.device)
    t = pos.long()[:, None] + n
    entry = table.long().gather(1, (t // page).clamp(0, table.shape[1] - 1))
    ok = (t >= 0) & (t < table.shape[1] * page) & (entry >= 0) & (entry < P)
    if counts is not None:
        ok &= n < counts.long()[:, None]
    b, i = ok.nonzero(as_tuple=True)
    at, slot = entry[b, i], (t % page)[b, i]
    y = x[b, :, i].clamp(-LARGEST, LARGEST)  # (tokens, HKV, D)
    group = at * blocks + slot // block
    top = y.abs().nan_to_num(0.0).amax(-1)
    most = torch.zeros(P * blocks, HKV, device=x.device).index_reduce_(0, group, top, "amax")
    first = torch.full((P * blocks,), block, device=x.device).scatter_reduce_(0, group, slot % block, "amin")
    was = scale.transpose(1, 2).reshape(P * blocks, HKV)
    was = torch.where((first[:, None] > 0) & (was > 0) & (was < math.inf), was, 0.0)
    now = torch.maximum(was, _need(most, code))
    # earlier tokens of blocks whose scale grows are rounded again
    grown = ((first < block)[:, None] & (was > 0) & (now > was)).any(1).nonzero().flatten()
    raw = codes.view(torch.int8).view(P, HKV, blocks, block, D)
    old = raw[grown // blocks, :, grown % blocks]  # (grown, HKV, block, D)
    ratio = torch.where(was > 0, was / now, 1.0)[grown][..., None, None]
    keep = torch.arange(block, device=x.device)[:, None] < first[grown][:, None, None, None]
    raw[grown // blocks, :, grown % blocks] = torch.where(
        keep, _round(old.view(code).float() * ratio, code).view(torch.int8), old)
    touched = (first < block).nonzero().flatten()
    scale[touched // blocks, :, touched % blocks] = now[touched]
    codes.view(torch.int8)[at, :, slot] = _round(y / now[group][..., None], code).view(torch.int8)


def _values(codes, scale):
    """The values that codes stand for, in 32 bits."""
    return (codes.float().view(*scale.shape, -1, codes.shape[-1]) * scale[..., None, None]).view(codes.shape)


def _plain_decode(s):
    q, table, lens = s["q"].float(), s["table"], s["lens"].long()
    B, HQ, M, D = q.shape
    num_pages, HKV, page, _ = s["k"].shape
    G = HQ // HKV
    pages = table.long().clamp(0, num_pages - 1)
    k, v = (_values(s[x].view(torch.int8)[pages].view(s[x].dtype).flatten(0, 1), s[x + "s"][pages].flatten(0, 1))
            .view(B, -1, HKV, page, D).permute(0, 2, 1, 3, 4).reshape(B, HKV, -1, D) for x in ("k", "v"))
    ask = s["counts"].long() if s["counts"] is not None else torch.full_like(lens, M)
    m = torch.arange(M, device=q.device)
    seen = torch.where(m < ask[:, None], (lens[:, None] - (ask[:, None] - 1 - m)).clamp(min=0), 0)  # (B, M)
    t = torch.arange(k.shape[2], device=q.device)
    scores = torch.matmul(q.reshape(B, HKV, G * M, D), k.transpose(2, 3)).div_(math.sqrt(D)).view(B, HKV, G, M, -1)
    scores.masked_fill_(t >= seen[:, None, None, :, None], -math.inf)
    v = v.masked_fill(t[:, None] >= lens[:, None, None, None], 0.0)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, HKV, G * M, -1), v).view(B, HKV, G, M, D)
    out = torch.where(total > 0, out / total.clamp(min=1e-38), 0.0)
    return out.view(B, HQ, M, D), (top + total.log()).view(B, HQ, M)


def _plain_append(s):
    kn, q = s["kn"].float(), None
    if s["q"] is not None:
        t = s["pos"].long()[:, None] + torch.arange(kn.shape[2], device=kn.device)
        kn, q = _turn(kn, t, s["w"]), _turn(s["q"], t, s["w"]).to(s["q"].dtype)
        if s["counts"] is not None:
            live = torch.arange(kn.shape[2], device=kn.device) < s["counts"].long()[:, None]
            q = torch.where(live[:, None, :, None], q, s["q_out"])
    _put(s["k"], s["ks"], kn, s["table"], s["pos"], s["counts"])
    _put(s["v"], s["vs"], s["vn"].float(), s["table"], s["pos"], s["counts"])
    return q


def _plain_read(s):
    B, HKV, N, D = s["out"][0].shape
    num_pages, _, page, _ = s["k"].shape
    n = torch.arange(N, device=s["k"].device)
    live = n < s["counts"].long()[:, None]
    t = s["pos"].long()[:, None] + n
    at = s["table"].long().gather(1, (t // page).clamp(0, s["table"].shape[1] - 1)).clamp(0, num_pages - 1)
    slot = t % page
    got = []
    for x, out in zip("kv", s["out"]):
        block = page // s[x + "s"].shape[2]
        codes = s[x].view(torch.int8)[at, :, slot].view(s[x].dtype).float()  # (B, N, HKV, D)
        y = (codes * s[x + "s"][at, :, slot // block][..., None]).transpose(1, 2).to(out.dtype)
        got.append(torch.where(live[:, None, :, None], y, out))
    return tuple(got)


def _plain_rotary(s):
    c = s["c"]
    t = s["pos"].long()[:, None] + torch.arange(c["N"], device=s["q"].device)
    return tuple(_turn(s[x], t, s["w"], c["interleaved"], c["factor"], c["adjoint"]).to(s[x].dtype) for x in "qk")


def _held(s):
    """The pools after an append.  e4m3 codes are values in units of their scale; int8 codes
    are given as the values they stand for, which are exact in bfloat16 (seven bits times
    a power of two)."""
    if s["k"].dtype is torch.int8:
        return tuple((s[x].to(torch.bfloat16).view(*s[x + "s"].shape, -1, s[x].shape[3])
                      * s[x + "s"].to(torch.bfloat16)[..., None, None]).view(s[x].shape) for x in "kv")
    return s["k"], s["ks"], s["v"], s["vs"]


def _own_pools(s):
    if "pools" not in s:
        from tritonkv_amd.paged8 import Paged8Pool

        s["pools"] = Paged8Pool(s["k"], s["ks"]), Paged8Pool(s["v"], s["vs"])
    return s["pools"]


def _own_rotary(s):
    if "rotary" not in s:
        from tritonkv_amd.rotary import Rotary

        c = s["c"]
        s["rotary"] = Rotary(inv_freq=s["w"], interleaved=c.get("interleaved", False), factor=c.get("factor", 1.0))
    return s["rotary"]


def run(state):
    s = state
    if s["kind"] == "decode":
        if own:
            from tritonkv_amd.paged8 import paged8_decode_attention

            paged8_decode_attention(s["q"], *_own_pools(s), s["table"], s["lens"], counts=s["counts"], out=s["out"],
                                    lse=s["lse"], _workspace=s["ws"])
            return s["out"], s["lse"]
        return _plain_decode(s)
    if s["kind"] == "append":
        if own:
            from tritonkv_amd.paged8 import paged8_append

            q = paged8_append(*_own_pools(s), s["kn"], s["vn"], s["table"], s["pos"], s["counts"], q=s["q"],
                              q_out=s["q_out"], rotary=_own_rotary(s) if s["q"] is not None else None,
                              _workspace=s["ws"])
        else:
            q = _plain_append(s)
        return _held(s) if q is None else (*_held(s), q)
    if s["kind"] == "read":
        if own:
            from tritonkv_amd.paged8 import paged8_read

            return paged8_read(*_own_pools(s), s["table"], s["pos"], s["counts"], out=s["out"], _workspace=s["ws"])
        return _plain_read(s)
    if own:
        from tritonkv_amd.rotary import apply_rotary

        return apply_rotary(s["q"], s["k"], s["pos"], _own_rotary(s), adjoint=s["c"]["adjoint"], out=s["out"],
                            _workspace=s["ws"])
    return _plain_rotary(s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    c = case
    size = {"float16": 2, "bfloat16": 2, "float32": 4}
    if c["kind"] == "decode":
        lens = _lengths(c)
        rows = c["B"] * c["HQ"] * c["M"]
        held = 2 * c["HKV"] * (c["D"] * sum(lens) + 4 * sum(_pages(lens, c["block"])))
        return {"bytes": held + rows * (c["D"] * (2 + 4) + 4) + 4 * (c["B"] + sum(_pages(lens, c["page"]))),
                "flops": 4.0 * c["HQ"] * c["M"] * c["D"] * sum(lens)}
    if c["kind"] == "append":
        tokens = sum(_append_counts(c))
        new = 2 * c["HKV"] * tokens * (c["D"] * (size[c["x"]] + 1) + 4.0 / c["block"])
        return {"bytes": new + (2 * c["HQ"] * c["D"] * tokens * size[c["x"]] if c["rot"] else 0),
                "flops": 3.0 * (c["HQ"] + c["HKV"]) * c["rot"] * tokens}
    if c["kind"] == "read":
        return {"bytes": 2 * c["HKV"] * sum(_lengths(c)) * (c["D"] * (1 + size[c["x"]]) + 4.0 / c["block"]),
                "flops": 0.0}
    values = c["B"] * c["N"] * (c["HQ"] + c["HKV"])
    return {"bytes": 2 * values * c["D"] * size[c["x"]], "flops": 3.0 * values * c["rot"]}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits, one row, block or pair of dims at a time
# ---------------------------------------------------------------------------


def _exact_codes(y, code):
    """The codes nearest to y, as numbers."""
    if code == "int8":
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_pages(codes, scale, pages):
    """Tokens of one row's pages as (HKV, tokens, D)."""
    block = codes.shape[2] // scale.shape[2]
    y = codes.view(torch.int8)[pages].view(codes.dtype).double()
    y = y * scale[pages].double().repeat_interleave(block, 2)[..., None]
    return y.transpose(0, 1).reshape(codes.shape[1], -1, codes.shape[3])


def _exact_decode(c, s):
    lens, table = s["lens"].tolist(), s["table"].tolist()
    asks = s["counts"].tolist() if c["counts"] else [c["M"]] * c["B"]
    G = c["HQ"] // c["HKV"]
    out = torch.zeros(c["B"], c["HQ"], c["M"], c["D"], dtype=torch.float64, device=DEV)
    lse = torch.full((c["B"], c["HQ"], c["M"]), -math.inf, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        at = torch.tensor(table[b][:-(-n // c["page"])], device=DEV)
        k, v = _exact_pages(s["k"], s["ks"], at), _exact_pages(s["v"], s["vs"], at)
        for m in range(asks[b]):
            L = n - (asks[b] - 1 - m)
            for h in range(c["HKV"]):
                if L > 0:
                    x = (k[h, :L] @ s["q"][b, h * G:(h + 1) * G, m].double().T).T * c["D"] ** -0.5
                    lse[b, h * G:(h + 1) * G, m] = torch.logsumexp(x, -1)
                    out[b, h * G:(h + 1) * G, m] = torch.softmax(x, -1) @ v[h, :L]
    return out, lse


def _exact_turn(x, t, c):
    """x (H, n, D) at the positions t .. t + n - 1, as complex numbers turned by exp(i angle)."""
    n, sign = c["rot"] // 2, -1.0 if c.get("adjoint") else 1.0
    y = x.double().clone()
    for i in range(n):
        p, q = (2 * i, 2 * i + 1) if c.get("interleaved") else (i, i + n)
        w = 500000.0 ** (-2.0 * i / c["rot"]) / c.get("stretch", 1.0)
        angle = torch.arange(t, t + x.shape[1], dtype=torch.float64, device=DEV) * w
        z = torch.complex(y[..., p], y[..., q]) * torch.polar(torch.full_like(angle, c.get("factor", 1.0)), sign * angle)
        y[..., p], y[..., q] = z.real, z.imag
    return y


def _exact_append(c, s):
    table, pos = s["table"].tolist(), s["pos"].tolist()
    counts = s["counts"].tolist() if c["counts"] else [c["N"]] * c["B"]
    top, block = 448.0 if c["codes"] == "e4m3" else 127.0, c["block"]
    q = s["q_out"].double() if c["rot"] else None
    got = []
    for name in "kv":
        codes, scale = s[name].double(), s[name + "s"].double()
        for b in range(c["B"]):
            x = s[name + "n"][b, :, :counts[b]].double()
            if c["rot"] and name == "k":
                x = _exact_turn(x, pos[b], c)
                q[b, :, :counts[b]] = _exact_turn(s["q"][b, :, :counts[b]], pos[b], c)
            n = 0
            while n < counts[b]:
                at, slot = divmod(pos[b] + n, c["page"])
                i, first = divmod(slot, block)
                m = min(block - first, counts[b] - n)
                y, page = x[:, n:n + m], table[b][at]
                need = torch.exp2(torch.ceil(torch.log2(y.abs().amax((1, 2)) / top)).clamp(min=-64.0))
                had = scale[page, :, i]
                now = need if first == 0 else torch.maximum(had, need)
                held = codes[page, :, i * block:(i + 1) * block]
                held[:, :first] = _exact_codes(held[:, :first] * (had / now)[:, None, None], c["codes"])
                held[:, first:first + m] = _exact_codes(y / now[:, None, None], c["codes"])
                scale[page, :, i] = now
                n += m
        got += [codes * scale.repeat_interleave(block, 2)[..., None]] if c["codes"] == "int8" else [codes, scale]
    return (*got, q) if c["rot"] else tuple(got)


def _exact_read(c, s):
    got = []
    for name, out in zip("kv", s["out"]):
        y = out.double()
        for b, (t, n) in enumerate(zip(s["pos"].tolist(), s["counts"].tolist())):
            at = s["table"][b, :-(-(t + n) // c["page"])].long()
            y[b, :, :n] = _exact_pages(s[name], s[name + "s"], at)[:, t:t + n]
        got.append(y)
    return tuple(got)


def _exact_rotary(c, s):
    return tuple(torch.stack([_exact_turn(s[x][b], t, c) for b, t in enumerate(s["pos"].tolist())]) for x in "qk")


def exact(case, seed):
    s = prepare(case, seed)
    return {"decode": _exact_decode, "append": _exact_append, "read": _exact_read,
            "rotary": _exact_rotary}[case["kind"]](case, s)
