"""The 8-bit page operators and rotary positions in 64 bits, one token at a time, on the CPU."""

from __future__ import annotations

import math

import torch

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
TOP = {E4M3: 448.0, INT8: 127.0}


def need(top: float, code) -> float:
    """The least power of two s, at least 2**-64, with top <= TOP * s."""
    s = 2.0 ** -64
    while top > TOP[code] * s:
        s *= 2.0
    return s


def nearest(y: torch.Tensor, code) -> torch.Tensor:
    """The numbers nearest to y (float64, |y| <= TOP) that codes hold, to even."""
    if code is INT8:
        return torch.round(torch.nan_to_num(y, nan=0.0))
    mag = y.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(mag)) - 3)
    return torch.round(y / step) * step


def clamped(x: torch.Tensor) -> torch.Tensor:
    return x.clamp(-2.0 ** 64, 2.0 ** 64)


def append(codes, scale, x, table, pos, counts, code, block):
    """codes (P, HKV, page, D) float64 numbers and scale (P, HKV, n) float64, changed in place."""
    P, HKV, page, D = codes.shape
    B, _, N, _ = x.shape
    for b in range(B):
        n = 0
        count = N if counts is None else min(int(counts[b]), N)
        while n < count:
            t = int(pos[b]) + n
            left = min(block - t % block, count - n) if t >= 0 else min(-t, count - n)
            if 0 <= t < table.shape[1] * page:
                p = int(table[b, t // page])
                if 0 <= p < P:
                    i, first = (t % page) // block, t % block
                    at = t % page - first
                    for h in range(HKV):
                        y = clamped(x[b, h, n:n + left])
                        s = need(float(torch.nan_to_num(y.abs(), nan=0.0).max()), code)
                        had = float(scale[p, h, i])
                        if first and 0 < had < math.inf:
                            if s > had:
                                old = codes[p, h, at:at + first]
                                codes[p, h, at:at + first] = nearest(old * (had / s), code)
                            s = max(s, had)
                        scale[p, h, i] = s
                        codes[p, h, at + first:at + first + left] = nearest(y / s, code)
            n += left


def turn(x, t, w, interleaved=False, factor=1.0, adjoint=False):
    """x (..., N, D) float64, t (..., N) positions broadcast against x's leading axes."""
    n = w.numel()
    ang = t.double()[..., None] * w * (-1.0 if adjoint else 1.0)
    c, s = factor * torch.cos(ang), factor * torch.sin(ang)
    y = x.clone()
    first = torch.arange(n) * 2 if interleaved else torch.arange(n)
    second = first + 1 if interleaved else first + n
    a, b = x[..., first], x[..., second]
    y[..., first] = a * c - b * s
    y[..., second] = a * s + b * c
    return y


def rows_of(codes, scale, table, b, L):
    """Row b's first L tokens, (HKV, L, D) float64."""
    P, HKV, page, D = codes.shape
    block = page // scale.shape[2]
    out = torch.zeros(HKV, L, D, dtype=torch.float64)
    for t in range(0, L, block):
        p = min(max(int(table[b, t // page]), 0), P - 1)
        m, s = min(block, L - t), t % page
        out[:, t:t + m] = codes[p, :, s:s + m].double() * scale[p, :, s // block].double()[:, None, None]
    return out


def decode(q, k, v, table, lens, counts, sm_scale):
    """q (B, HQ, M, D); k, v: (codes, scale).  out, lse, and how far a kernel may be off each.

    Bounds: products of fp16 queries and codes are exact in fp32, their sum over D is off by D 2^-24 of
    the sum of magnitudes, the factors, the exponential and P's two fp16 terms by 2^-21 of p
    together, the sums over tokens by 2^-24 for each of the chunks a wave and a join add up."""
    B, HQ, M, D = q.shape
    HKV = k[0].shape[1]
    G = HQ // HKV
    out = torch.zeros(B, HQ, M, D, dtype=torch.float64)
    lse = torch.full((B, HQ, M), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(B):
        L = int(lens[b])
        ask = M if counts is None else max(0, min(int(counts[b]), M))
        if L == 0 or ask == 0:
            continue
        kr, vr = rows_of(*k, table, b, L), rows_of(*v, table, b, L)
        for h in range(HQ):
            for m in range(ask):
                n = L - (ask - 1 - m)
                if n <= 0:
                    continue
                kk, vv, qq = kr[h // G, :n], vr[h // G, :n], q[b, h, m].double()
                x = (kk * qq).sum(-1) * sm_scale
                top = (kk * qq).abs().sum(-1) * abs(sm_scale)
                p = torch.softmax(x, -1)
                out[b, h, m] = p @ vv
                lse[b, h, m] = torch.logsumexp(x, -1)
                d = (D + 8) * 2.0 ** -24 * float(torch.nan_to_num(top).max()) + 2.0 ** -21
                sums = (n / 32 + 64) * 2.0 ** -24
                tol[b, h, m] = (2 * d + sums) * (p @ vv.abs())
                ltol[b, h, m] = d + sums + 2.0 ** -22 * abs(float(lse[b, h, m]))
    return out, lse, tol, ltol


def assert_within(got, want, tol, what=""):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), f"{what}: infinities in other places"
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()]), what
    over = ((got - want).abs() - tol)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, \
        f"{what}: {float((got - want).abs()[fin].max())} off, bound passed by {float(over.max())}"


def make_pool(P, HKV, page, D, code, block, seed, device="cuda", spread=True):
    """A Paged8Pool of random codes; scales are powers of two around 2^-6."""
    from tritonkv_amd.paged8 import empty_paged8_pool

    g = torch.Generator().manual_seed(seed)
    pool = empty_paged8_pool(P, HKV, page, D, code, block, device=device)
    x = torch.randn(P, HKV, page, D, generator=g, dtype=torch.float64) * (100.0 if code is E4M3 else 40.0)
    c = nearest(x.clamp(-TOP[code], TOP[code]), code)
    pool.codes.copy_(c.to(torch.float32).to(code))
    e = torch.randint(-8, -4, pool.scale.shape, generator=g) if spread else torch.full(pool.scale.shape, -6)
    pool.scale.copy_(torch.exp2(e.double()).float())
    return pool


def numbers(pool):
    """A pool's codes as float64 numbers and its scales, on the CPU."""
    return pool.codes.cpu().float().double(), pool.scale.cpu().double()


def make_table(B, width, P, seed, need_pages=None):
    """Distinct pages in no order; -1 past a row's pages."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(P, generator=g).to(torch.int32)
    t = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        n = width if need_pages is None else need_pages[b]
        t[b, :n] = order[at:at + n]
        at += n
    return t
