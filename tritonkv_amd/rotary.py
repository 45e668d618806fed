"""Rotary positions of queries and keys.

Every cache of this package holds keys as they attend, that is with their
positions.  :func:`apply_rotary` gives queries and keys theirs, in one launch;
:func:`~tritonkv_amd.paged8.paged8_append` can do it on the way into its pages.

A pair ``(a, b)`` of a head's first ``dims`` values turns by ``t = position *
inv_freq[i]``:

    (a, b) -> factor * (a cos t - b sin t, a sin t + b cos t)

Pair i is the values ``(i, i + dims / 2)``, or ``(2i, 2i + 1)`` with
``interleaved``; values past ``dims`` stay as they are.  Angles are worked out modulo whole
turns, in 64-bit integers, for any int32 position, so there is no table and no longest context.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .kernels.fused_decode_attn import _prepared
from .paged16 import _dense_rows, _keep16, _new_rows, _offset, _strides
from .quantize import _require_gpu

DTYPES = (torch.float16, torch.bfloat16, torch.float32)
MAX_HEAD_DIM = 256
MAX_TOKENS = 2 ** 25 - 1  # of a call: its workgroups' threads are counted in 32 bits


def _number(d: dict, kind: str, name: str, default=None) -> float:
    if name not in d and default is None:
        raise ValueError(f"scaling of type {kind!r} needs {name!r}")
    x = float(d.get(name, default))
    if not x > 0 or math.isinf(x):
        raise ValueError(f"scaling: {name} must be positive, got {x}")
    return x


_SCALINGS = {"linear": (), "ntk": (), "llama3": ("low_freq_factor", "high_freq_factor"),
             "yarn": ("beta_fast", "beta_slow", "attention_factor")}


def rotary_frequencies(dims: int, base: float = 10000.0, scaling: dict | None = None) -> tuple:
    """``(frequencies, factor)``: radians per position of the ``dims / 2`` pairs, and what
    multiplies cos and sin.

    Pair i turns by ``base ** (-2 i / dims)``.  ``scaling`` stretches that for contexts longer
    than a model was trained on, by its ``"factor"`` and its ``"type"`` (or ``"rope_type"``):

    * ``{"type": "linear"}``: every frequency divided by the factor;
    * ``{"type": "ntk"}``: ``base * factor ** (dims / (dims - 2))`` as the base, which
      leaves the fastest pair as it is and divides the slowest by the factor;
    * ``{"type": "llama3", "low_freq_factor", "high_freq_factor",
      "original_max_position_embeddings"}``: wavelengths up to ``original / high`` stay,
      those from ``original / low`` on are divided, those between are blended;
    * ``{"type": "yarn", "original_max_position_embeddings"}``, with ``"beta_fast"`` (32)
      and ``"beta_slow"`` (1): pairs that turn more often than beta_fast over the original
      context stay, those that turn less than beta_slow are divided, a ramp over the
      pairs between, and cos and sin take ``"attention_factor"`` (0.1 ln factor + 1).

    Other entries, which would change the angles in ways that these do not know, are refused.
    """
    if dims <= 0 or dims % 2:
        raise ValueError(f"dims must be positive and even, got {dims}")
    if not base > 1 or math.isinf(base):
        raise ValueError(f"base must be over 1, got {base}")
    plain = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if scaling is None:
        return plain, 1.0
    kind = scaling.get("rope_type", scaling.get("type"))
    if scaling.get("type", kind) != kind:
        raise ValueError(f"scaling: type {scaling['type']!r} and rope_type {kind!r}")
    if kind not in _SCALINGS:
        raise ValueError(f"scaling type must be 'linear', 'ntk', 'llama3' or 'yarn', got {kind!r}")
    known = ("type", "rope_type", "factor", "original_max_position_embeddings", *_SCALINGS[kind])
    if any(name not in known for name in scaling):
        raise ValueError(f"scaling of type {kind!r} does not know {[name for name in scaling if name not in known]}")
    factor = _number(scaling, kind, "factor")
    if kind == "linear":
        return [w / factor for w in plain], 1.0
    if kind == "ntk":
        if dims <= 2:
            raise ValueError("scaling of type 'ntk' needs more than 2 dims")
        wide = base * factor ** (dims / (dims - 2))
        return [wide ** (-2.0 * i / dims) for i in range(dims // 2)], 1.0
    original = _number(scaling, kind, "original_max_position_embeddings")
    if kind == "llama3":
        low, high = _number(scaling, kind, "low_freq_factor"), _number(scaling, kind, "high_freq_factor")
        if high <= low:
            raise ValueError(f"scaling: high_freq_factor must be over low_freq_factor, got {high} and {low}")
        kept = [min(1.0, max(0.0, (original * w / (2 * math.pi) - low) / (high - low))) for w in plain]
        return [w * (k + (1 - k) / factor) for w, k in zip(plain, kept)], 1.0

    def pair(turns: float) -> float:  # the pair that makes so many turns over the original context
        return dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    first = max(0, math.floor(pair(_number(scaling, kind, "beta_fast", 32.0))))
    last = min(dims - 1, math.ceil(pair(_number(scaling, kind, "beta_slow", 1.0))))
    ramp = [min(1.0, max(0.0, (i - first) / max(last - first, 1e-3))) for i in range(dims // 2)]
    return ([w * ((1 - x) + x / factor) for w, x in zip(plain, ramp)],
            _number(scaling, kind, "attention_factor", max(1.0, 0.1 * math.log(factor) + 1.0)))


# 1 / (2 pi) as a sum of four numbers of 24 bits, whose products with 26 bits are exact in float64.
_INV_2PI = (0x28be60 * 2.0 ** -24, 0xdb9391 * 2.0 ** -48, 0x054a7f * 2.0 ** -72, 0x09d5f4 * 2.0 ** -96)


def _turns(inv_freq: torch.Tensor) -> torch.Tensor:
    """float64 radians per position as turns in 2**-64, modulo 2**64: where they lie, without a wait."""
    far = inv_freq * 134217729.0  # 2**27 + 1
    high = far - (far - inv_freq)  # the upper 26 bits; the rest has no more
    pieces = torch.stack([high, inv_freq - high])
    parts = torch.stack([pieces * c for c in _INV_2PI])
    upper = (parts - parts.trunc()) * 2.0 ** 32
    lower = (upper - upper.trunc()) * 2.0 ** 32
    return ((upper.to(torch.int64) << 32) + lower.to(torch.int64)).sum((0, 1))


class Rotary:
    """The frequencies of a model's rotary positions, on a device.

    ``dims`` values of a head turn, with the frequencies of :func:`rotary_frequencies`;
    or ``inv_freq``, a tensor of radians per position of each pair, says them outright
    (per-pair factors of a long context are divided into it).  ``factor`` multiplies cos
    and sin (default: what ``scaling`` says, else 1).

    The frequencies are copied and turned into integers here, by some twenty launches: make one per model, and
    where they follow the length, one per length that is met, not one per step.
    """

    def __init__(self, dims: int | None = None, base: float = 10000.0, *, interleaved: bool = False,
                 scaling: dict | None = None, inv_freq: torch.Tensor | None = None, factor: float | None = None,
                 device="cuda"):
        if (dims is None) == (inv_freq is None):
            raise ValueError("give dims, or inv_freq, and not both")
        if inv_freq is None:
            freq, scaled = rotary_frequencies(dims, base, scaling)
            inv_freq = torch.tensor(freq, dtype=torch.float64, device=device)
        else:
            if scaling is not None:
                raise ValueError("scaling is for dims: divide it into inv_freq")
            if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1 or inv_freq.numel() == 0 \
                    or not inv_freq.is_floating_point():
                raise ValueError("inv_freq must be a floating-point tensor of radians per position, one for each pair")
            inv_freq, scaled = inv_freq.detach().to(torch.float64, copy=True).contiguous(), 1.0
        self.inv_freq = inv_freq
        self.turns = _turns(inv_freq)
        self.dims = 2 * inv_freq.numel()
        self.interleaved = bool(interleaved)
        self.factor = float(scaled if factor is None else factor)
        if not math.isfinite(self.factor):
            raise ValueError(f"factor must be finite, got {factor}")


def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and _strides(a, 1) == _strides(b, 1)


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a and b certainly share no memory.  Queries and keys that lie in turn in
    one projection's output do not: over a stride that both have, they keep to other places."""
    if a.numel() == 0 or b.numel() == 0:
        return True

    def extent(t, below):  # bytes from the first entry past the last, over the axes of smaller strides
        return sum((n - 1) * s for n, s in zip(t.shape, t.stride()) if s < below) * t.element_size() + t.element_size()

    a0, b0 = a.data_ptr(), b.data_ptr()
    every = 1 << 62
    if a0 + extent(a, every) <= b0 or b0 + extent(b, every) <= a0:
        return True
    if a.element_size() != b.element_size():
        return False
    size = a.element_size()
    for period in {s for n, s in zip(a.shape, a.stride()) if n > 1} & {s for n, s in zip(b.shape, b.stride()) if n > 1}:
        if period <= 0 or any(s > period and s % period for t in (a, b) for n, s in zip(t.shape, t.stride()) if n > 1):
            continue
        step, between = period * size, (b0 - a0) % (period * size)
        if extent(a, period) <= between and between + extent(b, period) <= step:
            return True
    return False


_R = {f: _offset(_lib.RotaryArgs, f) for f in ("q", "k", "q_out", "k_out", "positions", "turns")}
_APART, _WRITTEN = 2, 4  # flags of a kept call's tensors: apart from written ones; written


def _check_rotary(rotary, D: int, device) -> None:
    if not isinstance(rotary, Rotary):
        raise TypeError(f"rotary must be a Rotary, got {type(rotary).__name__}")
    if rotary.dims > D:
        raise ValueError(f"rotary turns {rotary.dims} values of a head of {D}")
    if rotary.inv_freq.device != device:
        raise ValueError(f"rotary is on {rotary.inv_freq.device}, q on {device}")


def _no_grad(*tensors) -> None:
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise ValueError("a tensor requires grad, which this call does not record: run it under torch.no_grad() "
                         "(apply_rotary's gradient is the same call on the output's gradient with adjoint=True)")


def _out_like(x: torch.Tensor, out, name: str, align: int) -> torch.Tensor:
    if out is None:
        fresh = torch.empty_like(x)
        return fresh if _dense_rows(fresh, align) else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if not isinstance(out, torch.Tensor) or out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{name} must be a {tuple(x.shape)} tensor of {x.dtype} on {x.device}")
    if not _dense_rows(out, align) or any(s <= 0 for s in _strides(out, align)):
        raise ValueError(f"{name} must hold each head's values densely, on 16-byte boundaries")
    return out


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, rotary: Rotary, *,
                 adjoint: bool = False, out=None, _workspace: dict | None = None) -> tuple:
    """Queries and keys turned to their positions, in one launch: ``(q_out, k_out)``.

    q: ``(B, HQ, N, D)`` and k: ``(B, HKV, N, D)`` (None: queries alone), or for one
    token ``(B, HQ, D)`` and ``(B, HKV, D)``; float16, bfloat16 or float32, both alike,
    in any strides (token-major projections are read as they lie).  D is a multiple of
    16, at most 256.  positions: int32, ``(B,)`` for the position of each row's first
    token, or ``(B, N)`` for that of every token; negative ones turn the other way.

    ``adjoint=True`` turns back, which is the gradient's way: the gradient of the
    inputs out of the outputs'.  (With factor 1 it undoes the call.)  ``out``: a pair of
    tensors of q's and k's form for the results; they may be q and k themselves.

    With ``_workspace``, a dict of this call site, a call like the previous one is checked and
    launched natively.  Nothing is synchronised, and with ``out`` nothing allocated.
    """
    _no_grad(q, k)
    key = None
    if _workspace is not None and isinstance(out, (tuple, list)) and len(out) == 2 and isinstance(rotary, Rotary):
        inside = out[0] is q and out[1] is k
        key = ("rotary", bool(adjoint), rotary.factor, rotary.interleaved, inside)
        prep = _prepared(_workspace, key)
        if prep is not None and prep.run(q, k, *out, positions, rotary.turns):
            return out[0], out[1]
    if not isinstance(q, torch.Tensor) or q.dim() not in (3, 4):
        raise ValueError("q must be a (B, HQ, N, D) or (B, HQ, D) tensor")
    if q.dtype not in DTYPES:
        raise TypeError(f"q must be float16, bfloat16 or float32, got {q.dtype}")
    device, short = q.device, q.dim() == 3
    if k is not None and (not isinstance(k, torch.Tensor) or k.dim() != q.dim() or k.shape[0] != q.shape[0]
                          or k.shape[2:] != q.shape[2:]):
        raise ValueError(f"k must have q's rows, tokens and head dim, got {tuple(getattr(k, 'shape', ()))} "
                         f"and {tuple(q.shape)}")
    if k is not None and (k.dtype != q.dtype or k.device != device):
        raise ValueError(f"q and k must have one dtype and device, got {q.dtype} on {device} and {k.dtype} on {k.device}")
    if out is None:
        outs = [None, None]
    elif isinstance(out, (tuple, list)) and len(out) == 2 and (out[1] is None) == (k is None) and out[0] is not None:
        outs = list(out)
    else:
        raise ValueError("out must be a pair of tensors, the second None where k is")
    D = q.shape[-1]
    if D % 16 or not 0 < D <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be a multiple of 16, at most {MAX_HEAD_DIM}, got {D}")
    _check_rotary(rotary, D, device)
    B, N = q.shape[0], 1 if short else q.shape[2]
    if not isinstance(positions, torch.Tensor) or positions.dtype != torch.int32 or positions.device != device \
            or tuple(positions.shape) not in ((B,), (B, N)):
        raise ValueError(f"positions must be an int32 ({B},) or ({B}, {N}) tensor on {device}")
    if B * N > MAX_TOKENS or any(x is not None and x.shape[1] > 65535 for x in (q, k)):
        raise ValueError(f"at most {MAX_TOKENS} tokens and 65535 heads")
    align = 16 // q.element_size()
    outs = [_out_like(x, o, name, align) if x is not None else None
            for x, o, name in ((q, outs[0], "out[0]"), (k, outs[1], "out[1]"))]
    given = [(x, o) for x, o in zip((q, k), outs) if x is not None]
    for i, (x, o) in enumerate(given):
        if not _same_place(x, o) and not _apart(x, o):
            raise ValueError("an output must be its input itself or share no memory with it")
        if not all(_apart(o, t) for t in (*(t for pair in given[i + 1:] for t in pair), positions,
                                          rotary.turns, *(y for y, _ in given[:i]))):
            raise ValueError("an output must not share memory with the other tensors")
    _require_gpu(q, "apply_rotary")
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return outs[0], outs[1]
    if q.shape[1] == 0 or (k is not None and k.shape[1] == 0):
        raise ValueError("q and k must have heads")
    read = [None if x is None else _new_rows(x) for x in (q, k)]

    def strides(t):
        if t is None:
            return (0, 0, 0)
        s = _strides(t, align)
        return (s[0], s[1], align) if short else s

    args = _lib.RotaryArgs(
        q=read[0].data_ptr(), k=_lib.ptr(read[1]), q_out=outs[0].data_ptr(), k_out=_lib.ptr(outs[1]),
        q_strides=strides(read[0]), k_strides=strides(read[1]), q_out_strides=strides(outs[0]),
        k_out_strides=strides(outs[1]), positions=positions.data_ptr(),
        position_strides=(positions.stride(0), positions.stride(1) if positions.dim() == 2 else 0),
        turns=rotary.turns.data_ptr(), factor=rotary.factor, position_step=int(positions.dim() == 1),
        x_type=DTYPES.index(q.dtype), interleaved=int(rotary.interleaved), adjoint=int(adjoint), B=B, HQ=q.shape[1],
        HKV=0 if k is None else k.shape[1], N=N, D=D, dims=rotary.dims)
    _lib.check(_lib.launch(device, "tkv_rotary", args), "apply_rotary")
    if key is not None and read[0] is q and read[1] is k:
        # In place q and k are what is written; the outputs, the same tensors, need not lie apart from them.
        read, written = (_WRITTEN, 0) if inside else (_APART, _WRITTEN)
        _keep16(_workspace, key, args, "tkv_rotary", "apply_rotary", device, (),
                ((q, _R["q"], 16, 1 | read), (k, _R["k"], 16, 1 | read), (outs[0], _R["q_out"], 16, 1 | written),
                 (outs[1], _R["k_out"], 16, 1 | written), (positions, _R["positions"], 4, 1 | _APART),
                 (rotary.turns, _R["turns"], 8, _APART)))
    return outs[0], outs[1]


__all__ = ["Rotary", "apply_rotary", "rotary_frequencies"]
