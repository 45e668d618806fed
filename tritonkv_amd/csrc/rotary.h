// Rotary positions: pairs (a, b) of a head's first `dims` values turn by an angle
// theta = position * frequency[pair],
//
//   (a, b) -> factor * (a cos(theta) - b sin(theta), a sin(theta) + b cos(theta)),
//
// pairs of the values (i, i + dims / 2) or, interleaved, (2i, 2i + 1); values past
// `dims` pass through.
#pragma once

#include "tkv_device.h"

namespace tkv {

// A frequency is turns per position in units of 2^-64, so that the product with a position,
// which wraps at whole turns, is exact to 2^-32 of a turn at any position: in 32-bit floats the
// angle of position 2^20 at a frequency of 1 would be 0.06 radians off.  Cosine and sine, times
// `factor` and `sin_factor`, are rounded once: the angle is kept as x + xl, 24 bits and what stands behind
// them, and the series' terms after the first are added to what the first one's rounding left (0.72 * 2^-24 off at
// most over 4 million angles, 0.246 in the mean square, where values rounded once from 64 bits have 0.244; on
// x alone it was 1.6 and 0.34).
__device__ __forceinline__ float2 turn_of(int64_t position, uint64_t frequency, float factor, float sin_factor) {
  const uint32_t p = (uint32_t)position, w0 = (uint32_t)frequency, w1 = (uint32_t)(frequency >> 32);
  const uint32_t t = p * w1 + __umulhi(p, w0) + (uint32_t)((uint64_t)position >> 32) * w0;
  const uint32_t quarter = (t + 0x20000000u) >> 30;
  const int n = (int)(t - (quarter << 30));
  constexpr float kAngle = 1.4629180792671596e-9f;  // 2 pi / 2^32, and what its 24 bits leave
  constexpr float kAngleRest = (float)(1.4629180792671596e-9 - (double)kAngle);
  const float nh = (float)n, nl = (float)(n - (int)nh);
  const float x = nh * kAngle;  // within pi / 4
  const float xl = fmaf(nh, kAngle, -x) + fmaf(nh, kAngleRest, nl * kAngle);
  // Taylor's series: the first terms left out are x^11 / 11! and x^12 / 12!, under 2e-9.
  const float z = x * x, w = fmaf(-0.5f, z, 1.0f);
  float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(z, s, 8.3333333e-3f);
  s = fmaf(z, s, -1.6666667e-1f);
  s = fmaf(x * z, s, xl * w);  // sine less x
  float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(z, c, -1.3888889e-3f);
  c = fmaf(z, c, 4.1666667e-2f);
  c = fmaf(z * z, c, fmaf(-0.5f, z, 1.0f - w) - fmaf(x, xl, 0.5f * fmaf(x, x, -z)));  // cosine less w
  const float sn = quarter & 1 ? w : x, sn_rest = quarter & 1 ? c : s;
  const float cs = quarter & 1 ? x : w, cs_rest = quarter & 1 ? s : c;
  const float fc = (quarter + 1) & 2 ? -factor : factor, fs = quarter & 2 ? -sin_factor : sin_factor;
  return make_float2(fmaf(cs, fc, cs_rest * fc), fmaf(sn, fs, sn_rest * fs));
}

// ---------------------------------------------------------------------------
// Values of the three types, in 32 bits.
// ---------------------------------------------------------------------------
enum { kF16 = 0, kBf16 = 1, kF32 = 2 };

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));

template <int T>
constexpr int kBytes = T == kF32 ? 4 : 2;

__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
  const bf2 v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}

// Eight values as they lie at an address on 16 bytes.  NT: past the caches, for streams.
template <int T>
struct Raw8 {
  u4 w[kBytes<T> / 2];
  template <bool NT>
  __device__ __forceinline__ void load(const void* p) {
#pragma unroll
    for (int i = 0; i < kBytes<T> / 2; ++i) {
      const u4* const at = static_cast<const u4*>(p) + i;
      w[i] = NT ? __builtin_nontemporal_load(at) : *at;
    }
  }
  __device__ __forceinline__ void values(float* y) const {
    if constexpr (T == kF32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t v = w[i / 4][i % 4];
        y[i] = __builtin_bit_cast(float, v);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[2 * i] = T == kF16 ? half_lo(w[0][i]) : __builtin_bit_cast(float, w[0][i] << 16);
        y[2 * i + 1] = T == kF16 ? half_hi(w[0][i]) : __builtin_bit_cast(float, w[0][i] & 0xffff0000u);
      }
    }
  }
};
template <bool NT, class V>
__device__ __forceinline__ void put(void* p, V v) {
  if constexpr (NT) __builtin_nontemporal_store(v, static_cast<V*>(p));
  else *static_cast<V*>(p) = v;
}
template <int T, bool NT>
__device__ __forceinline__ void store8(void* p, const float* y) {
  if constexpr (T == kF32) {
    put<NT>(p, f4{y[0], y[1], y[2], y[3]});
    put<NT>(static_cast<char*>(p) + 16, f4{y[4], y[5], y[6], y[7]});
  } else {
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = T == kF16 ? pack_h2(y[2 * i], y[2 * i + 1]) : pack_bf2(y[2 * i], y[2 * i + 1]);
    put<NT>(p, w);
  }
}
template <int T>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (T == kF32) return static_cast<const float*>(p)[i];
  if constexpr (T == kF16) return (float)static_cast<const _Float16*>(p)[i];
  return __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}
template <int T>
__device__ __forceinline__ void store1(void* p, int64_t i, float y) {
  if constexpr (T == kF32) static_cast<float*>(p)[i] = y;
  if constexpr (T == kF16) static_cast<_Float16*>(p)[i] = (_Float16)y;
  if constexpr (T == kBf16) static_cast<uint16_t*>(p)[i] = (uint16_t)pack_bf2(y, y);
}

__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
  const float x = a;
  a = x * c - b * s;
  b = x * s + b * c;
}

// Item e of a head's D / 16 is the values from place(e) on and those from place(e) + far on, 8 each:
// neighbouring items read neighbouring 16 bytes.  far is half of what turns, whose pairs then
// lie in one item (the halves' layout, dims a multiple of 16), half of the rest, or half of the head
// (interleaved pairs).
struct Places {
  int first, second;
  __device__ __forceinline__ Places(int e, int dims, bool interleaved, int D) {
    if (interleaved) dims = 0;
    const bool turned = 16 * e < dims;
    const int rest = D - dims;
    first = turned ? 8 * e : dims + 8 * (e - dims / 16);
    second = first + (turned ? dims / 2 : rest / 2);
  }
};

// The turns of an item's 8 pairs, and the item turned by them.  Interleaved: 4 pairs of the
// first place, 4 of the second.  Pairs past `dims` are left alone.
struct Turns {
  float2 of[8];
  uint32_t mask;  // a bit for each pair that turns
  // The item's pairs, those that do not turn as pair 0.
  __device__ __forceinline__ void pick(int e, int dims, bool interleaved, int D, int* pairs) {
    mask = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pair = interleaved ? 4 * e + (i & 3) + (i >> 2) * (D / 4) : 8 * e + i;
      const bool turns = pair < dims / 2;
      mask |= turns ? 1u << i : 0u;
      pairs[i] = turns ? pair : 0;
    }
  }
  template <bool INTER>
  __device__ __forceinline__ void turn(float* y) const {
    if constexpr (INTER) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float a = y[2 * i], b = y[2 * i + 1];
        turn_pair(a, b, of[i].x, of[i].y);
        y[2 * i] = mask >> i & 1 ? a : y[2 * i];
        y[2 * i + 1] = mask >> i & 1 ? b : y[2 * i + 1];
      }
    } else if (mask) {  // all of the item's pairs turn
#pragma unroll
      for (int i = 0; i < 8; ++i) turn_pair(y[i], y[8 + i], of[i].x, of[i].y);
    }
  }
};

// ---------------------------------------------------------------------------
// Tokens turned by a workgroup: its turns go to LDS once, then a thread takes an item of a
// token and walks over heads, with the item's turns in registers.
// ---------------------------------------------------------------------------
struct TurnRows {
  const void* x;
  void* out;
  int64_t xs[3], outs[3];  // strides in elements: batch, head, token
  int H;
};

struct TurnPlan {
  const int32_t* positions;
  int64_t position_strides[2];  // batch, token
  int position_step;            // added per token
  const int32_t* counts;        // a row's live tokens, or null
  const uint64_t* turns;        // of a position, for each pair, in 2^-64
  float factor;                 // of cos; of sin with the direction's sign:
  float sin_factor;
  int interleaved, dims, D;
};

// The position of a row's token n.
__device__ __forceinline__ int64_t position_of(const TurnPlan& p, int b, int n) {
  return (int64_t)p.positions[b * p.position_strides[0] + n * p.position_strides[1]] + (int64_t)p.position_step * n;
}

// Tokens of 256 threads: few, so that it reads a token's heads together, but not one, whose
// turns would be all of a thread's start (4 x 8213 tokens, 32 + 8 heads, bf16, us at 1 / 2 / 4 / 8 /
// 16 / 32 tokens: 145 / 115 / 114 / 118 / 135 / 171).
constexpr int kTurnTile = 4;
// Tokens from which on there are workgroups enough for that (one / several tokens a workgroup, 32 + 8 heads of
// 128 dims, us: 2048 tokens 10.2 / 10.0, 4096 16.4 / 17.1, 6144 27.2 / 24.2, 16384 63 / 58; 1024 of one token
// 6.9 / 7.6; an append of 1024-token prompts gains from 1024 tokens on, 12.6 / 11.1).
constexpr int64_t kTurnMany = 4096;
// Up to here the heads are shared out over workgroups too (shared / not, us: 1 to 16 tokens of 128 + 16 heads 3.4 /
// 4.5, 64 4.0 / 4.8, 256 6.5 / 6.9, 500 10.2 / 8.8; of 32 + 8 heads 16 3.4 / 3.6, 256 4.1 / 3.9, 500 4.8 / 4.6,
// 1024 8.2 / 6.9).
constexpr int64_t kTurnFew = 384;

// Heads that a thread has under way at once.  (Four: 113 us for 115 of the case above, but more
// registers than the append's own work needs: 4 x 2049 tokens with rotary 42.7 us against 36.5.)
constexpr int kTurnHeads = 2;

// Tokens i < tokens, which lie at (row, token) = token(i), of the heads part, part + parts, ... (in
// strides of the heads that the workgroup's threads hold at once) of q and then k.
// lds: tokens * dims / 2 turns.  tokens times the items of a head is at most the threads.
// VEC: halves of whole groups of 8 (or INTERleaved pairs); else an item is a pair (of halves).
template <int T, bool VEC, bool INTER, bool NT, class Token>
__device__ __forceinline__ void turn_tokens(const TurnPlan& p, const TurnRows& q, const TurnRows& k, int tokens,
                                            int part, int parts, float2* lds, Token token) {
  const int threads = (int)blockDim.x, tid = (int)threadIdx.x;
  const int pairs = p.dims / 2, per = p.D / (VEC ? 16 : 2), slots = tokens * per, lanes = threads / slots;
  for (int u = tid; u < tokens * pairs; u += threads) {
    const int i = u / pairs, pair = u - i * pairs;
    const int2 at = token(i);
    lds[u] = turn_of(position_of(p, at.x, at.y), p.turns[pair], p.factor, p.sin_factor);
  }
  __syncthreads();
  const int lane = tid / slots, slot = tid - lane * slots, i = slot / per, e = slot - i * per;
  if (lane >= lanes) return;
  const int2 at = token(i);
  if (p.counts && at.y >= p.counts[at.x]) return;
  const float2* const turns = lds + i * pairs;
  const int heads = q.H + k.H, step = lanes * parts;
  auto rows = [&](int h, const char*& x, char*& o) {
    const TurnRows& r = h < q.H ? q : k;
    const int g = h < q.H ? h : h - q.H;
    x = static_cast<const char*>(r.x) + (at.x * r.xs[0] + g * r.xs[1] + at.y * r.xs[2]) * kBytes<T>;
    o = static_cast<char*>(r.out) + (at.x * r.outs[0] + g * r.outs[1] + at.y * r.outs[2]) * kBytes<T>;
  };
  if constexpr (VEC) {
    const Places pl(e, p.dims, INTER, p.D);
    Turns my;
    int pair[8];
    my.pick(e, p.dims, INTER, p.D, pair);
#pragma unroll
    for (int n = 0; n < 8; ++n) my.of[n] = turns[pair[n]];
    constexpr int HEADS = kTurnHeads;
    for (int h0 = lane + lanes * part; h0 < heads; h0 += step * HEADS) {
      Raw8<T> a[HEADS], b[HEADS];
      char* o[HEADS];
#pragma unroll
      for (int n = 0; n < HEADS; ++n) {
        const int h = h0 + n * step;
        if (h >= heads) break;
        const char* x;
        rows(h, x, o[n]);
        a[n].template load<NT>(x + pl.first * kBytes<T>);
        b[n].template load<NT>(x + pl.second * kBytes<T>);
      }
#pragma unroll
      for (int n = 0; n < HEADS; ++n) {
        if (h0 + n * step >= heads) break;
        float y[16];
        a[n].values(y);
        b[n].values(y + 8);
        my.turn<INTER>(y);
        store8<T, NT>(o[n] + pl.first * kBytes<T>, y);
        store8<T, NT>(o[n] + pl.second * kBytes<T>, y + 8);
      }
    }
  } else {
    const bool turned = e < pairs;
    const int first = turned ? e : 2 * e, second = turned ? e + pairs : 2 * e + 1;
    const float2 t = turned ? turns[e] : make_float2(1.0f, 0.0f);
    for (int h = lane + lanes * part; h < heads; h += step) {
      const char* x;
      char* o;
      rows(h, x, o);
      float a = load1<T>(x, first), c = load1<T>(x, second);
      if (turned) turn_pair(a, c, t.x, t.y);
      store1<T>(o, first, a);
      store1<T>(o, second, c);
    }
  }
}

}  // namespace tkv
