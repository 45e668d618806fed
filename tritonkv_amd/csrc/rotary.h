// Rotary positions: pairs (a, b) of a head's first `dims` values turn by an angle
// theta = position * inv_freq[pair],
//
//   (a, b) -> factor * (a cos(theta) - b sin(theta), a sin(theta) + b cos(theta)),
//
// pairs of the values (i, i + dims / 2) or, interleaved, (2i, 2i + 1); values past
// `dims` pass through.
#pragma once

#include "tkv_device.h"

namespace tkv {

// The angle is taken in 64 bits, as quarter turns less whole turns: a position of 2^20 times a
// frequency of 1 would be 0.06 radians off in 32.  What remains, at most a
// half of a quarter turn, is exact to 2^-25 of itself in 32 bits.
__device__ __forceinline__ float2 turn_of(double position, double inv_freq) {
  double v = position * inv_freq * 0.15915494309189535;  // turns
  v = 4.0 * (v - __builtin_rint(v));
  const double k = __builtin_rint(v);
  const float x = (float)(v - k) * 1.5707963267948966f;  // within pi / 4
  // Taylor's series: the first terms left out are x^11 / 11! and x^12 / 12!, under 2e-9.
  const float z = x * x;
  float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(z, s, 8.3333333e-3f);
  s = fmaf(z, s, -1.6666667e-1f);
  s = fmaf(z * x, s, x);
  float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(z, c, -1.3888889e-3f);
  c = fmaf(z, c, 4.1666667e-2f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.0f);
  const int quarter = (int)k & 3;
  const float sn = quarter & 1 ? c : s, cs = quarter & 1 ? s : c;
  return make_float2(quarter == 1 || quarter == 2 ? -cs : cs, quarter & 2 ? -sn : sn);
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

// Eight values at p, which is on 16 bytes.
template <int T>
__device__ __forceinline__ void load8(const void* p, float* y) {
  if constexpr (T == kF32) {
    const f4 a = *static_cast<const f4*>(p), b = *(static_cast<const f4*>(p) + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = a[i], y[4 + i] = b[i];
  } else {
    const u4 w = *static_cast<const u4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = T == kF16 ? half_lo(w[i]) : __builtin_bit_cast(float, w[i] << 16);
      y[2 * i + 1] = T == kF16 ? half_hi(w[i]) : __builtin_bit_cast(float, w[i] & 0xffff0000u);
    }
  }
}
template <int T>
__device__ __forceinline__ void store8(void* p, const float* y) {
  if constexpr (T == kF32) {
    *static_cast<f4*>(p) = f4{y[0], y[1], y[2], y[3]};
    *(static_cast<f4*>(p) + 1) = f4{y[4], y[5], y[6], y[7]};
  } else {
    u4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = T == kF16 ? pack_h2(y[2 * i], y[2 * i + 1]) : pack_bf2(y[2 * i], y[2 * i + 1]);
    *static_cast<u4*>(p) = w;
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

// How a head's 16 values of item e (of D / 16) lie: at two places of 8, `first` and `second`.
// Item e of the halves' layout holds 8 pairs, the others 16 neighbours.
struct Places {
  int first, second;
  __device__ __forceinline__ Places(int e, int dims, bool interleaved) {
    const bool halves = !interleaved && 16 * e < dims;
    first = halves ? 8 * e : 16 * e;
    second = halves ? 8 * e + dims / 2 : 16 * e + 8;
  }
};

// Turns the 16 values of an item, whose turns come from at(pair) (factor and direction included).
template <class At>
__device__ __forceinline__ void turn16(float* y, int e, int dims, bool interleaved, At at) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (8 * e + i < dims / 2) {
        const float2 t = at(8 * e + i);
        turn_pair(y[2 * i], y[2 * i + 1], t.x, t.y);
      }
  } else if (16 * e < dims) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 t = at(8 * e + i);
      turn_pair(y[i], y[8 + i], t.x, t.y);
    }
  }
}

// ---------------------------------------------------------------------------
// Tokens turned by a workgroup of THREADS: `tokens` of them from flat token `from` (row
// token / N, token % N) on, all H heads.  lds: tokens * dims / 2 turns.
// ---------------------------------------------------------------------------
struct TurnRows {
  const void* x;
  void* out;
  int64_t xs[3], outs[3];  // strides in elements: batch, head, token
  int H;
  bool heads_first;        // a token's heads lie nearer than a head's tokens
};

struct TurnPlan {
  const int32_t* positions;
  int64_t position_strides[2];  // batch, token
  int position_step;            // added per token
  const int32_t* counts;        // a row's live tokens, or null
  const double* inv_freq;
  float factor;                 // of cos; of sin with the direction's sign:
  float sin_factor;
  int interleaved, dims, D, N, B;
};

template <int THREADS>
__device__ __forceinline__ void make_turns(const TurnPlan& p, uint32_t from, int tokens, float2* lds) {
  const uint32_t pairs = (uint32_t)p.dims / 2, total = (uint32_t)tokens * pairs;
  for (uint32_t u = threadIdx.x; u < total; u += THREADS) {
    const uint32_t i = u / pairs, pair = u - i * pairs, token = from + i, b = token / (uint32_t)p.N,
                   n = token - b * (uint32_t)p.N;
    const int64_t pos = (int64_t)p.positions[b * p.position_strides[0] + n * p.position_strides[1]] +
                        (int64_t)p.position_step * n;
    const float2 t = turn_of((double)pos, p.inv_freq[pair]);
    lds[u] = make_float2(t.x * p.factor, t.y * p.sin_factor);
  }
}

// VEC: halves of whole groups of 8 (or interleaved pairs); else a thread takes a pair.
template <int T, bool VEC, int THREADS>
__device__ __forceinline__ void turn_tokens(const TurnPlan& p, const TurnRows& r, uint32_t from, int tokens,
                                            const float2* lds) {
  const uint32_t pairs = (uint32_t)p.dims / 2, per = (uint32_t)p.D / (VEC ? 16 : 2), H = r.H, total = per * H * tokens;
  for (uint32_t u = threadIdx.x; u < total; u += THREADS) {
    const uint32_t rest = u / per, e = u - rest * per;
    uint32_t i, h;
    if (r.heads_first) {
      i = rest / H;
      h = rest - i * H;
    } else {
      h = rest / (uint32_t)tokens;
      i = rest - h * (uint32_t)tokens;
    }
    const uint32_t token = from + i, b = token / (uint32_t)p.N, n = token - b * (uint32_t)p.N;
    if (p.counts && (int)n >= p.counts[b]) continue;
    const int64_t in = b * r.xs[0] + h * r.xs[1] + n * r.xs[2], out = b * r.outs[0] + h * r.outs[1] + n * r.outs[2];
    const float2* turns = lds + i * pairs;
    if constexpr (VEC) {
      float y[16];
      const Places at((int)e, p.dims, p.interleaved);
      const char* x = static_cast<const char*>(r.x) + in * kBytes<T>;
      char* o = static_cast<char*>(r.out) + out * kBytes<T>;
      load8<T>(x + at.first * kBytes<T>, y);
      load8<T>(x + at.second * kBytes<T>, y + 8);
      turn16(y, (int)e, p.dims, p.interleaved, [&](int pair) { return turns[pair]; });
      store8<T>(o + at.first * kBytes<T>, y);
      store8<T>(o + at.second * kBytes<T>, y + 8);
    } else {
      const bool turned = e < pairs;
      const int first = turned && !p.interleaved ? (int)e : (int)(2 * e),
                second = turned && !p.interleaved ? (int)(e + pairs) : (int)(2 * e + 1);
      float a = load1<T>(r.x, in + first), c = load1<T>(r.x, in + second);
      if (turned) turn_pair(a, c, turns[e].x, turns[e].y);
      store1<T>(r.out, out + first, a);
      store1<T>(r.out, out + second, c);
    }
  }
}

}  // namespace tkv
