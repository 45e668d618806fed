// An 8-bit paged cache for gfx950: attention of a row's last tokens over it, the append
// that quantizes tokens into it, and its tokens back as values.
//
// A pool holds codes, e4m3 (largest 448) or int8 (largest 127), and a scale for every
// block of 32, 64 or 128 tokens of a page and KV head: value = code * scale.  With L_b
// tokens in row b, c_b of them asking (the last ones),
//
//   out[b, h, m] = sum_t p_t v_t / sum_t p_t,  p_t = exp(sm_scale q[b, h, m] . k_t - max),
//   lse[b, h, m] = max + log sum_t p_t,        t < L_b - (c_b - 1 - m),  m < c_b.
//
// The decode reads every live token's K and V row (2 * D bytes per token and KV head)
// once for every block of up to 32 queries of a KV head, for 4 * D * G * M flops, so HBM
// bounds it for G * M up to 32.  Layout and split are the 16-bit pages' (paged16.hip): a
// workgroup takes a share of the batch's tokens for one KV head, each of its four waves
// walks 32-token chunks as two 16-row MFMA tiles, scores are S^T = K Q^T, whose
// accumulator layout is the B operand layout of O^T = V^T P^T.
//
// Precision: codes are exact in fp16, so both products run on the fp16 MFMA.  bf16 queries are
// scaled by a power of two each, so that their largest value lies in [2^14, 2^15):
// exact for what is over 2^-30 of it.  P enters as two fp16 terms (22 bits).  A block's
// scale of V multiplies its chunks' product in fp32, one of K the scores.
//
// Measured (split kernel, us): 32 rows of 32768, HKV 8, G 4, e4m3 317-325, 6.7 TB/s; 32 rows of
// 1000-16384, HKV 8, G 8, e4m3 94, 6.1 TB/s; 16 rows of 500-8000 with four queries of 64 heads, int8,
// 42: 32 columns a workgroup, bound by the vector units (about 600 instructions a chunk; e4m3 48 in all for
// int8's 49, of 16 columns 43 for 36: its chunk of NaN places holds 13 registers in scratch); one row of
// 505 7.4, four chunks in turn per wave.  The join takes 2-5 us more.
#include <algorithm>

#include "page_shares.h"
#include "rotary.h"

namespace tkv {

// ---------------------------------------------------------------------------
// Codes.
// ---------------------------------------------------------------------------
struct E4m3 {
  static constexpr bool kHasNan = true;
  // Biased exponent of the least scale of a magnitude: a * 2^k with a in [1, 2) fits 448 = 1.75 * 2^8.
  static constexpr int kTop = 8;
  static constexpr uint32_t kTopMantissa = 0x600000;
  // Four codes as fp16 (exact), two to a dword.
  static __device__ __forceinline__ u2 halves(uint32_t w) {
    return u2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
              __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
  }
  static __device__ __forceinline__ void values(uint32_t w, float* y) {
    y[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
    y[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
    y[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
    y[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
  }
  // Four values of at most 448, rounded to nearest even; NaN stays NaN.
  static __device__ __forceinline__ uint32_t codes(const float* y) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  }
};

struct Int8 {
  static constexpr bool kHasNan = false;
  static constexpr int kTop = 6;
  static constexpr uint32_t kTopMantissa = 0x7e0000;
  // 0x64uu is 1024 + u in fp16; u = code + 128.
  static __device__ __forceinline__ u2 halves(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const h2 bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const h2 lo = __builtin_bit_cast(h2, perm(0x64646464u, u, 0x04010400u)) + bias;
    const h2 hi = __builtin_bit_cast(h2, perm(0x64646464u, u, 0x04030402u)) + bias;
    return u2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  }
  static __device__ __forceinline__ void values(uint32_t w, float* y) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (float)(int)(int8_t)(w >> (8 * i));
  }
  // int8 has no NaN: one becomes 0 (as the conversion to an integer does).
  static __device__ __forceinline__ uint32_t codes(const float* y) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)__builtin_rintf(y[i]) & 0xffu) << (8 * i);
    return w;
  }
};

// ---------------------------------------------------------------------------
// The split kernel of the decode.
// ---------------------------------------------------------------------------
struct Paged8Params {
  tkv_paged8_args a;
  int G, cols;     // query heads of a KV head; G * M columns
  float qk_scale;  // sm_scale * log2(e)
  uint32_t k16[3], v16[3];  // the pools' strides in 16 bytes: products of 32 bits by 32
};

constexpr float kShift8 = 14.0f;  // P is scaled by 2^14, clear of fp16's smallest steps

// HT: tiles of 16 columns (a KV head's queries) per workgroup.  MULTI: more than one query per row.
template <class C, int D, int HT, int NW, bool MULTI>
__global__ void __launch_bounds__(NW * 64, D == 256 ? 3 - HT : 4 - HT)
paged8_split_kernel(const int32_t* lens, int B, int S, int workgroups, int least_chunks, int long_workgroups,
                    int long_chunks, Paged8Params prm) {
  constexpr int NKL = D / 64;  // 16-byte loads of a K row's lane
  constexpr int EPL = D / 16;  // V dims per lane (and V MFMAs)
  constexpr int VW = EPL / 4;  // dwords of them
  const tkv_paged8_args& a = prm.a;
  constexpr int QROW = D + 8;  // elements of a query row in LDS: 16 rows meet no bank twice
  constexpr int OROW = D + 4;  // floats of an output row there: 16-byte pieces
  // The queries, their powers of two, then per wave of the merge: rows of OROW floats,
  // maximum and sum of each.
  extern __shared__ float lds_all[];
  uint16_t* const lds_q = reinterpret_cast<uint16_t*>(lds_all);
  float* const lds_qs = lds_all + 8 * HT * QROW;
  float* const lds = lds_qs + 16 * HT;

  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, j = lane >> 4;
  RowLens rows{lens, B, S, lane, 0, 0};
  Shares sh;
  Segment g;
  uint32_t share_end;
  if (!first_segment(SharePlan{lens, B, S, workgroups, least_chunks, long_workgroups, long_chunks}, blockIdx.y, rows, sh,
                     g, share_end))
    return;
  const int hk = blockIdx.x % a.HKV, cb0 = (blockIdx.x / a.HKV) * 16 * HT;
  const int nc = min(16 * HT, prm.cols - cb0), c0 = hk * prm.cols + cb0, HQM = a.HQ * a.M;

  const int64_t kts = a.k_strides[2], vts = a.v_strides[2];
  const uint32_t kspan = (uint32_t)(31 * kts + D), vspan = (uint32_t)(31 * vts + D);
  const uint32_t klane = (uint32_t)(r * kts + 16 * j), ktile = (uint32_t)(16 * kts);
  uint32_t vlane[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) vlane[i] = (uint32_t)(slot_token(j, i) * vts + EPL * r);

  // Addresses.  Lane l looks up the wave's chunk l: the table entries, addresses and
  // scales of 64 chunks come from one load each.
  const uint64_t khead = (uint64_t)a.k + 16 * ((uint64_t)hk * prm.k16[1]);
  const uint64_t vhead = (uint64_t)a.v + 16 * ((uint64_t)hk * prm.v16[1]);
  uint64_t kt = 0, vt = 0;      // this lane's chunk
  float kscale = 0, vscale = 0;
  int lo, hi;                   // tokens of the segment
  int entry = 0;
  uint32_t at = 0;
  auto look_up = [&](int c) {   // asks for the table entries from the wave's chunk c on
    const int t = lo + 32 * (w + NW * (c + lane));
    at = 0;
    entry = -1;                 // past the segment: the pool's first chunk, never used
    if (t < hi) {
      const uint32_t pg = (uint32_t)t / (uint32_t)a.page_size;
      at = (uint32_t)t - pg * (uint32_t)a.page_size;
      entry = a.block_table[(int64_t)g.b * a.block_table_stride + pg];
    }
  };
  auto place = [&] {            // and turns them into addresses
    const uint32_t page = min(max(entry, 0), a.num_pages - 1);
    kt = khead + 16 * ((uint64_t)page * prm.k16[0] + (uint64_t)at * prm.k16[2]);
    vt = vhead + 16 * ((uint64_t)page * prm.v16[0] + (uint64_t)at * prm.v16[2]);
    const int64_t i = at / (uint32_t)a.block;
    kscale = a.k_scale[page * a.k_scale_strides[0] + hk * a.k_scale_strides[1] + i * a.k_scale_strides[2]];
    vscale = a.v_scale[page * a.v_scale_strides[0] + hk * a.v_scale_strides[1] + i * a.v_scale_strides[2]];
  };
  auto lane_ptr = [&](uint64_t x, int l) {
    const uint32_t x0 = __builtin_amdgcn_readlane((int)(uint32_t)x, l);
    const uint32_t x1 = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), l);
    return reinterpret_cast<const void*>(((uint64_t)x1 << 32) | x0);
  };
  auto lane_float = [&](float x, int l) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
  };
  u4 kx[2][NKL];
  uint32_t vx[8][VW];
  auto load_k = [&](int c) {
    const rsrc_t rk = make_rsrc(lane_ptr(kt, c & 63), kspan);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int m = 0; m < NKL; ++m) kx[t][m] = buf_u4<kPolF16>(rk, klane + t * ktile + 64 * m);
  };
  auto load_v = [&](int c) {
    const rsrc_t rv = make_rsrc(lane_ptr(vt, c & 63), vspan);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (VW == 4) {
        const u4 x = buf_u4<kPolF16>(rv, vlane[i]);
#pragma unroll
        for (int y = 0; y < 4; ++y) vx[i][y] = x[y];
      } else if constexpr (VW == 2) {
        const u2 x = buf_u2<kPolF16>(rv, vlane[i]);
        vx[i][0] = x[0];
        vx[i][1] = x[1];
      } else {
        vx[i][0] = buf_u32<kPolF16>(rv, vlane[i]);
      }
    }
  };

  int ask;              // tokens of the row that ask
  int seen[HT];         // MULTI: tokens that this lane's columns attend to
  float qs[HT];         // their scores' factor
  // Starts segment g: what its first chunk needs is on its way afterwards.
  auto begin_segment = [&] {
    const int bt = (int)opaque(tid);
    lo = 32 * (int)g.begin;
    hi = min(g.L, 32 * (int)g.end);
    // 8 dims of a column per thread and round, zero past the columns.
    constexpr int QV = 16 * HT * (D / 8), QR = (QV + NW * 64 - 1) / (NW * 64);
    u4 q8[QR];
#pragma unroll
    for (int i = 0; i < QR; ++i) {
      const int u = bt + NW * 64 * i, col = u / (D / 8);
      q8[i] = u4{0u, 0u, 0u, 0u};
      if (col < nc) {
        const int at = cb0 + col, head = MULTI ? at / a.M : at, m = MULTI ? at - head * a.M : 0;
        q8[i] = *reinterpret_cast<const u4*>(static_cast<const uint16_t*>(a.q) + g.b * a.q_strides[0] +
                                             (hk * prm.G + head) * a.q_strides[1] + m * a.q_strides[2] +
                                             8 * (u % (D / 8)));
      }
    }
    look_up(0);
    ask = a.counts ? min(max(a.counts[g.b], 0), a.M) : a.M;
#pragma unroll
    for (int i = 0; i < QR; ++i) {
      const int u = bt + NW * 64 * i, col = u / (D / 8);
      if (a.q_is_bf16) {
        // The column's largest finite magnitude; D / 8 neighbouring lanes hold it.
        float y[8];
        uint32_t top = 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t e0 = q8[i][x] & 0x7fffu, e1 = q8[i][x] >> 16 & 0x7fffu;
          top = max(top, max(e0 < 0x7f80u ? e0 : 0u, e1 < 0x7f80u ? e1 : 0u));
          y[2 * x] = __builtin_bit_cast(float, q8[i][x] << 16);
          y[2 * x + 1] = __builtin_bit_cast(float, q8[i][x] & 0xffff0000u);
        }
#pragma unroll
        for (int x = 1; x < D / 8; x *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, x));
        const int e = (int)(top >> 7) - 127 - 14;  // (a column of zeros: any)
#pragma unroll
        for (int x = 0; x < 4; ++x) q8[i][x] = pack_h2(ldexpf(y[2 * x], -e), ldexpf(y[2 * x + 1], -e));
        if (u % (D / 8) == 0 && u < QV) lds_qs[col] = ldexpf(1.0f, e);
      } else if (u % (D / 8) == 0 && u < QV) {
        lds_qs[col] = 1.0f;
      }
      if (u < QV) *reinterpret_cast<u4*>(lds_q + col * QROW + 8 * (u % (D / 8))) = q8[i];
    }
    place();  // (the queries were made ready while the table was on its way)
    if (lo + 32 * w < hi) {
      load_k(0);
      load_v(0);
    }
    __syncthreads();
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      qs[ht] = lds_qs[16 * ht + r] * prm.qk_scale;
      const int m = (cb0 + 16 * ht + r) % a.M;
      seen[ht] = MULTI && m < ask ? g.L - (ask - 1 - m) : g.L;
    }
  };

  begin_segment();
  for (;;) {
    const int last = hi - 1;
    f4 accv[HT][EPL];
    float m_run[HT], l_run[HT];
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
      for (int mv = 0; mv < EPL; ++mv) accv[ht][mv] = f4{0.f, 0.f, 0.f, 0.f};
      m_run[ht] = -INFINITY;
      l_run[ht] = 0.0f;
    }

    auto step = [&](int c, int cb, auto tail) {
      constexpr bool TAIL = decltype(tail)::value;
      const bool more = cb + 32 * NW < hi;
      const float ks = lane_float(kscale, c & 63), vs = lane_float(vscale, c & 63);
      float x[HT][8], f[HT];  // scores, and what they are in powers of two
      auto hidden = [&](int ht, int i) {
        return TAIL && cb + slot_token(j, i) > (MULTI ? min(last, seen[ht] - 1) : last);
      };
      {
        // (opaque: read again in every chunk, not kept in registers)
        const uint16_t* ql = lds_q + (int)opaque((uint32_t)(r * QROW + 16 * j));
        f4 s[HT][2];
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) s[ht][0] = s[ht][1] = f4{0.f, 0.f, 0.f, 0.f};
        // The dims of step (m, e): 64 m + 16 j + 8 e and the next 7 of lane (r, j), of K and q alike.
#pragma unroll
        for (int m = 0; m < NKL; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            u4 kf[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const u2 h0 = C::halves(kx[t][m][2 * e]), h1 = C::halves(kx[t][m][2 * e + 1]);
              kf[t] = u4{h0[0], h0[1], h1[0], h1[1]};
            }
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) {
              const u4 qf = *reinterpret_cast<const u4*>(ql + 16 * ht * QROW + 64 * m + 8 * e);
#pragma unroll
              for (int t = 0; t < 2; ++t) s[ht][t] = mfma_k32(kf[t], qf, s[ht][t]);
            }
          }
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
          f[ht] = ks * qs[ht];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[ht][i] = s[ht][i / 4][i % 4];
        }
      }
      if (!TAIL && more) {
        if (((c + 1) & 63) == 0) {  // V of chunk c is on its way already, its scale in vs
          look_up(c + 1);
          place();
        }
        load_k(c + 1);
      }
      // Online softmax in base 2; the accumulators are rescaled only in chunks
      // where a column's maximum rose.
      u4 pt[HT][2];
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, hidden(ht, i) ? -INFINITY : x[ht][i] * f[ht]);
        if (__builtin_amdgcn_ballot_w64(top > m_run[ht]) != 0) {
          const float mn = vmax(m_run[ht], xor_max16_32(top));
          const float alpha = safe_exp2_diff(m_run[ht], mn);
          m_run[ht] = mn;
          l_run[ht] *= alpha;
#pragma unroll
          for (int mv = 0; mv < EPL; ++mv) accv[ht][mv] *= alpha;
        }
        // Scores of -inf under a maximum of -inf give p = 0, not NaN.  The product is not rounded
        // before the maximum is off: at scores of 32 and more that alone was 1.3e-6 of p.  (With the shift in the
        // exponent that is rounded to 2^-21 at most, 3.3e-7 of p; a product behind the power, 8 more instructions
        // a tile, would be exact.)
        const float off = kShift8 - (m_run[ht] == -INFINITY ? 0.0f : m_run[ht]);
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = hidden(ht, i) ? 0.0f : __builtin_amdgcn_exp2f(fmaf(x[ht][i], f[ht], off));
          l_run[ht] += p[i];
        }
        // The first term cut, what is left of p, exact, rounded: 2^-22 of p at most, under what the sums in 32
        // bits add.  (Both rounded: 2^-23, outputs as far from 64 bits, 3.16e-7 of the norm for 3.18e-7 at one
        // row of 505, 7.7e-8 for 7.5e-8 at D 64; 16 rows of four queries 48.8 us for 47.7.)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(p[2 * i], p[2 * i + 1]));
          pt[ht][0][i] = hi;
          pt[ht][1][i] = pack_h2(fma_mix_h<false>(hi, -1.0f, p[2 * i]), fma_mix_h<true>(hi, -1.0f, p[2 * i + 1]));
        }
      }
      if constexpr (TAIL) {
        // Rows past the sequence are whatever the page holds there (possibly
        // NaN); p = 0 alone would not cancel them in the MFMA.
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (cb + slot_token(j, i) > last)
#pragma unroll
            for (int e = 0; e < VW; ++e) vx[i][e] = 0u;
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int y = 0; y < VW; ++y)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          // Dims 4 y + 2 z and the next of this lane's: their codes of token pairs, then fp16.
          u4 av[2];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const u2 h = C::halves(perm(vx[2 * i + 1][y], vx[2 * i][y], z ? 0x07030602u : 0x05010400u));
            av[0][i] = h[0];
            av[1][i] = h[1];
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int mv = 4 * y + 2 * z + e;
            u4 iv;  // 1 in the places of NaN, which a column that does not see them takes for 0
            if constexpr (TAIL && MULTI && C::kHasNan) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t n = ((av[e][i] & 0x7fffu) > 0x7c00u ? 0xffffu : 0u) |
                                   ((av[e][i] >> 16 & 0x7fffu) > 0x7c00u ? 0xffff0000u : 0u);
                iv[i] = n & 0x3c003c00u;
                av[e][i] &= ~n;
              }
            }
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) {
              f4 o = mfma_k32(av[e], pt[ht][1], f4{0.f, 0.f, 0.f, 0.f});
              o = mfma_k32(av[e], pt[ht][0], o);
              // V's scale, 0 for a column that sees none of the chunk (a scale of NaN would reach it; opaque:
              // in a register of its own it cost drafts of 32 tokens 3%).
              const float vf = TAIL && MULTI && (int)opaque((uint32_t)seen[ht]) <= cb ? 0.0f : vs;
#pragma unroll
              for (int i = 0; i < 4; ++i) accv[ht][mv][i] = fmaf(o[i], vf, accv[ht][mv][i]);
              if constexpr (TAIL && MULTI && C::kHasNan) {
                u4 sees;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int lim = min(last, seen[ht] - 1);
                  sees[i] = (cb + slot_token(j, 2 * i) <= lim ? 0x3c00u : 0u) |
                            (cb + slot_token(j, 2 * i + 1) <= lim ? 0x3c000000u : 0u);
                }
                const f4 nans = mfma_k32(iv, sees, f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (nans[i] > 0.0f) accv[ht][mv][i] = __builtin_nanf("");
              }
            }
          }
        }
      if (!TAIL && more) load_v(c + 1);
    };

    // Chunks that every column sees whole, then the rest: a wave has at most one of them, since
    // the last kMaxAsk tokens of a row lie in two neighbouring chunks.
    const int full = MULTI ? min(hi, g.L - max(ask, 1) + 1) : hi;
    int c = 0, cb = lo + 32 * w;
    for (; cb + 32 <= full; cb += 32 * NW, ++c) step(c, cb, std::false_type{});
    if (cb < hi) step(c, cb, std::true_type{});

    // Merge of the waves.  (opaque: the addresses of this part would else be kept in
    // registers over the whole loop.)
    const int mr = (int)opaque(r), mj = (int)opaque(j), mt = (int)opaque(tid);
    const int b = g.b, mine_rows = min(16 * HT, prm.cols), asked = ask;
    const int stride = (mine_rows * (OROW + 2) + 3) / 4 * 4;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const float lt = xor_sum16_32(l_run[ht]);
      const int n = mr + 16 * ht;
      if (n >= nc) continue;
      float* mine = lds + w * stride;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int mv = 0; mv < EPL; mv += 4)
          *reinterpret_cast<f4*>(mine + n * OROW + EPL * (4 * mj + i) + mv) =
              f4{accv[ht][mv][i], accv[ht][mv + 1][i], accv[ht][mv + 2][i], accv[ht][mv + 3][i]};
      if (mj == 0) {
        mine[mine_rows * OROW + n] = m_run[ht];
        mine[mine_rows * (OROW + 1) + n] = lt;
      }
    }
    __syncthreads();
    // Where this segment goes.
    const uint32_t l = chunks_of(g.L);
    const bool whole = g.begin == 0 && g.end == l;
    const uint32_t slot = 2 * blockIdx.y + (g.begin == 0 ? 1 : 0);
    if (workgroups && g.begin == 0 && blockIdx.x == 0 && mt == 0)
      reinterpret_cast<int2*>(a.row_pieces)[b] =
          make_int2(blockIdx.y, whole ? 1 : (int)(sh.of(g.at + l - 1) - blockIdx.y + 1));
    // The next segment, whose first loads run behind this one's merge.
    const bool again = g.at + g.end < share_end;
    if (again) {
      g.at += l;
      ++g.b;
      g.L = rows.of(g.b);
      g.begin = 0;
      g.end = min(share_end - g.at, chunks_of(g.L));
      begin_segment();
    }
    for (int idx = mt; idx < nc * (D / 4); idx += NW * 64) {
      const int n = idx / (D / 4), d = 4 * (idx % (D / 4));
      float mw[NW], mstar = -INFINITY;
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        mw[x] = lds[x * stride + mine_rows * OROW + n];
        mstar = fmaxf(mstar, mw[x]);
      }
      f4 o = f4{0.f, 0.f, 0.f, 0.f};
      float ls = 0.0f;
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        // A wave whose scores were all NaN keeps a maximum of -inf and a sum of
        // NaN, which the factor 0 hands on.
        const float f = safe_exp2_diff(mw[x], mstar);
        o += *reinterpret_cast<const f4*>(lds + x * stride + n * OROW + d) * f;
        ls = fmaf(f, lds[x * stride + mine_rows * (OROW + 1) + n], ls);
      }
      if ((cb0 + n) % a.M >= asked) {  // a column of no query
        o = f4{0.f, 0.f, 0.f, 0.f};
        mstar = -INFINITY;
        ls = 0.0f;
      }
      if (whole) {
        store_row4(a.out, a.lse, D, kShift8, (int64_t)b * HQM + c0 + n, d, o, mstar, ls);
      } else {
        const int64_t row = partial_row(HQM, slot, c0 + n);
        *reinterpret_cast<f4*>(a.partials + row * D + d) = o;
        if (d == 0)
          *reinterpret_cast<float2*>(partial_ml(a.partials, workgroups, HQM, D) + 2 * row) = make_float2(mstar, ls);
      }
    }
    if (!again) break;
    __syncthreads();  // the partials in LDS have been read
  }
}

// ---------------------------------------------------------------------------
// Append: token n < counts[b] of row b goes to position positions[b] + n.
//
// A workgroup takes the tokens of one block of the row, of K or V, of a few KV heads in
// turn: a head's values stay in registers from the load over the block's largest magnitude to the
// codes, so each is read and written once, and the turns of its keys are worked out once for
// the heads.  The scale is the least power of two s with |x| <= top * s, or the block's
// own where that is larger: by powers of two nothing is rounded twice in e4m3 (but what
// falls under its smallest normal code), and a scale rises seldom.  Where it rises, the
// codes of the block's earlier tokens are rounded again under the new one.
//
// Bound by HBM (4 x 8213 tokens, counts of half to all, 8 heads, fp16: 151 MB in 29.8 us, 5.1 TB/s; with
// each head's loads behind the one's before 30.4, with 16 neighbouring values to a thread 52), short
// ones by the chain of position, value, scale: 64 rows of a token with rotary 5.5 us.
// ---------------------------------------------------------------------------
struct Append8Params {
  tkv_paged8_append_args a;
  TurnPlan turn;
  TurnRows q;
  uint32_t kv_groups;    // workgroups of K and V per row; those of the queries follow
  int heads;             // of a workgroup of K or V
  int q_tile, q_parts;   // tokens of a workgroup of queries, and the workgroups that share their heads
};

constexpr int kAppendHeads = 2;

constexpr float kLargest = 18446744073709551616.0f;  // 2^64

template <class C>
__device__ __forceinline__ float least_scale(float top) {
  const uint32_t u = __builtin_bit_cast(uint32_t, top);
  const int e = (int)(u >> 23) - C::kTop + ((u & 0x7fffffu) > C::kTopMantissa ? 1 : 0);
  return __builtin_bit_cast(float, (uint32_t)max(e, 127 - 64) << 23);
}

// y / s for n values: by the reciprocal of a power of two, exactly.
template <int N>
__device__ __forceinline__ void over_scale(float* y, float s) {
  const uint32_t u = __builtin_bit_cast(uint32_t, s), e = u >> 23;
  if ((u & 0x7fffffu) == 0 && e > 0 && e < 254) {
    const float inv = __builtin_bit_cast(float, (254 - e) << 23);
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] *= inv;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] /= s;
  }
}

// Whether a scale can be a block's: positive and finite.
__device__ __forceinline__ bool is_scale(float s) { return s > 0.0f && s < INFINITY; }

// The largest of the wave's values, in every lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max_dpp<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v = max_dpp<0x112, 0xF>(v);
  v = max_dpp<0x114, 0xF>(v);
  v = max_dpp<0x118, 0xF>(v);
  v = max_dpp<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v = max_dpp<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// ROT: 0 no rotary positions, 1 by halves, 2 interleaved.
template <class C, int T, int ITEMS, int ROT>
__global__ void __launch_bounds__(1024) paged8_append_kernel(Append8Params prm) {
  const tkv_paged8_append_args& a = prm.a;
  const int D = a.D, PER = D / 16, shift = D == 64 ? 2 : D == 128 ? 3 : 4;  // items of a token's head
  extern __shared__ float2 lds_turns[];
  __shared__ uint32_t tops[kAppendHeads][16];
  const int b = blockIdx.y, tid = threadIdx.x;
  if constexpr (ROT != 0)
    if (blockIdx.x >= prm.kv_groups) {
      const int at = (int)(blockIdx.x - prm.kv_groups), n0 = at / prm.q_parts * prm.q_tile;
      turn_tokens<T, true, ROT == 2, true>(prm.turn, prm.q, TurnRows{}, min(prm.q_tile, a.N - n0), at % prm.q_parts,
                                           prm.q_parts, lds_turns, [&](int i) { return make_int2(b, n0 + i); });
      return;
    }
  const int64_t pos = a.positions[b], room = (int64_t)a.max_pages * a.page_size;
  const int count = a.counts ? min(a.counts[b], a.N) : a.N;
  const uint32_t sets = (uint32_t)((a.HKV + prm.heads - 1) / prm.heads), of = blockIdx.x / (2 * sets),
                 hv = blockIdx.x - of * (2 * sets);
  const bool isv = hv & 1;
  const int h0 = (int)(hv >> 1) * prm.heads, h1 = min(h0 + prm.heads, a.HKV);
  const int64_t begin = max(pos, (int64_t)0), end = min(pos + count, room);
  const int64_t base = (begin / a.block + of) * a.block;  // the block's first position
  const int64_t t0 = max(begin, base), t1 = min(end, base + a.block);
  if (t0 >= t1) return;
  const int rows = (int)(t1 - t0), first = (int)(t0 - base);
  const int64_t* const xs = isv ? a.v_new_strides : a.k_new_strides;
  const char* x = static_cast<const char*>(isv ? a.v_new : a.k_new) +
                  (b * xs[0] + h0 * xs[1] + (t0 - pos) * xs[2]) * kBytes<T>;
  const bool turned = ROT && !isv;
  constexpr bool interleaved = ROT == 2;
  const int dims = turned ? prm.turn.dims : 0;
  // The turns of the thread's items: the frequencies are asked for first, the values next, and while
  // those are on their way the angles are worked out.
  Turns my[ITEMS];
  uint64_t w[ITEMS][8];
  const bool few = blockDim.x == 64;  // few tokens: the angles by all threads, into LDS
  const int pairs = dims / 2;
  if (turned && !few)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int u = tid + i * (int)blockDim.x;
      int pair[8];
      my[i].pick(u & (PER - 1), u >> shift < rows ? dims : 0, interleaved, D, pair);
#pragma unroll
      for (int n = 0; n < 8; ++n) w[i][n] = prm.turn.turns[pair[n]];
    }
  Raw8<T> raw[kAppendHeads][ITEMS][2];
#pragma unroll
  for (int n = 0; n < kAppendHeads; ++n) {  // (under way before the table is known)
    if (h0 + n >= h1) continue;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int u = tid + i * (int)blockDim.x, row = u >> shift, e = u & (PER - 1);
      if (row >= rows) continue;
      const Places pl(e, dims, interleaved, D);
      const char* const at = x + (n * xs[1] + row * xs[2]) * kBytes<T>;
      raw[n][i][0].template load<true>(at + pl.first * kBytes<T>);
      raw[n][i][1].template load<true>(at + pl.second * kBytes<T>);
    }
  }
  const uint32_t pg = (uint32_t)((uint64_t)base / (uint32_t)a.page_size);
  const int page = a.block_table[(int64_t)b * a.block_table_stride + pg];
  const auto turn = [&](int row, uint64_t freq) {
    return turn_of(t0 + row, freq, prm.turn.factor, prm.turn.sin_factor);
  };
  if (turned && few) {
    for (int u = tid; u < rows * pairs; u += 64) lds_turns[u] = turn(u / pairs, prm.turn.turns[u % pairs]);
    __syncthreads();
    int pair[8];
    my[0].pick(tid & (PER - 1), tid >> shift < rows ? dims : 0, interleaved, D, pair);
#pragma unroll
    for (int n = 0; n < 8; ++n) my[0].of[n] = lds_turns[min(tid >> shift, rows - 1) * pairs + pair[n]];
  } else if (turned) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int n = 0; n < 8; ++n) my[i].of[n] = turn((tid + i * (int)blockDim.x) >> shift, w[i][n]);
  }
  if (page < 0 || page >= a.num_pages) return;
  const int at = (int)(base - (int64_t)pg * a.page_size);
  const int64_t* const ss = isv ? a.v_scale_strides : a.k_scale_strides;
  const int64_t* const ps = isv ? a.v_strides : a.k_strides;
  float* sp = (isv ? a.v_scale : a.k_scale) + page * ss[0] + h0 * ss[1] + at / a.block * ss[2];
  uint8_t* to = static_cast<uint8_t*>(isv ? a.v : a.k) + page * ps[0] + h0 * ps[1] + at * ps[2];
#pragma unroll
  for (int n = 0; n < kAppendHeads; ++n, sp += ss[1], to += ps[1]) {
    if (h0 + n >= h1) continue;
    const float held = first ? *sp : 0.0f;
    float y[ITEMS][16];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if ((tid + i * (int)blockDim.x) >> shift >= rows) continue;
      raw[n][i][0].values(y[i]);
      raw[n][i][1].values(y[i] + 8);
      if (turned) my[i].template turn<interleaved>(y[i]);
#pragma unroll
      for (int d = 0; d < 16; ++d) top = fmaxf(top, fabsf(y[i][d]));  // (a NaN does not count)
    }
    uint32_t most = wave_max(__builtin_bit_cast(uint32_t, top));
    if (blockDim.x > 64) {
      uint32_t* const all = tops[n];
      if ((tid & 63) == 0) all[tid >> 6] = most;
      __syncthreads();
      for (int i = 0; i < (int)blockDim.x / 64; ++i) most = max(most, all[i]);
    }
    // Magnitudes past 2^64: in every type, since fp16 holds infinities and a turn's factor may take its
    // keys as far; looked for only where the block's largest is one (for every value of an fp16 prompt
    // 32.2 us against 30.1).
    constexpr uint32_t kMost = __builtin_bit_cast(uint32_t, kLargest);
    if (most > kMost) {
      most = kMost;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int d = 0; d < 16; ++d)  // (comparisons, which leave a NaN as it is)
          y[i][d] = y[i][d] > kLargest ? kLargest : y[i][d] < -kLargest ? -kLargest : y[i][d];
    }
    const bool known = first > 0 && is_scale(held);
    const float need = least_scale<C>(__builtin_bit_cast(float, most)), scale = known ? fmaxf(held, need) : need;
    if (tid == 0) *sp = scale;
    if (known && scale > held) {
      const float ratio = held / scale;
      for (int u = tid; u < first << shift; u += blockDim.x) {
        u4* const p = reinterpret_cast<u4*>(to + (u >> shift) * ps[2] + 16 * (u & (PER - 1)));
        u4 c = *p;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          float z[4];
          C::values(c[d], z);
#pragma unroll
          for (int n = 0; n < 4; ++n) z[n] *= ratio;
          c[d] = C::codes(z);
        }
        *p = c;
      }
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int u = tid + i * (int)blockDim.x, row = u >> shift, e = u & (PER - 1);
      if (row >= rows) continue;
      const Places pl(e, dims, interleaved, D);
      over_scale<16>(y[i], scale);
      uint8_t* const p = to + (first + row) * ps[2];
      __builtin_nontemporal_store(u2{C::codes(y[i]), C::codes(y[i] + 4)}, reinterpret_cast<u2*>(p + pl.first));
      __builtin_nontemporal_store(u2{C::codes(y[i] + 8), C::codes(y[i] + 12)}, reinterpret_cast<u2*>(p + pl.second));
    }
  }
}

// ---------------------------------------------------------------------------
// Read: tokens positions[b] .. positions[b] + counts[b] - 1 of row b as values.
//
// A workgroup takes 32 slots of a page (one block, so that page and scale are the same for all of
// its threads) of K or V, of one or two heads; an item is 16 bytes of output, and a thread asks for
// eight before it writes any.  Workgroups follow each other along the tokens of a head.  Bound by
// HBM: 8 rows of 2000-16384 tokens, 8 heads, bf16, 451 MB in 85.8 us, 5.3 TB/s (heads before
// tokens in the order of workgroups 89, a thread for a token's dims of all heads 87; a place for
// every item 125).
// ---------------------------------------------------------------------------
template <class C, int T, int D>
__global__ void __launch_bounds__(256) paged8_read_kernel(tkv_paged8_read_args a, int heads) {
  constexpr int DIMS = 16 / kBytes<T>, PER = D / DIMS, ITEMS = 32 * PER / 256;
  constexpr int HEADS = ITEMS >= 8 ? 1 : 8 / ITEMS;  // under way at once
  const int b = blockIdx.y;
  const uint32_t sets = (uint32_t)((a.HKV + heads - 1) / heads), blocks = gridDim.x / (2 * sets),
                 hv = blockIdx.x / blocks, of = blockIdx.x - hv * blocks;
  const bool isv = hv & 1;
  const int h0 = (int)(hv >> 1) * heads, h1 = min(h0 + heads, a.HKV);
  const int64_t pos = a.positions ? (int64_t)a.positions[b] : 0, begin = max(pos, (int64_t)0);
  const int64_t end = min(pos + (a.counts ? min(a.counts[b], a.N) : a.N), (int64_t)a.max_pages * a.page_size);
  const int64_t base = (begin / 32 + of) * 32, t0 = max(begin, base), t1 = min(end, base + 32);
  if (t0 >= t1) return;
  const uint32_t pg = (uint32_t)((uint64_t)base / (uint32_t)a.page_size);
  const int page = a.block_table[(int64_t)b * a.block_table_stride + pg];
  if (page < 0 || page >= a.num_pages) return;
  const int at = (int)(base - (int64_t)pg * a.page_size), first = (int)(t0 - base), last = (int)(t1 - base);
  const int64_t* const ps = isv ? a.v_strides : a.k_strides;
  const int64_t* const ss = isv ? a.v_scale_strides : a.k_scale_strides;
  const int64_t* const os = isv ? a.v_out_strides : a.k_out_strides;
  const float* const s = (isv ? a.v_scale : a.k_scale) + page * ss[0] + at / a.block * ss[2];
  const uint8_t* const p = static_cast<const uint8_t*>(isv ? a.v : a.k) + page * ps[0] + at * ps[2];
  char* const o = static_cast<char*>(isv ? a.v_out : a.k_out) + (b * os[0] + (base - pos) * os[2]) * kBytes<T>;
  for (int h = h0; h < h1; h += HEADS) {
    u2 c[HEADS][ITEMS];
    float f[HEADS];
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      if (h + n >= h1) break;
      f[n] = s[(h + n) * ss[1]];
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int u = (int)threadIdx.x + 256 * i, slot = u / PER, e = u % PER;
        if (slot < first || slot >= last) continue;
        const uint8_t* const q = p + (h + n) * ps[1] + slot * ps[2] + DIMS * e;
        if constexpr (DIMS == 8) c[n][i] = __builtin_nontemporal_load(reinterpret_cast<const u2*>(q));
        else c[n][i][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(q));
      }
    }
#pragma unroll
    for (int n = 0; n < HEADS; ++n) {
      if (h + n >= h1) break;
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int u = (int)threadIdx.x + 256 * i, slot = u / PER, e = u % PER;
        if (slot < first || slot >= last) continue;
        float y[8];
        u4 w;
        C::values(c[n][i][0], y);
        if constexpr (DIMS == 8) {
          C::values(c[n][i][1], y + 4);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            w[x] = T == kF16 ? pack_h2(y[2 * x] * f[n], y[2 * x + 1] * f[n])
                             : pack_bf2(y[2 * x] * f[n], y[2 * x + 1] * f[n]);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x) w[x] = __builtin_bit_cast(uint32_t, y[x] * f[n]);
        }
        __builtin_nontemporal_store(w, reinterpret_cast<u4*>(o + ((h + n) * os[1] + slot * os[2] + DIMS * e) * kBytes<T>));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side: validation and dispatch.
// ---------------------------------------------------------------------------
constexpr int kMaxAsk = 32;  // queries per row: two neighbouring chunks hold the last tokens of a row

static bool format_ok(const void* k, const void* v, const float* ks, const float* vs, const int64_t* kst,
                      const int64_t* vst, const int64_t* kss, const int64_t* vss, int block, int page_size,
                      int num_pages) {
  if (!pool_ok(k, kst, 16) || !pool_ok(v, vst, 16) || !ks || !vs || ((uintptr_t)ks | (uintptr_t)vs) & 3) return false;
  for (int i = 0; i < 3; ++i)
    if (kss[i] < 0 || vss[i] < 0) return false;
  if (block != 32 && block != 64 && block != 128) return false;
  return page_size > 0 && page_size % block == 0 && page_size <= kMaxPageTokens && num_pages > 0;
}

template <class C, int D, int HT, bool MULTI>
static int launch_paged8(const Paged8Params& p, hipStream_t st) {
  constexpr int NW = 4;
  const int rows = p.cols < 16 * HT ? p.cols : 16 * HT, blocks = (p.cols + 16 * HT - 1) / (16 * HT);
  const dim3 grid((unsigned)(p.a.HKV * blocks), (unsigned)(p.a.workgroups ? p.a.workgroups : p.a.B));
  const int wave = (rows * (D + 6) + 3) / 4 * 4;  // floats of a wave's partial
  const size_t lds = 32 * HT * (D + 8) + sizeof(float) * (16 * HT + NW * wave);
  return launch(paged8_split_kernel<C, D, HT, NW, MULTI>, grid, dim3(NW * 64), lds, st, p.a.seq_lens, p.a.B,
                p.a.max_pages * p.a.page_size, p.a.workgroups, p.a.least_chunks, p.a.long_workgroups, p.a.long_chunks, p);
}

template <class C, int D>
static int dispatch_paged8(const Paged8Params& p, hipStream_t st) {
  const bool multi = p.a.M > 1 || p.a.counts;
  const int rc = p.cols <= 16 ? (multi ? launch_paged8<C, D, 1, true>(p, st) : launch_paged8<C, D, 1, false>(p, st))
                              : (multi ? launch_paged8<C, D, 2, true>(p, st) : launch_paged8<C, D, 2, false>(p, st));
  if (rc || !p.a.workgroups) return rc;
  return join_shares(D, p.a.B, p.a.HQ * p.a.M, p.a.workgroups, p.a.row_pieces, p.a.partials, p.a.out, p.a.lse, kShift8,
                     st);
}

template <class C>
static int dispatch_paged8(const Paged8Params& p, hipStream_t st) {
  if (p.a.D == 64) return dispatch_paged8<C, 64>(p, st);
  if (p.a.D == 128) return dispatch_paged8<C, 128>(p, st);
  return dispatch_paged8<C, 256>(p, st);
}

template <class C, int T, int ROT>
static int launch_append8(Append8Params p, hipStream_t st) {
  const tkv_paged8_append_args& a = p.a;
  const int PER = a.D / 16;
  // Few tokens: a wave holds them all.  Else a thread for 16 values of a block, or for 32 of the
  // largest block of the largest heads.
  const bool few = a.N * (int64_t)PER <= 64;
  const int items = a.block * PER, threads = few ? 64 : items < 1024 ? items : 1024;
  const int64_t blocks = ((int64_t)a.N + a.block - 2) / a.block + 1;  // that N tokens may touch
  // Two heads to a workgroup, whose turns are then worked out once for both, where that leaves
  // workgroups enough (blocks of 32 tokens of 128 dims times heads, one / two, us: prompts of 288 5.2 / 5.4, 544
  // 6.5 / 6.2, 1088 9.3 / 8.5, 4128 25.2 / 21.2, with rotary 1088 25.7 / 23.5, 4128 86 / 77; steps of 512 4.0 /
  // 4.6, 1024 4.5 / 4.5, 4096 8.2 / 6.9; blocks of 128 tokens of 256 dims 320 14.7 / 15.1, 1056 44.4 / 44.7).
  p.heads = a.HKV > 1 && blocks * a.B * a.HKV > 1024 ? kAppendHeads : 1;
  const int sets = (a.HKV + p.heads - 1) / p.heads;
  int64_t groups = blocks * 2 * sets;
  p.kv_groups = (uint32_t)groups;
  size_t lds = 0;
  if (p.q.x) {  // (in one launch with the keys: 4 x 2049 tokens, 32 + 8
                // heads, 33.8 us; in two 41)
    const int64_t total = (int64_t)a.B * a.N;
    p.q_tile = total >= kTurnMany ? std::min(kTurnTile * std::max(1, threads / 256), threads / PER) : 1;
    const int lanes = threads / (p.q_tile * PER);
    p.q_parts = total < kTurnFew ? (p.q.H + lanes - 1) / lanes : 1;
    groups += ((int64_t)a.N + p.q_tile - 1) / p.q_tile * p.q_parts;
    lds = sizeof(float2) * p.q_tile * (p.turn.dims / 2);
  }
  if (ROT && few) lds = std::max(lds, sizeof(float2) * a.N * (p.turn.dims / 2));
  if (groups * threads > UINT32_MAX) return TKV_EINVAL;
  return launch(!few && items > 1024 ? paged8_append_kernel<C, T, 2, ROT> : paged8_append_kernel<C, T, 1, ROT>,
                dim3((unsigned)groups, (unsigned)a.B), dim3((unsigned)threads), lds, st, p);
}

template <class C, int T>
static int dispatch_append8(const Append8Params& p, hipStream_t st) {
  return !p.a.turns        ? launch_append8<C, T, 0>(p, st)
         : p.a.interleaved ? launch_append8<C, T, 2>(p, st)
                           : launch_append8<C, T, 1>(p, st);
}

template <class F>
static int by_type(int type, F start) {
  return type == kF16    ? start(std::integral_constant<int, kF16>{})
         : type == kBf16 ? start(std::integral_constant<int, kBf16>{})
                         : start(std::integral_constant<int, kF32>{});
}

}  // namespace tkv

extern "C" int tkv_paged8_decode_attention(const tkv_paged8_args* a, tkv_stream_t stream) {
  using namespace tkv;
  if (!a || !a->q || !a->out || !a->block_table) return TKV_EINVAL;
  if (a->B <= 0 || a->HQ <= 0 || a->HKV <= 0 || a->M <= 0 || a->M > kMaxAsk || a->HQ % a->HKV) return TKV_EINVAL;
  if ((int64_t)a->B * a->HQ * a->M > INT32_MAX) return TKV_EINVAL;
  if (a->max_pages <= 0 || a->block_table_stride < a->max_pages) return TKV_EINVAL;
  if (!format_ok(a->k, a->v, a->k_scale, a->v_scale, a->k_strides, a->v_strides, a->k_scale_strides, a->v_scale_strides,
                 a->block, a->page_size, a->num_pages))
    return TKV_EINVAL;
  if (!shares_ok(a->B, a->max_pages, a->page_size, a->least_chunks, a->workgroups, a->long_workgroups, a->long_chunks,
                 a->partials, a->row_pieces))
    return TKV_EINVAL;
  if (!rows_ok(a->q, a->q_strides, 3, 8) || (uintptr_t)a->out & 15) return TKV_EINVAL;
  if (a->D != 64 && a->D != 128 && a->D != 256) return TKV_EUNSUPPORTED;
  Paged8Params p;
  p.a = *a;
  p.G = a->HQ / a->HKV;
  p.cols = p.G * a->M;
  if ((int64_t)a->HKV * ((p.cols + 15) / 16) > INT32_MAX) return TKV_EINVAL;
  p.qk_scale = a->sm_scale * kLog2e;
  for (int i = 0; i < 3; ++i) {
    p.k16[i] = (uint32_t)(a->k_strides[i] / 16);
    p.v16[i] = (uint32_t)(a->v_strides[i] / 16);
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return a->is_int8 ? dispatch_paged8<Int8>(p, st) : dispatch_paged8<E4m3>(p, st);
}

extern "C" int tkv_paged8_append(const tkv_paged8_append_args* a, tkv_stream_t stream) {
  using namespace tkv;
  if (!a || !a->k_new || !a->v_new || !a->positions || !a->block_table) return TKV_EINVAL;
  if (a->B <= 0 || a->B > 65535 || a->HKV <= 0 || a->N <= 0 || a->max_pages <= 0 || a->block_table_stride < a->max_pages)
    return TKV_EINVAL;
  if (!format_ok(a->k, a->v, a->k_scale, a->v_scale, a->k_strides, a->v_strides, a->k_scale_strides, a->v_scale_strides,
                 a->block, a->page_size, a->num_pages))
    return TKV_EINVAL;
  if ((int64_t)a->max_pages * a->page_size > UINT32_MAX) return TKV_EINVAL;
  if (a->x_type < TKV_F16 || a->x_type > TKV_F32) return TKV_EINVAL;
  const int align = a->x_type == TKV_F32 ? 4 : 8;
  if (!rows_ok(a->k_new, a->k_new_strides, 3, align) || !rows_ok(a->v_new, a->v_new_strides, 3, align)) return TKV_EINVAL;
  if (a->D != 64 && a->D != 128 && a->D != 256) return TKV_EUNSUPPORTED;
  if (((int64_t)a->N / a->block + 2) * 2 * a->HKV > INT32_MAX) return TKV_EINVAL;
  if (!a->q != !a->q_out || (a->q && !a->turns)) return TKV_EINVAL;
  Append8Params p{};
  p.a = *a;
  if (a->turns) {
    if (a->dims <= 0 || a->dims > a->D || a->dims % 16) return TKV_EINVAL;
    p.turn = TurnPlan{a->positions, {1, 0}, 1, a->counts, a->turns, a->factor, a->factor, a->interleaved, a->dims, a->D};
    if (a->q) {
      if (a->HQ <= 0 || a->HQ > 65535 || (int64_t)a->B * a->N > INT32_MAX || !rows_ok(a->q, a->q_strides, 3, align) ||
          !rows_ok(a->q_out, a->q_out_strides, 3, align))
        return TKV_EINVAL;
      p.q = TurnRows{a->q, a->q_out, {a->q_strides[0], a->q_strides[1], a->q_strides[2]},
                     {a->q_out_strides[0], a->q_out_strides[1], a->q_out_strides[2]}, a->HQ};
    }
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return by_type(a->x_type, [&](auto type) {
    constexpr int T = decltype(type)::value;
    return a->is_int8 ? dispatch_append8<Int8, T>(p, st) : dispatch_append8<E4m3, T>(p, st);
  });
}

extern "C" int tkv_paged8_read(const tkv_paged8_read_args* a, tkv_stream_t stream) {
  using namespace tkv;
  if (!a || !a->k_out || !a->v_out || !a->block_table) return TKV_EINVAL;
  if (a->B <= 0 || a->B > 65535 || a->HKV <= 0 || a->N <= 0 || a->max_pages <= 0 || a->block_table_stride < a->max_pages)
    return TKV_EINVAL;
  if (a->D != 64 && a->D != 128 && a->D != 256) return TKV_EUNSUPPORTED;
  if (!format_ok(a->k, a->v, a->k_scale, a->v_scale, a->k_strides, a->v_strides, a->k_scale_strides, a->v_scale_strides,
                 a->block, a->page_size, a->num_pages))
    return TKV_EINVAL;
  if ((int64_t)a->max_pages * a->page_size > UINT32_MAX) return TKV_EINVAL;
  if (a->x_type < TKV_F16 || a->x_type > TKV_F32) return TKV_EINVAL;
  const int align = a->x_type == TKV_F32 ? 4 : 8;
  if (!rows_ok(a->k_out, a->k_out_strides, 3, align) || !rows_ok(a->v_out, a->v_out_strides, 3, align)) return TKV_EINVAL;
  const int64_t blocks = ((int64_t)a->N + 30) / 32 + 1;  // of 32 slots that N tokens may touch
  // Two heads to a workgroup where that leaves workgroups enough (blocks times heads, one / two, us: bf16 544 7.1 /
  // 7.3, 1088 10.1 / 9.9, 1632 12.9 / 11.9, 4352 26.3 / 23.5; fp32 1088 13.3 / 14.1, 1632 18.8 / 16.0).
  const int heads = a->HKV > 1 && blocks * a->B * a->HKV > 1280 ? 2 : 1;
  const int64_t groups = blocks * 2 * ((a->HKV + heads - 1) / heads);
  if (groups * 256 > UINT32_MAX) return TKV_EINVAL;
  const dim3 grid((unsigned)groups, (unsigned)a->B);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return by_type(a->x_type, [&](auto type) {
    constexpr int T = decltype(type)::value;
    auto kernel = [&](auto code) {
      using C = decltype(code);
      return a->D == 64 ? paged8_read_kernel<C, T, 64> : a->D == 128 ? paged8_read_kernel<C, T, 128> : paged8_read_kernel<C, T, 256>;
    };
    return launch(a->is_int8 ? kernel(Int8{}) : kernel(E4m3{}), grid, dim3(256), 0, st, *a, heads);
  });
}
