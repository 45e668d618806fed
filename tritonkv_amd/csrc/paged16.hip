// Attention of one new token over 16-bit (fp16 or bf16) page pools, and the
// append that fills them, for gfx950.
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(sm_scale q[b, h] . k_t - max),
//   lse[b, h] = max + log sum_t p_t,        t < L_b
//
// The decode reads every live token's K and V row (2 * D * 2 bytes per token and KV
// head) once for every block of up to 32 query heads of a KV head, for 4 * D * G flops: G
// per byte where G <= 32, so HBM bounds it there.  Wider groups repeat the reads and the
// chunks' work per block (8 rows of 8192, 2 KV heads, bf16: G 32 20.6 us, 33 29.0, 64 29.7, 128
// 50.3).  One workgroup = a share of the batch's tokens for one KV head and up to
// 32 of its query heads; each of its four waves walks 32-token chunks, two 16-row
// MFMA tiles.  Scores are S^T = K Q^T (tokens as rows, heads as columns), whose
// accumulator layout is the B operand layout of O^T = V^T P^T, so the
// probabilities stay in registers (as in the contiguous fp16 kernel).
//
// Precision: out is fp32, and P enters the matrix cores as a sum of 16-bit
// terms, two for fp16 (22 bits) and three for bf16 (24): with P rounded once
// the output would be 2e-4 (fp16) or 2e-3 (bf16) off, and the extra MFMAs
// run in the shadow of the loads.  Its lower terms may be 0 or below, which times an
// infinite V would be NaN where p * V is infinite: a wave that finds NaN among its
// results goes over its chunks again, with V's infinities in a product of their own
// against p > 0.  Looking for NaN costs 0.1 us of a step.
//
// Measured, at steps of the sizes that a serving loop has (bytes of K, V, q and out
// over the time of both launches): 32 rows of 32768, HKV 8, G 4, fp16, pages of 256:
// 607 us one call after the other and 641 in a graph, 7.1 and 6.7 TB/s; 32 rows of
// 1000-16384, HKV 8, G 8, bf16, pages of 64, with the append: 177 us, 6.5 TB/s.  32 rows of
// 8192 in pages of 256, 64 and 16: 165, 166 and 172 us.  Small steps are bound by the two
// launches and the chain of lengths, table, K and V: one row of 505 tokens (12 / 2 heads)
// takes 6.8 us.
#include "page_shares.h"

namespace tkv {

// ---------------------------------------------------------------------------
// Element types.
// ---------------------------------------------------------------------------
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

struct Bf16;
struct Half {
  using Other = Bf16;
  static constexpr int kTerms = 2;
  static constexpr uint32_t kInf = 0x7c00;
  // P is scaled by 2^14: the low term of a small p would else fall below
  // fp16's smallest step (2^-24), e.g. 3e-5 of a p of 2^-10.
  static constexpr float kShift = 14.0f;
  static __device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) { return mfma_k32(a, b, c); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_h2(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return half_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return half_hi(w); }
};

struct Bf16 {
  using Other = Half;
  static constexpr int kTerms = 3;
  static constexpr uint32_t kInf = 0x7f80;
  static constexpr float kShift = 0.0f;
  static __device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c,
                                                   0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const b2 v = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
  static __device__ __forceinline__ float lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
};

// The infinities among two values, zeros in the others' place.
template <class T>
__device__ __forceinline__ uint32_t infinities(uint32_t w) {
  const uint32_t lo = (w & 0x7fffu) == T::kInf ? 0x0000ffffu : 0u;
  const uint32_t hi = (w >> 16 & 0x7fffu) == T::kInf ? 0xffff0000u : 0u;
  return w & (lo | hi);
}

struct Paged16Params {
  tkv_paged16_args a;
  int G, page_tiles;
  float qk_scale;  // sm_scale * log2(e)
  uint32_t k16[3], v16[3];  // the pools' strides in 16 bytes: products of 32 bits by 32
};

// ---------------------------------------------------------------------------
// The split kernel.
// ---------------------------------------------------------------------------
// HT: tiles of 16 query heads per workgroup, 1 or (G > 16) 2.  A second workgroup for
// heads 16 to 31 would read all of K and V again: 16 rows of up to 8192, HKV 8, G 24
// took 82 us with one tile and 62 with two (G 16: 56).
template <class T, int D, int HT, int NW, bool APPEND>
__global__ void __launch_bounds__(NW * 64, D == 256 ? 1 : D == 128 ? 4 - HT : 5 - HT)
paged16_split_kernel(const int32_t* lens, int B, int S, int workgroups, int least_chunks, int long_workgroups,
                     int long_chunks, Paged16Params prm) {
  constexpr int NKM = D / 32;  // 16x16x32 steps over the head dim
  constexpr int EPL = D / 16;  // V dims per lane (and V MFMAs)
  constexpr int VW = EPL / 2;  // dwords of them
  const tkv_paged16_args& a = prm.a;
  constexpr int QROW = D + 8;  // elements of a query row in LDS: 16 rows meet no bank twice
  constexpr int OROW = D + 4;  // floats of an output row there: 16-byte pieces
  // The queries of the heads, the new token's K and V rows (APPEND), then per wave
  // of the merge: rows of OROW floats, maximum and sum of each.
  extern __shared__ float lds_all[];
  uint16_t* const lds_q = reinterpret_cast<uint16_t*>(lds_all);
  uint16_t* const lds_new = lds_q + 16 * HT * QROW;
  float* const lds = lds_all + 8 * HT * QROW + (APPEND ? D : 0);

  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, j = lane >> 4;
  RowLens rows{lens, B, S, lane, 0, 0};
  Shares sh;
  Segment g;
  uint32_t share_end;
  if (!first_segment(SharePlan{lens, B, S, workgroups, least_chunks, long_workgroups, long_chunks}, blockIdx.y, rows, sh,
                     g, share_end))
    return;
  const int hk = blockIdx.x % a.HKV, hb0 = (blockIdx.x / a.HKV) * 16 * HT;
  const int nh = min(16 * HT, prm.G - hb0), h0 = hk * prm.G + hb0;

  const int64_t kts = a.k_strides[2], vts = a.v_strides[2];
  const uint32_t kspan = (uint32_t)(15 * kts + D) * 2, vspan = (uint32_t)(15 * vts + D) * 2;
  const uint32_t klane = (uint32_t)(r * kts + 8 * j) * 2;
  uint32_t vlane[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) vlane[i] = (uint32_t)((4 * j + i) * vts + EPL * r) * 2;

  // Addresses.  Lane l looks up tile l % 2 of the wave's chunk l / 2: the
  // table entries and 64-bit tile addresses of 32 chunks come from one load.
  const uint64_t khead = (uint64_t)a.k + 16 * ((uint64_t)hk * prm.k16[1]);
  const uint64_t vhead = (uint64_t)a.v + 16 * ((uint64_t)hk * prm.v16[1]);
  uint64_t kt = 0, vt = 0;  // this lane's tile
  int lo, hi;               // tokens of the segment
  auto tiles = [&](int c0) {
    const int t = lo + 32 * (w + NW * (c0 + (lane >> 1))) + 16 * (lane & 1);
    uint32_t page = 0, at = 0;  // past the segment: the pool's first tile, whose rows are masked
    if (t < hi) {
      const uint32_t t16 = (uint32_t)t / 16, pg = t16 / (uint32_t)prm.page_tiles;
      at = 16 * (t16 - pg * prm.page_tiles);
      page = min(max(a.block_table[(int64_t)g.b * a.block_table_stride + pg], 0), a.num_pages - 1);
    }
    kt = khead + 16 * ((uint64_t)page * prm.k16[0] + (uint64_t)at * prm.k16[2]);
    vt = vhead + 16 * ((uint64_t)page * prm.v16[0] + (uint64_t)at * prm.v16[2]);
  };
  auto lane_ptr = [&](uint64_t x, int l) {
    const uint32_t x0 = __builtin_amdgcn_readlane((int)(uint32_t)x, l);
    const uint32_t x1 = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), l);
    return reinterpret_cast<const void*>(((uint64_t)x1 << 32) | x0);
  };
  u4 kx[2][NKM];
  uint32_t vx[8][VW];
  auto load_k = [&](int c) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const rsrc_t rk = make_rsrc(lane_ptr(kt, 2 * (c & 31) + t), kspan);
#pragma unroll
      for (int m = 0; m < NKM; ++m) kx[t][m] = buf_u4<kPolF16>(rk, klane + 64 * m);
    }
  };
  auto load_v = [&](int c) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const rsrc_t rv = make_rsrc(lane_ptr(vt, 2 * (c & 31) + t), vspan);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (VW >= 4) {
#pragma unroll
          for (int e = 0; e < VW; e += 4) {
            const u4 x = buf_u4<kPolF16>(rv, vlane[i] + 4 * e);
#pragma unroll
            for (int y = 0; y < 4; ++y) vx[4 * t + i][e + y] = x[y];
          }
        } else {
          const u2 x = buf_u2<kPolF16>(rv, vlane[i]);
          vx[4 * t + i][0] = x[0];
          vx[4 * t + i][1] = x[1];
        }
      }
    }
  };

  bool app, owner;  // the segment takes the new token; in this wave
  // Starts segment g: what its first chunk needs is on its way afterwards.
  auto begin_segment = [&] {
    const int bt = (int)opaque(tid), bl = bt & 63;
    lo = 32 * (int)g.begin;
    hi = min(g.L, 32 * (int)g.end);
    app = APPEND && hi == g.L && hi > lo && !(hi == S && lens && lens[g.b] > S);  // (a place past the table: none)
    owner = app && w == ((hi - 1 - lo) / 32) % NW;
    u4 new8 = {0u, 0u, 0u, 0u};  // lanes 0 .. D / 8 - 1: 8 dims of the new key; then of the value
    const bool mine = APPEND && owner && bl < D / 4;
    if (APPEND && mine) {
      const bool isv = bl >= D / 8;
      const int64_t* st = isv ? a.v_new_strides : a.k_new_strides;
      new8 = *reinterpret_cast<const u4*>(static_cast<const uint16_t*>(isv ? a.v_new : a.k_new) + g.b * st[0] +
                                          hk * st[1] + 8 * (bl & (D / 8 - 1)));
    }
    // The queries: 8 dims of a head per thread and round, zero past the group.  They and
    // the new rows wait in LDS, which leaves the registers to K and V.
    constexpr int QV = 16 * HT * (D / 8), QR = (QV + NW * 64 - 1) / (NW * 64);
    u4 q8[QR];
#pragma unroll
    for (int i = 0; i < QR; ++i) {
      const int u = bt + NW * 64 * i, head = u / (D / 8);
      q8[i] = u4{0u, 0u, 0u, 0u};
      if (head < nh)
        q8[i] = *reinterpret_cast<const u4*>(static_cast<const uint16_t*>(a.q) + g.b * a.q_strides[0] +
                                             (h0 + head) * a.q_strides[1] + 8 * (u % (D / 8)));
    }
    tiles(0);
#pragma unroll
    for (int i = 0; i < QR; ++i) {
      const int u = bt + NW * 64 * i, head = u / (D / 8);
      if (u < QV) *reinterpret_cast<u4*>(lds_q + head * QROW + 8 * (u % (D / 8))) = q8[i];
    }
    if (APPEND && mine) *reinterpret_cast<u4*>(lds_new + 8 * bl) = new8;
    if (lo + 32 * w < hi) {
      load_k(0);
      load_v(0);
    }
    __syncthreads();
  };

  begin_segment();
  for (;;) {
    const int last = hi - 1;
    f4 accv[HT][EPL];
    float m_run[HT], l_run[HT];
    auto start = [&] {
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
        for (int mv = 0; mv < EPL; ++mv) accv[ht][mv] = f4{0.f, 0.f, 0.f, 0.f};
        m_run[ht] = -INFINITY;
        l_run[ht] = 0.0f;
      }
    };
    start();

    auto step = [&](int c, int cb, int r, int j, auto tail, auto infinite) {
      constexpr bool TAIL = decltype(tail)::value, INF = decltype(infinite)::value;
      const bool more = cb + 32 * NW < hi;
      if constexpr (TAIL && APPEND) {
        if (owner) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (cb + 16 * t + r == last)
#pragma unroll
              for (int m = 0; m < NKM; ++m) kx[t][m] = *reinterpret_cast<const u4*>(lds_new + 32 * m + 8 * j);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (cb + slot_token(j, i) == last)
#pragma unroll
              for (int e = 0; e < VW; ++e) vx[i][e] = reinterpret_cast<const uint32_t*>(lds_new + D + EPL * r)[e];
        }
      }
      float x[HT][8];
      {
        // (opaque: read again in every chunk, not kept in registers)
        const uint16_t* ql = lds_q + (int)opaque((uint32_t)(r * QROW + 8 * j));
        f4 s[HT][2];
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) s[ht][0] = s[ht][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < NKM; ++m)
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) {
            const u4 qf = *reinterpret_cast<const u4*>(ql + 16 * ht * QROW + 32 * m);
#pragma unroll
            for (int t = 0; t < 2; ++t) s[ht][t] = T::mfma(kx[t][m], qf, s[ht][t]);
          }
#pragma unroll
        for (int ht = 0; ht < HT; ++ht)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[ht][i] = s[ht][i / 4][i % 4] * prm.qk_scale;
      }
      if constexpr (TAIL) {
#pragma unroll
        for (int ht = 0; ht < HT; ++ht)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (cb + slot_token(j, i) > last) x[ht][i] = -INFINITY;
      }
      if (!TAIL && more) {
        if (((c + 1) & 31) == 0) tiles(c + 1);  // V of chunk c is on its way already
        load_k(c + 1);
      }
      // Online softmax in base 2; the accumulators are rescaled only in chunks
      // where a head's maximum rose.
      u4 pt[HT][T::kTerms], some[HT];  // some (INF): 1 where p > 0
#pragma unroll
      for (int ht = 0; ht < HT; ++ht) {
        float top = x[ht][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, x[ht][i]);
        if (__builtin_amdgcn_ballot_w64(top > m_run[ht]) != 0) {
          const float mn = vmax(m_run[ht], xor_max16_32(top));
          const float alpha = safe_exp2_diff(m_run[ht], mn);
          m_run[ht] = mn;
          l_run[ht] *= alpha;
#pragma unroll
          for (int mv = 0; mv < EPL; ++mv) accv[ht][mv] *= alpha;
        }
        // scores of -inf under a maximum of -inf give p = 0, not NaN
        const float off = T::kShift - (m_run[ht] == -INFINITY ? 0.0f : m_run[ht]);
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(x[ht][i] + off);
          l_run[ht] += p[i];
        }
        if constexpr (INF)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            some[ht][i] = T::pack(p[2 * i] > 0.0f ? 1.0f : 0.0f, p[2 * i + 1] > 0.0f ? 1.0f : 0.0f);
#pragma unroll
        for (int n = 0; n < T::kTerms; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t wd = T::pack(p[2 * i], p[2 * i + 1]);
            pt[ht][n][i] = wd;
            p[2 * i] -= T::lo(wd);
            p[2 * i + 1] -= T::hi(wd);
          }
      }
      if constexpr (TAIL) {
        // Rows past the sequence are whatever the page holds there (possibly
        // NaN or Inf); p = 0 alone would not cancel them in the MFMA.
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (cb + slot_token(j, i) > last)
#pragma unroll
            for (int e = 0; e < VW; ++e) vx[i][e] = 0u;
      }
      // V is waited for behind the softmax: left to itself the compiler may ask for it, and with
      // it for the next K, ahead of the exponentials (32 rows of 8000-16384, head dim 64: 134 us
      // against 129).
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int mv = 0; mv < EPL; ++mv) {
        const uint32_t sel = (mv & 1) ? 0x07060302u : 0x05040100u;
        u4 av;
#pragma unroll
        for (int i = 0; i < 4; ++i) av[i] = perm(vx[2 * i + 1][mv / 2], vx[2 * i][mv / 2], sel);
        if constexpr (INF) {
          u4 iv;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            iv[i] = infinities<T>(av[i]);
            av[i] ^= iv[i];
          }
#pragma unroll
          for (int ht = 0; ht < HT; ++ht) accv[ht][mv] = T::mfma(iv, some[ht], accv[ht][mv]);
        }
#pragma unroll
        for (int ht = 0; ht < HT; ++ht)
#pragma unroll
          for (int n = T::kTerms - 1; n >= 0; --n) accv[ht][mv] = T::mfma(av, pt[ht][n], accv[ht][mv]);
      }
      if (!TAIL && more) load_v(c + 1);
    };

    // Full chunks, then the row's partial last one, or the one that takes the new token.
    const int full = app ? last : hi;
    int c = 0, cb = lo + 32 * w;
    for (; cb + 32 <= full; cb += 32 * NW, ++c) step(c, cb, r, j, std::false_type{}, std::false_type{});
    if (cb < hi) step(c, cb, r, j, std::true_type{}, std::false_type{});

    f4 all = f4{0.f, 0.f, 0.f, 0.f};  // NaN if one of them is
#pragma unroll
    for (int ht = 0; ht < HT; ++ht)
#pragma unroll
      for (int mv = 0; mv < EPL; ++mv) all += accv[ht][mv];
    const float sum = (all[0] + all[1]) + (all[2] + all[3]);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(sum != sum) != 0, 0)) {
      start();
      for (c = 0, cb = lo + 32 * w; cb < hi; cb += 32 * NW, ++c) {
        if ((c & 31) == 0) tiles(c);
        load_k(c);
        load_v(c);
        step(c, cb, (int)opaque(r), (int)opaque(j), std::true_type{}, std::true_type{});
      }
    }

    if (APPEND && owner && hb0 == 0) {
      const uint32_t t16 = (uint32_t)last / 16, pg = t16 / (uint32_t)prm.page_tiles;
      const int page = a.block_table[(int64_t)g.b * a.block_table_stride + pg];
      if (page >= 0 && page < a.num_pages) {
        const int64_t at = last - (int64_t)pg * prm.page_tiles * 16;
        uint16_t* kd = static_cast<uint16_t*>(a.k) + page * a.k_strides[0] + hk * a.k_strides[1] + at * kts;
        uint16_t* vd = static_cast<uint16_t*>(a.v) + page * a.v_strides[0] + hk * a.v_strides[1] + at * vts;
        if (lane < D / 8) {
          *reinterpret_cast<u4*>(kd + 8 * lane) = *reinterpret_cast<const u4*>(lds_new + 8 * lane);
          *reinterpret_cast<u4*>(vd + 8 * lane) = *reinterpret_cast<const u4*>(lds_new + D + 8 * lane);
        }
      }
    }

    // Merge of the waves.  (opaque: the addresses of this part would else be kept in
    // registers over the whole loop.)
    const int mr = (int)opaque(r), mj = (int)opaque(j), mt = (int)opaque(tid);
    const int b = g.b, mine_rows = min(16 * HT, prm.G);
    const int stride = (mine_rows * (OROW + 2) + 3) / 4 * 4;
#pragma unroll
    for (int ht = 0; ht < HT; ++ht) {
      const float lt = xor_sum16_32(l_run[ht]);
      const int n = mr + 16 * ht;
      if (n >= nh) continue;
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
    for (int idx = mt; idx < nh * (D / 4); idx += NW * 64) {
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
      if (whole) {
        store_row4(a.out, a.lse, D, T::kShift, (int64_t)b * a.HQ + h0 + n, d, o, mstar, ls);
      } else {
        const int64_t row = partial_row(a.HQ, slot, h0 + n);
        *reinterpret_cast<f4*>(a.partials + row * D + d) = o;
        if (d == 0)
          *reinterpret_cast<float2*>(partial_ml(a.partials, workgroups, a.HQ, D) + 2 * row) = make_float2(mstar, ls);
      }
    }
    if (!again) break;
    __syncthreads();  // the partials in LDS have been read
  }
}

// ---------------------------------------------------------------------------
// Append: token n < counts[b] of row b's N goes to logical position
// positions[b] + n, rounded to the pools' type once.  Thread = 8 dims of a (token,
// head), two at a time, of K (even blockIdx.x) or V (odd) of row blockIdx.y; heads
// vary before tokens, so that token-major inputs, which the projections leave, are
// read in order.  Bound by HBM: the new rows are read once and written once.  Their
// loads start before the table is known, everything but the addresses is 32 bits, and the
// stores do not wait in the caches (non-temporal).  4 x 8213 tokens, HKV 8, D 128, fp16: 35
// us, 5.7 TB/s (four pieces a thread 37.5; with stores that stay in the caches as well 42;
// with 64-bit indices as well 54); one token for 64 rows 2.0 us (four pieces 2.3).
// ---------------------------------------------------------------------------
constexpr int kAppendPer = 2;

// IN: the new rows' type: the pools', fp32, or the other 16-bit type, which is exact in
// fp32 and takes no longer than the pools' own (4 x 8213 tokens 47.6 and 47.4 us, fp32 71.1).
template <class T, int IN>
__global__ void __launch_bounds__(256) paged16_append_kernel(tkv_paged16_append_args a, uint32_t items) {
  const bool isv = blockIdx.x & 1;
  const int b = blockIdx.y;
  const uint32_t per = (uint32_t)a.D / 8, HKV = a.HKV;
  const int64_t xb = isv ? a.v_new_strides[0] : a.k_new_strides[0], xh = isv ? a.v_new_strides[1] : a.k_new_strides[1],
                xn = isv ? a.v_new_strides[2] : a.k_new_strides[2];
  const int64_t pp = isv ? a.v_strides[0] : a.k_strides[0], ph = isv ? a.v_strides[1] : a.k_strides[1],
                pt = isv ? a.v_strides[2] : a.k_strides[2];
  const int count = a.counts ? min(a.counts[b], a.N) : a.N;
  const int64_t pos = a.positions[b];
  const uint32_t first = (blockIdx.x >> 1) * (256 * kAppendPer) + threadIdx.x;
  u4 y[kAppendPer];
  int n[kAppendPer];
  int64_t to[kAppendPer];
#pragma unroll
  for (int i = 0; i < kAppendPer; ++i) {
    const uint32_t u = first + 256 * i, rest = u / per, e = u - rest * per, h = rest % HKV;
    n[i] = u < items ? (int)(rest / HKV) : INT_MAX;
    if (n[i] >= count) continue;
    const int64_t from = b * xb + h * xh + n[i] * xn + 8 * e;
    to[i] = h * ph + 8 * e;
    if constexpr (IN == TKV_NEW_FP32) {
      const float* x = static_cast<const float*>(isv ? a.v_new : a.k_new) + from;
      const f4 x0 = *reinterpret_cast<const f4*>(x), x1 = *reinterpret_cast<const f4*>(x + 4);
      y[i] = u4{T::pack(x0[0], x0[1]), T::pack(x0[2], x0[3]), T::pack(x1[0], x1[1]), T::pack(x1[2], x1[3])};
    } else {
      y[i] = *reinterpret_cast<const u4*>(static_cast<const uint16_t*>(isv ? a.v_new : a.k_new) + from);
      if constexpr (IN == TKV_NEW_OTHER) {
#pragma unroll
        for (int x = 0; x < 4; ++x) y[i][x] = T::pack(T::Other::lo(y[i][x]), T::Other::hi(y[i][x]));
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kAppendPer; ++i) {
    if (n[i] >= count) continue;
    const int64_t t = pos + n[i];
    if (t < 0 || t >= (int64_t)a.max_pages * a.page_size) continue;
    const uint32_t pg = (uint32_t)t / (uint32_t)a.page_size;
    const int page = a.block_table[(int64_t)b * a.block_table_stride + pg];
    if (page < 0 || page >= a.num_pages) continue;
    __builtin_nontemporal_store(
        y[i], reinterpret_cast<u4*>(static_cast<uint16_t*>(isv ? a.v : a.k) + page * pp +
                                    (int64_t)((uint32_t)t - pg * (uint32_t)a.page_size) * pt + to[i]));
  }
}

// ---------------------------------------------------------------------------
// Host side: validation and dispatch.
// ---------------------------------------------------------------------------
static int check_paged16(const tkv_paged16_args* a) {
  if (!a || !a->q || !a->out || !a->block_table) return TKV_EINVAL;
  if (a->B <= 0 || a->HQ <= 0 || a->HKV <= 0 || a->D <= 0 || a->HQ % a->HKV) return TKV_EINVAL;
  if ((int64_t)a->B * a->HQ > INT32_MAX) return TKV_EINVAL;
  if (a->page_size <= 0 || a->page_size % 16 || a->page_size > kMaxPageTokens || a->max_pages <= 0 ||
      a->num_pages <= 0 || a->block_table_stride < a->max_pages)
    return TKV_EINVAL;
  if (!shares_ok(a->B, a->max_pages, a->page_size, a->least_chunks, a->workgroups, a->long_workgroups, a->long_chunks,
                 a->partials, a->row_pieces))
    return TKV_EINVAL;
  if (!pool_ok(a->k, a->k_strides, 8) || !pool_ok(a->v, a->v_strides, 8)) return TKV_EINVAL;
  if (!rows_ok(a->q, a->q_strides, 2, 8)) return TKV_EINVAL;
  if ((uintptr_t)a->out & 15) return TKV_EINVAL;
  if (a->k_new || a->v_new) {
    if (!a->k_new || !a->v_new || !rows_ok(a->k_new, a->k_new_strides, 2, 8) ||
        !rows_ok(a->v_new, a->v_new_strides, 2, 8))
      return TKV_EINVAL;
  }
  if (a->D != 64 && a->D != 128 && a->D != 256) return TKV_EUNSUPPORTED;
  return TKV_OK;
}

template <class T, int D, int HT>
static int launch_paged16(const Paged16Params& p, hipStream_t st) {
  constexpr int NW = 4;
  const int rows = p.G < 16 * HT ? p.G : 16 * HT, blocks = (p.G + 16 * HT - 1) / (16 * HT);
  const dim3 grid((unsigned)(p.a.HKV * blocks), (unsigned)(p.a.workgroups ? p.a.workgroups : p.a.B));
  const int wave = (rows * (D + 6) + 3) / 4 * 4;  // floats of a wave's partial
  const size_t lds = 32 * HT * (D + 8) + sizeof(float) * NW * wave;
  const auto kernel = p.a.k_new ? paged16_split_kernel<T, D, HT, NW, true> : paged16_split_kernel<T, D, HT, NW, false>;
  return launch(kernel, grid, dim3(NW * 64), p.a.k_new ? lds + 4 * D : lds, st, p.a.seq_lens, p.a.B,
                p.a.max_pages * p.a.page_size, p.a.workgroups, p.a.least_chunks, p.a.long_workgroups, p.a.long_chunks, p);
}

template <class T, int D>
static int dispatch_paged16(const Paged16Params& p, hipStream_t st) {
  const int rc = p.G <= 16 ? launch_paged16<T, D, 1>(p, st) : launch_paged16<T, D, 2>(p, st);
  if (rc || !p.a.workgroups) return rc;
  return join_shares(D, p.a.B, p.a.HQ, p.a.workgroups, p.a.row_pieces, p.a.partials, p.a.out, p.a.lse, T::kShift, st);
}

template <class T>
static int dispatch_paged16(const Paged16Params& p, hipStream_t st) {
  if (p.a.D == 64) return dispatch_paged16<T, 64>(p, st);
  if (p.a.D == 128) return dispatch_paged16<T, 128>(p, st);
  return dispatch_paged16<T, 256>(p, st);
}

}  // namespace tkv

extern "C" int tkv_paged16_decode_attention(const tkv_paged16_args* a, tkv_stream_t stream) {
  using namespace tkv;
  const int rc = check_paged16(a);
  if (rc) return rc;
  Paged16Params p;
  p.a = *a;
  p.G = a->HQ / a->HKV;
  p.page_tiles = a->page_size / 16;
  p.qk_scale = a->sm_scale * kLog2e;
  for (int i = 0; i < 3; ++i) {
    p.k16[i] = (uint32_t)(a->k_strides[i] / 8);
    p.v16[i] = (uint32_t)(a->v_strides[i] / 8);
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return a->is_bf16 ? dispatch_paged16<Bf16>(p, st) : dispatch_paged16<Half>(p, st);
}

extern "C" int tkv_paged16_append(const tkv_paged16_append_args* a, tkv_stream_t stream) {
  using namespace tkv;
  if (!a || !a->k_new || !a->v_new || !a->positions || !a->block_table) return TKV_EINVAL;
  if (a->B <= 0 || a->HKV <= 0 || a->N <= 0 || a->D <= 0 || a->D % 8) return TKV_EINVAL;
  if (a->page_size <= 0 || a->max_pages <= 0 || a->num_pages <= 0 || a->block_table_stride < a->max_pages)
    return TKV_EINVAL;
  if (!pool_ok(a->k, a->k_strides, 8) || !pool_ok(a->v, a->v_strides, 8)) return TKV_EINVAL;
  if (a->new_is_fp32 < TKV_NEW_SAME || a->new_is_fp32 > TKV_NEW_OTHER) return TKV_EINVAL;
  const int align = a->new_is_fp32 == TKV_NEW_FP32 ? 4 : 8;
  if (!rows_ok(a->k_new, a->k_new_strides, 3, align) || !rows_ok(a->v_new, a->v_new_strides, 3, align))
    return TKV_EINVAL;
  if ((int64_t)a->max_pages * a->page_size > UINT32_MAX || a->B > 65535) return TKV_EINVAL;
  const int64_t items = (int64_t)a->N * a->HKV * (a->D / 8);
  if (items > INT32_MAX) return TKV_EINVAL;
  const int64_t blocks = (items + 256 * kAppendPer - 1) / (256 * kAppendPer);
  const dim3 grid((unsigned)(2 * blocks), (unsigned)a->B);
  const uint32_t n = (uint32_t)items;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto start = [&](auto type) {
    using T = decltype(type);
    return launch(a->new_is_fp32 == TKV_NEW_SAME   ? paged16_append_kernel<T, TKV_NEW_SAME>
                  : a->new_is_fp32 == TKV_NEW_FP32 ? paged16_append_kernel<T, TKV_NEW_FP32>
                                                   : paged16_append_kernel<T, TKV_NEW_OTHER>,
                  grid, dim3(256), 0, st, *a, n);
  };
  return a->is_bf16 ? start(Bf16{}) : start(Half{});
}
