// Attention of one new token over 16-bit (fp16 or bf16) page pools, and the
// append that fills them, for gfx950.
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(sm_scale q[b, h] . k_t - max),
//   lse[b, h] = max + log sum_t p_t,        t < L_b
//
// The decode reads every live token's K and V row once (2 * D * 2 bytes per
// token and KV head) for 4 * D * G flops: it is bound by HBM for every GQA
// group.  One workgroup = one piece of one row's tokens for one KV head and up
// to 16 of its query heads; each wave walks 32-token chunks, two 16-row MFMA
// tiles.  Scores are S^T = K Q^T (tokens as rows, heads as columns), whose
// accumulator layout is the B operand layout of O^T = V^T P^T, so the
// probabilities stay in registers (as in the contiguous fp16 kernel).
//
// Precision: out is fp32, and P enters the matrix cores as a sum of 16-bit
// terms, two for fp16 (22 bits) and three for bf16 (24): with P rounded once
// the output would be 2e-4 (fp16) or 2e-3 (bf16) off, and the extra MFMAs
// run in the shadow of the loads.
#include "decode_common.h"

namespace tkv {

// ---------------------------------------------------------------------------
// Element types.
// ---------------------------------------------------------------------------
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

struct Half {
  static constexpr int kTerms = 2;
  // P is scaled by 2^14: the low term of a small p would else fall below
  // fp16's smallest step (2^-24), e.g. 3e-5 of a p of 2^-10.
  static constexpr float kShift = 14.0f;
  static __device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) { return mfma_k32(a, b, c); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_h2(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return half_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return half_hi(w); }
  static __device__ __forceinline__ float value(uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); }
  static __device__ __forceinline__ uint16_t round(float x) {
    return __builtin_bit_cast(uint16_t, (_Float16)x);
  }
};

struct Bf16 {
  static constexpr int kTerms = 3;
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
  static __device__ __forceinline__ float value(uint16_t u) {
    return __builtin_bit_cast(float, (uint32_t)u << 16);
  }
  static __device__ __forceinline__ uint16_t round(float x) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
  }
};

// ---------------------------------------------------------------------------
// The plan of the pieces, made on the device from the rows' lengths.
//
// A serving loop's table is as wide as its longest request may get, and the
// lengths live on the device, so a split of the table's capacity would leave
// most pieces empty.  Instead every workgroup derives the same plan from the
// lengths: with l_b = ceil(L_b / 32) chunks, a piece holds at most
//   c = max(least, ceil(sum_b l_b / target))
// chunks, row b is cut evenly into n_b = ceil(l_b / c) pieces (an empty row
// keeps one, which writes its zeros), and workgroup `slot` takes the slot-th
// piece in row order: sum_b n_b <= target + B pieces.  target == 0: one piece
// per row.
// ---------------------------------------------------------------------------
struct Paged16Params {
  tkv_paged16_args a;
  int G, page_tiles, S;
  float qk_scale;  // sm_scale * log2(e)
};

struct Piece {
  int b, L, lo, hi;   // tokens [lo, hi) of row b, which holds L
  int base, count;    // the row's first piece and how many it has
  bool live;
};

__device__ __forceinline__ int clamp_len(int L, int S) { return max(0, min(L, S)); }

// Pieces of a row of l chunks, and how many chunks each holds.
__device__ __forceinline__ void cut_row(uint32_t l, uint32_t c, uint32_t& count, uint32_t& chunks) {
  if (l <= c) {
    count = 1;
    chunks = l;
  } else {
    const uint32_t n = (l + c - 1) / c;
    chunks = (l + n - 1) / n;
    count = (l + chunks - 1) / chunks;
  }
}

__device__ __forceinline__ Piece find_piece(const Paged16Params& prm, int slot) {
  const int32_t* __restrict__ lens = prm.a.seq_lens;
  const int B = prm.a.B, S = prm.S, lane = threadIdx.x & 63;
  const uint32_t least = prm.a.least_chunks, target = prm.a.target_pieces;
  Piece p;
  uint32_t count, chunks, s;
  if (target == 0) {  // one piece per row
    p.live = slot < B;
    if (!p.live) return p;
    p.b = slot;
    p.L = lens ? clamp_len(__builtin_amdgcn_readfirstlane(lens[slot]), S) : S;
    p.base = slot;
    count = 1;
    chunks = ((uint32_t)p.L + 31) / 32;
    s = 0;
  } else if (!lens || B == 1) {  // every row alike
    p.L = lens ? clamp_len(__builtin_amdgcn_readfirstlane(lens[0]), S) : S;
    const uint32_t l = ((uint32_t)p.L + 31) / 32;
    const uint32_t c = max(least, (l * B + target - 1) / target);
    cut_row(l, c, count, chunks);
    p.b = (uint32_t)slot / count;
    p.live = p.b < B;
    if (!p.live) return p;
    p.base = p.b * count;
    s = slot - p.base;
  } else {
    uint32_t sum = 0;
    for (int b0 = 0; b0 < B; b0 += 64)
      if (b0 + lane < B) sum += ((uint32_t)clamp_len(lens[b0 + lane], S) + 31) / 32;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) sum += __shfl_xor((int)sum, off, 64);
    const uint32_t c = max(least, (sum + target - 1) / target);
    uint32_t before = 0;
    p.live = false;
    for (int b0 = 0; b0 < B; b0 += 64) {
      const bool in = b0 + lane < B;
      const int L = in ? clamp_len(lens[b0 + lane], S) : 0;
      uint32_t n, m;
      cut_row(((uint32_t)L + 31) / 32, c, n, m);
      n = in ? n : 0;
      uint32_t end = n;  // inclusive sum over the lanes
#pragma unroll
      for (int off = 1; off < 64; off *= 2) {
        const uint32_t o = __shfl_up((int)end, off, 64);
        end += lane >= off ? o : 0;
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(before + end > (uint32_t)slot);
      if (past) {
        const int at = __builtin_ctzll(past);
        p.live = true;
        p.b = b0 + at;
        p.L = __builtin_amdgcn_readlane(L, at);
        count = __builtin_amdgcn_readlane((int)n, at);
        chunks = __builtin_amdgcn_readlane((int)m, at);
        p.base = before + __builtin_amdgcn_readlane((int)end, at) - count;
        s = slot - p.base;
        break;
      }
      before += __builtin_amdgcn_readlane((int)end, 63);
    }
    if (!p.live) return p;
  }
  p.count = count;
  p.lo = (int)(32 * s * chunks);
  p.hi = s + 1 == count ? p.L : (int)(32 * (s + 1) * chunks);
  return p;
}

// Where the partial of head h of piece `slot` lives.
__device__ __forceinline__ int64_t partial_row(const tkv_paged16_args& a, int slot, int h) {
  return (int64_t)slot * a.HQ + h;
}
__device__ __forceinline__ float* partial_ml(const tkv_paged16_args& a) {
  return a.partials + (int64_t)a.max_pieces * a.HQ * a.D;
}

__device__ __forceinline__ void store_row4(const tkv_paged16_args& a, float shift, int64_t row, int d, f4 o,
                                           float m, float l) {
  // A row that saw nothing (no tokens, or scores of -inf alone) is zero.
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<f4*>(a.out + row * a.D + d) = o * inv;
  if (a.lse && d == 0)
    a.lse[row] = l == 0.0f ? -INFINITY : (m - shift + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// ---------------------------------------------------------------------------
// The split kernel.
// ---------------------------------------------------------------------------
template <class T, int D, int NW, bool APPEND>
__global__ void __launch_bounds__(NW * 64) paged16_split_kernel(Paged16Params prm) {
  constexpr int NKM = D / 32;  // 16x16x32 steps over the head dim
  constexpr int EPL = D / 16;  // V dims per lane (and V MFMAs)
  constexpr int VW = EPL / 2;  // dwords of them
  const tkv_paged16_args& a = prm.a;
  extern __shared__ float lds[];  // per wave: rows of D + 1 floats, then max and sum of each row

  const int slot = blockIdx.y;
  const Piece pc = find_piece(prm, slot);
  if (!pc.live) return;
  const int hk = blockIdx.x % a.HKV, hb0 = (blockIdx.x / a.HKV) * 16;
  const int nh = min(16, prm.G - hb0), h0 = hk * prm.G + hb0;
  const int b = pc.b, lo = pc.lo, hi = pc.hi, last = hi - 1;

  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 15, j = lane >> 4;
  // The row's last piece takes the new token in place of the page's row.
  const bool app = APPEND && hi == pc.L && hi > lo;

  // Addresses.  Lane l looks up tile l % 2 of the wave's chunk l / 2: the
  // table entries and 64-bit tile addresses of 32 chunks come from one load.
  const int64_t kts = a.k_strides[2], vts = a.v_strides[2];
  uint64_t kt = 0, vt = 0;  // this lane's tile
  auto tiles = [&](int c0) {
    const int t = lo + 32 * (w + NW * (c0 + (lane >> 1))) + 16 * (lane & 1);
    uint32_t page = 0, at = 0;  // past the piece: the pool's first tile, whose rows are masked
    if (t < hi) {
      const uint32_t t16 = (uint32_t)t / 16, pg = t16 / (uint32_t)prm.page_tiles;
      at = 16 * (t16 - pg * prm.page_tiles);
      page = min(max(a.block_table[(int64_t)b * a.block_table_stride + pg], 0), a.num_pages - 1);
    }
    kt = (uint64_t)a.k + 2 * (page * a.k_strides[0] + hk * a.k_strides[1] + at * kts);
    vt = (uint64_t)a.v + 2 * (page * a.v_strides[0] + hk * a.v_strides[1] + at * vts);
  };
  auto lane_ptr = [&](uint64_t x, int l) {
    const uint32_t x0 = __builtin_amdgcn_readlane((int)(uint32_t)x, l);
    const uint32_t x1 = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), l);
    return reinterpret_cast<const void*>(((uint64_t)x1 << 32) | x0);
  };
  const uint32_t kspan = (uint32_t)(15 * kts + D) * 2, vspan = (uint32_t)(15 * vts + D) * 2;
  const uint32_t klane = (uint32_t)(r * kts + 8 * j) * 2;
  uint32_t vlane[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) vlane[i] = (uint32_t)((4 * j + i) * vts + EPL * r) * 2;

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

  tiles(0);
  const int cb0 = lo + 32 * w;
  if (cb0 < hi) {
    load_k(0);
    load_v(0);
  }

  u4 knew[NKM];
  uint32_t vnew[VW];
  const bool owner = app && w == ((last - lo) / 32) % NW;
  if (APPEND && owner) {
    const uint16_t* kn = static_cast<const uint16_t*>(a.k_new) + b * a.k_new_strides[0] + hk * a.k_new_strides[1];
    const uint16_t* vn = static_cast<const uint16_t*>(a.v_new) + b * a.v_new_strides[0] + hk * a.v_new_strides[1];
#pragma unroll
    for (int m = 0; m < NKM; ++m) knew[m] = *reinterpret_cast<const u4*>(kn + 32 * m + 8 * j);
#pragma unroll
    for (int e = 0; e < VW; e += 2) {
      const u2 x = *reinterpret_cast<const u2*>(vn + EPL * r + 2 * e);
      vnew[e] = x[0];
      vnew[e + 1] = x[1];
    }
  }

  u4 qf[NKM];
  {
    const bool hv = r < nh;
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + b * a.q_strides[0] + (h0 + (hv ? r : 0)) * a.q_strides[1];
#pragma unroll
    for (int m = 0; m < NKM; ++m) {
      const u4 x = *reinterpret_cast<const u4*>(q + 32 * m + 8 * j);
      qf[m] = hv ? x : u4{0u, 0u, 0u, 0u};
    }
  }

  f4 accv[EPL];
#pragma unroll
  for (int mv = 0; mv < EPL; ++mv) accv[mv] = f4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.0f;

  auto step = [&](int c, int cb, auto tail) {
    constexpr bool TAIL = decltype(tail)::value;
    const bool more = cb + 32 * NW < hi;
    if constexpr (TAIL && APPEND) {
      if (owner && cb + 32 >= hi) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (cb + 16 * t + r == last)
#pragma unroll
            for (int m = 0; m < NKM; ++m) kx[t][m] = knew[m];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (cb + slot_token(j, i) == last)
#pragma unroll
            for (int e = 0; e < VW; ++e) vx[i][e] = vnew[e];
      }
    }
    float x[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f4 s = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < NKM; ++m) s = T::mfma(kx[t][m], qf[m], s);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * t + i] = s[i] * prm.qk_scale;
    }
    if constexpr (TAIL) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (cb + slot_token(j, i) > last) x[i] = -INFINITY;
    }
    if (!TAIL && more) {
      if (((c + 1) & 31) == 0) {
        // V of chunk c is in registers already: its loads were issued from the old tiles.
        tiles(c + 1);
      }
      load_k(c + 1);
    }
    // Online softmax in base 2; the accumulators are rescaled only in chunks
    // where a head's maximum rose.
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    if (__builtin_amdgcn_ballot_w64(top > m_run) != 0) {
      const float mn = vmax(m_run, xor_max16_32(top));
      const float alpha = safe_exp2_diff(m_run, mn);
      m_run = mn;
      l_run *= alpha;
#pragma unroll
      for (int mv = 0; mv < EPL; ++mv) accv[mv] *= alpha;
    }
    // scores of -inf under a maximum of -inf give p = 0, not NaN
    const float off = T::kShift - (m_run == -INFINITY ? 0.0f : m_run);
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = __builtin_amdgcn_exp2f(x[i] + off);
      l_run += p[i];
    }
    u4 pt[T::kTerms];
#pragma unroll
    for (int n = 0; n < T::kTerms; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t wd = T::pack(p[2 * i], p[2 * i + 1]);
        pt[n][i] = wd;
        p[2 * i] -= T::lo(wd);
        p[2 * i + 1] -= T::hi(wd);
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
#pragma unroll
    for (int mv = 0; mv < EPL; ++mv) {
      const uint32_t sel = (mv & 1) ? 0x07060302u : 0x05040100u;
      u4 av;
#pragma unroll
      for (int i = 0; i < 4; ++i) av[i] = perm(vx[2 * i + 1][mv / 2], vx[2 * i][mv / 2], sel);
#pragma unroll
      for (int n = T::kTerms - 1; n >= 0; --n) accv[mv] = T::mfma(av, pt[n], accv[mv]);
    }
    if (!TAIL && more) load_v(c + 1);
  };

  // Full chunks, then the partial last one, or the one that takes the new token.
  const int full = app ? last : hi;
  int c = 0, cb = cb0;
  for (; cb + 32 <= full; cb += 32 * NW, ++c) step(c, cb, std::false_type{});
  if (cb < hi) step(c, cb, std::true_type{});

  if (APPEND && owner && hb0 == 0) {
    const uint32_t t16 = (uint32_t)last / 16, pg = t16 / (uint32_t)prm.page_tiles;
    const int page = a.block_table[(int64_t)b * a.block_table_stride + pg];
    if (page >= 0 && page < a.num_pages) {
      const int64_t at = last - (int64_t)pg * prm.page_tiles * 16;
      uint16_t* kd = static_cast<uint16_t*>(a.k) + page * a.k_strides[0] + hk * a.k_strides[1] + at * kts;
      uint16_t* vd = static_cast<uint16_t*>(a.v) + page * a.v_strides[0] + hk * a.v_strides[1] + at * vts;
      if (r == 0)
#pragma unroll
        for (int m = 0; m < NKM; ++m) *reinterpret_cast<u4*>(kd + 32 * m + 8 * j) = knew[m];
      if (j == 0)
#pragma unroll
        for (int e = 0; e < VW; e += 2) *reinterpret_cast<u2*>(vd + EPL * r + 2 * e) = u2{vnew[e], vnew[e + 1]};
    }
  }

  // Merge of the waves.
  const int rows = min(16, prm.G);
  const int stride = rows * (D + 1) + 2 * rows;
  float* mine = lds + w * stride;
  const float lt = xor_sum16_32(l_run);
  if (r < nh) {
#pragma unroll
    for (int mv = 0; mv < EPL; ++mv)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[r * (D + 1) + EPL * (4 * j + i) + mv] = accv[mv][i];
    if (j == 0) {
      mine[rows * (D + 1) + r] = m_run;
      mine[rows * (D + 2) + r] = lt;
    }
  }
  __syncthreads();
  for (int idx = tid; idx < nh * (D / 4); idx += NW * 64) {
    const int n = idx / (D / 4), d = 4 * (idx % (D / 4));
    float mw[NW], mstar = -INFINITY;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      mw[x] = lds[x * stride + rows * (D + 1) + n];
      mstar = fmaxf(mstar, mw[x]);
    }
    f4 o = f4{0.f, 0.f, 0.f, 0.f};
    float l = 0.0f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      // A wave whose scores were all NaN keeps a maximum of -inf and a sum of
      // NaN, which the factor 0 hands on.
      const float f = safe_exp2_diff(mw[x], mstar);
      const float* ow = lds + x * stride + n * (D + 1) + d;
      o += f4{ow[0], ow[1], ow[2], ow[3]} * f;
      l = fmaf(f, lds[x * stride + rows * (D + 2) + n], l);
    }
    if (pc.count == 1) {
      store_row4(a, T::kShift, (int64_t)b * a.HQ + h0 + n, d, o, mstar, l);
    } else {
      const int64_t row = partial_row(a, slot, h0 + n);
      *reinterpret_cast<f4*>(a.partials + row * D + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(partial_ml(a) + 2 * row) = make_float2(mstar, l);
    }
  }
  if (a.target_pieces && slot == pc.base && blockIdx.x == 0 && tid == 0)
    reinterpret_cast<int2*>(a.row_pieces)[b] = make_int2(pc.base, pc.count);
}

// ---------------------------------------------------------------------------
// The join of rows cut into pieces: one 256-thread workgroup per (b, h); rows
// of one piece were written by the split kernel.  Thread (g, dq) merges float4
// column dq of pieces g, g + SG, ...; the SG groups meet in LDS.
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) paged16_join_kernel(Paged16Params prm, float shift) {
  constexpr int DQ = D / 4, SG = 256 / DQ;
  __shared__ float sm_m[SG], sm_l[SG];
  __shared__ f4 sm_a[SG][DQ];
  const tkv_paged16_args& a = prm.a;
  const int b = blockIdx.x / a.HQ, h = blockIdx.x % a.HQ;
  const int2 pieces = reinterpret_cast<const int2*>(a.row_pieces)[b];
  if (pieces.y <= 1) return;
  const int t = threadIdx.x, dq = t % DQ, g = t / DQ;
  const float* ml = partial_ml(a);
  float m = -INFINITY, l = 0.0f;
  f4 o = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = g; s < pieces.y; s += SG) {
    const int64_t row = partial_row(a, pieces.x + s, h);
    const float2 x = *reinterpret_cast<const float2*>(ml + 2 * row);
    const f4 os = *reinterpret_cast<const f4*>(a.partials + row * D + 4 * dq);
    const float mn = fmaxf(m, x.x);
    const float al = safe_exp2_diff(m, mn), be = safe_exp2_diff(x.x, mn);
    o = o * al + os * be;
    l = l * al + x.y * be;
    m = mn;
  }
  if (dq == 0) {
    sm_m[g] = m;
    sm_l[g] = l;
  }
  sm_a[g][dq] = o;
  __syncthreads();
  if (g == 0) {
    float mstar = -INFINITY, lt = 0.0f;
#pragma unroll
    for (int x = 0; x < SG; ++x) mstar = fmaxf(mstar, sm_m[x]);
    f4 ot = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < SG; ++x) {
      const float f = safe_exp2_diff(sm_m[x], mstar);
      ot += sm_a[x][dq] * f;
      lt += sm_l[x] * f;
    }
    store_row4(a, shift, (int64_t)b * a.HQ + h, 4 * dq, ot, mstar, lt);
  }
}

// ---------------------------------------------------------------------------
// Append: token n < counts[b] of row b's N goes to logical position
// positions[b] + n, rounded to the pools' type once.  Thread = 8 dims of one
// (b, token, head) of K (blockIdx.y 0) or V (1); heads vary before tokens, so
// token-major inputs, which the projections leave, are read in order.
// ---------------------------------------------------------------------------
struct AppendParams {
  tkv_paged16_append_args a;
  int64_t items;  // B * N * HKV * D / 8
};

template <class T, bool F32>
__global__ void __launch_bounds__(256) paged16_append_kernel(AppendParams prm) {
  const tkv_paged16_append_args& a = prm.a;
  const bool isv = blockIdx.y != 0;
  const int per = a.D / 8;
  const int64_t* xs = isv ? a.v_new_strides : a.k_new_strides;
  const int64_t* ps = isv ? a.v_strides : a.k_strides;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < prm.items; i += (int64_t)gridDim.x * 256) {
    const int e = i % per;
    const int64_t rest = i / per;
    const int h = rest % a.HKV;
    const int64_t bn = rest / a.HKV;
    const int n = bn % a.N, b = bn / a.N;
    if (a.counts && n >= a.counts[b]) continue;
    const int64_t t = (int64_t)a.positions[b] + n;
    if (t < 0 || t >= (int64_t)a.max_pages * a.page_size) continue;
    const int pg = t / a.page_size;
    const int page = a.block_table[(int64_t)b * a.block_table_stride + pg];
    if (page < 0 || page >= a.num_pages) continue;
    const int64_t from = b * xs[0] + h * xs[1] + n * xs[2] + 8 * e;
    const int64_t to = page * ps[0] + h * ps[1] + (t - (int64_t)pg * a.page_size) * ps[2] + 8 * e;
    u4 y;
    if constexpr (F32) {
      const float* x = static_cast<const float*>(isv ? a.v_new : a.k_new) + from;
      const f4 x0 = *reinterpret_cast<const f4*>(x), x1 = *reinterpret_cast<const f4*>(x + 4);
      y = u4{T::pack(x0[0], x0[1]), T::pack(x0[2], x0[3]), T::pack(x1[0], x1[1]), T::pack(x1[2], x1[3])};
    } else {
      y = *reinterpret_cast<const u4*>(static_cast<const uint16_t*>(isv ? a.v_new : a.k_new) + from);
    }
    *reinterpret_cast<u4*>(static_cast<uint16_t*>(isv ? a.v : a.k) + to) = y;
  }
}

// ---------------------------------------------------------------------------
// Host side: validation and dispatch.
// ---------------------------------------------------------------------------
constexpr int kMaxPageTokens = 1 << 24;

// Pool rows are read and written 16 bytes at a time; one 16-row tile spans 32 bits.
static bool pool_ok(const void* p, const int64_t* strides) {
  if (!p || (uintptr_t)p & 15) return false;
  for (int i = 0; i < 3; ++i)
    if (strides[i] < 0 || strides[i] % 8) return false;
  return strides[2] > 0 && strides[2] < (int64_t(1) << 26);
}
static bool rows_ok(const void* p, const int64_t* strides, int n, int align) {
  if ((uintptr_t)p & 15) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] % align) return false;
  return true;
}

static int check_paged16(const tkv_paged16_args* a) {
  if (!a || !a->q || !a->out || !a->block_table) return TKV_EINVAL;
  if (a->B <= 0 || a->HQ <= 0 || a->HKV <= 0 || a->D <= 0 || a->HQ % a->HKV) return TKV_EINVAL;
  if ((int64_t)a->B * a->HQ > INT32_MAX) return TKV_EINVAL;
  if (a->page_size <= 0 || a->page_size % 16 || a->page_size > kMaxPageTokens || a->max_pages <= 0 ||
      a->num_pages <= 0 || a->block_table_stride < a->max_pages)
    return TKV_EINVAL;
  if ((int64_t)a->max_pages * a->page_size > INT32_MAX - 65536) return TKV_EINVAL;
  // the plan sums the rows' chunks in 32 bits
  if ((int64_t)a->B * ((int64_t)a->max_pages * a->page_size / 32 + 1) > INT32_MAX) return TKV_EINVAL;
  if (!pool_ok(a->k, a->k_strides) || !pool_ok(a->v, a->v_strides)) return TKV_EINVAL;
  if (!rows_ok(a->q, a->q_strides, 2, 8)) return TKV_EINVAL;
  if ((uintptr_t)a->out & 15) return TKV_EINVAL;
  if (a->k_new || a->v_new) {
    if (!a->k_new || !a->v_new || !rows_ok(a->k_new, a->k_new_strides, 2, 8) ||
        !rows_ok(a->v_new, a->v_new_strides, 2, 8))
      return TKV_EINVAL;
  }
  if (a->least_chunks <= 0 || a->target_pieces < 0) return TKV_EINVAL;
  if (a->max_pieces <= 0 || a->max_pieces > 65535) return TKV_EINVAL;
  if ((int64_t)a->target_pieces + a->B > a->max_pieces) return TKV_EINVAL;
  if (a->target_pieces && (!a->partials || (uintptr_t)a->partials & 15 || !a->row_pieces ||
                           (uintptr_t)a->row_pieces & 7))
    return TKV_EINVAL;
  if (a->waves != 0 && a->waves != 4 && a->waves != 8) return TKV_EINVAL;
  if (a->D != 64 && a->D != 128 && a->D != 256) return TKV_EUNSUPPORTED;
  return TKV_OK;
}

template <class T, int D, int NW>
static void launch_paged16(const Paged16Params& p, dim3 grid, hipStream_t st) {
  const int rows = p.G < 16 ? p.G : 16;
  const size_t lds = sizeof(float) * NW * (rows * (D + 1) + 2 * rows);
  if (p.a.k_new)
    paged16_split_kernel<T, D, NW, true><<<grid, dim3(NW * 64), lds, st>>>(p);
  else
    paged16_split_kernel<T, D, NW, false><<<grid, dim3(NW * 64), lds, st>>>(p);
}

template <class T>
static void dispatch_paged16(const Paged16Params& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.a.HKV * ((p.G + 15) / 16)), (unsigned)p.a.max_pieces);
  const bool wide = p.a.waves == 8;
  if (p.a.D == 64) {
    if (wide) launch_paged16<T, 64, 8>(p, grid, st);
    else launch_paged16<T, 64, 4>(p, grid, st);
  } else if (p.a.D == 128) {
    if (wide) launch_paged16<T, 128, 8>(p, grid, st);
    else launch_paged16<T, 128, 4>(p, grid, st);
  } else {
    launch_paged16<T, 256, 4>(p, grid, st);  // 8 waves' partials would not fit the LDS
  }
  if (!p.a.target_pieces) return;
  const dim3 rows((unsigned)(p.a.B * p.a.HQ));
  if (p.a.D == 64) paged16_join_kernel<64><<<rows, dim3(256), 0, st>>>(p, T::kShift);
  else if (p.a.D == 128) paged16_join_kernel<128><<<rows, dim3(256), 0, st>>>(p, T::kShift);
  else paged16_join_kernel<256><<<rows, dim3(256), 0, st>>>(p, T::kShift);
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
  p.S = a->max_pages * a->page_size;
  p.qk_scale = a->sm_scale * kLog2e;
  (void)hipGetLastError();
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a->is_bf16) dispatch_paged16<Bf16>(p, st);
  else dispatch_paged16<Half>(p, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TKV_OK : (int)e;
}

extern "C" int tkv_paged16_append(const tkv_paged16_append_args* a, tkv_stream_t stream) {
  using namespace tkv;
  if (!a || !a->k_new || !a->v_new || !a->positions || !a->block_table) return TKV_EINVAL;
  if (a->B <= 0 || a->HKV <= 0 || a->N <= 0 || a->D <= 0 || a->D % 8) return TKV_EINVAL;
  if (a->page_size <= 0 || a->max_pages <= 0 || a->num_pages <= 0 || a->block_table_stride < a->max_pages)
    return TKV_EINVAL;
  if (!pool_ok(a->k, a->k_strides) || !pool_ok(a->v, a->v_strides)) return TKV_EINVAL;
  const int align = a->new_is_fp32 ? 4 : 8;
  if (!rows_ok(a->k_new, a->k_new_strides, 3, align) || !rows_ok(a->v_new, a->v_new_strides, 3, align))
    return TKV_EINVAL;
  AppendParams p;
  p.a = *a;
  p.items = (int64_t)a->B * a->N * a->HKV * (a->D / 8);
  const int64_t blocks = (p.items + 255) / 256;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), 2);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  (void)hipGetLastError();
  if (a->is_bf16) {
    if (a->new_is_fp32) paged16_append_kernel<Bf16, true><<<grid, dim3(256), 0, st>>>(p);
    else paged16_append_kernel<Bf16, false><<<grid, dim3(256), 0, st>>>(p);
  } else {
    if (a->new_is_fp32) paged16_append_kernel<Half, true><<<grid, dim3(256), 0, st>>>(p);
    else paged16_append_kernel<Half, false><<<grid, dim3(256), 0, st>>>(p);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TKV_OK : (int)e;
}
