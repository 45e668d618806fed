// The join of the rows that a page-pool decode cut, for gfx950.
#include "page_shares.h"

namespace tkv {

// ---------------------------------------------------------------------------
// The join of rows that several workgroups shared; whole rows were written by the
// split kernel.  LANES lanes take a (b, h): lane (g, dq) merges float4 column dq of
// pieces g, g + SG, ..., and the SG groups meet in LDS.
// Few rows have many pieces and take 256 lanes each; many rows have one to three
// pieces each, and four of them share a workgroup.
// ---------------------------------------------------------------------------
template <int D, int LANES>
__global__ void __launch_bounds__(256) shares_join_kernel(const int2* row_pieces, float* partials, float* out,
                                                           float* lse, int HQ, int rows, int workgroups, float shift) {
  constexpr int DQ = D / 4, SG = LANES / DQ, ROWS = 256 / LANES;
  __shared__ float sm_m[ROWS][SG], sm_l[ROWS][SG];
  __shared__ f4 sm_a[ROWS][SG][DQ];
  const int in = threadIdx.x / LANES, row0 = blockIdx.x * ROWS + in;
  const bool live = row0 < rows;
  const int b = live ? row0 / HQ : 0, h = row0 - b * HQ;
  const int2 pieces = live ? row_pieces[b] : make_int2(0, 0);
  if (ROWS == 1 && pieces.y <= 1) return;
  const int t = threadIdx.x % LANES, dq = t % DQ, g = t / DQ;
  const float* ml = partial_ml(partials, workgroups, HQ, D);
  float m = -INFINITY, l = 0.0f;
  f4 o = f4{0.f, 0.f, 0.f, 0.f};
  const int n = pieces.y > 1 ? pieces.y : 0;
#pragma unroll 4
  for (int s = g; s < n; s += SG) {
    const int64_t row = partial_row(HQ, 2 * (pieces.x + s) + (s == 0 ? 1 : 0), h);
    const float2 x = *reinterpret_cast<const float2*>(ml + 2 * row);
    const f4 os = *reinterpret_cast<const f4*>(partials + row * D + 4 * dq);
    const float mn = fmaxf(m, x.x);
    const float al = safe_exp2_diff(m, mn), be = safe_exp2_diff(x.x, mn);
    o = o * al + os * be;
    l = l * al + x.y * be;
    m = mn;
  }
  if (dq == 0) {
    sm_m[in][g] = m;
    sm_l[in][g] = l;
  }
  sm_a[in][g][dq] = o;
  __syncthreads();
  if (g == 0 && n) {
    float mstar = -INFINITY, lt = 0.0f;
#pragma unroll
    for (int x = 0; x < SG; ++x) mstar = fmaxf(mstar, sm_m[in][x]);
    f4 ot = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < SG; ++x) {
      const float f = safe_exp2_diff(sm_m[in][x], mstar);
      ot += sm_a[in][x][dq] * f;
      lt += sm_l[in][x] * f;
    }
    store_row4(out, lse, D, shift, row0, 4 * dq, ot, mstar, lt);
  }
}

constexpr int kJoinRows = 512;  // (b, h) rows from which on the join takes a wave for each

template <int D>
static int launch_join(int B, int HQ, int workgroups, const int32_t* row_pieces, float* partials, float* out, float* lse,
                       float shift, hipStream_t st) {
  const int rows = B * HQ;
  const bool many = rows >= kJoinRows;
  return launch(many ? shares_join_kernel<D, 64> : shares_join_kernel<D, 256>,
                dim3((unsigned)(many ? (rows + 3) / 4 : rows)), dim3(256), 0, st,
                reinterpret_cast<const int2*>(row_pieces), partials, out, lse, HQ, rows, workgroups, shift);
}

int join_shares(int D, int B, int HQ, int workgroups, const int32_t* row_pieces, float* partials, float* out, float* lse,
                float shift, hipStream_t st) {
  const auto start = D == 64 ? launch_join<64> : D == 128 ? launch_join<128> : launch_join<256>;
  return start(B, HQ, workgroups, row_pieces, partials, out, lse, shift, st);
}

}  // namespace tkv
