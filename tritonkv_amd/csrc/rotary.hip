// Rotary positions of queries and keys, for gfx950.
//
// Every value is read and written once, for 6 flops a pair: bound by HBM.  A
// workgroup takes a few tokens with all their heads, so that the angles, modulo whole turns,
// are worked out once a token and not once a head.  4 x 8213 tokens, 32 + 8 heads, bf16: 673 MB in
// 111 us, 6.1 TB/s (a copy's rate is 4.8); one token of 64 rows 3.4 us.  Halves of
// 64 of 128 dims take 141 us, halves that are no groups of 8, which go one value at a time, 198 (20 of 128
// dims; of 80 156).
#include <algorithm>
#include <type_traits>

#include "../../include/tkv.h"
#include "launch.h"
#include "rotary.h"

namespace tkv {

constexpr int kTurnThreads = 256;

template <int T, bool VEC, bool INTER, bool NT>
__global__ void __launch_bounds__(kTurnThreads) rotary_kernel(TurnPlan p, TurnRows q, TurnRows k, int N, uint32_t total,
                                                              int tile) {
  extern __shared__ float2 turns[];
  const uint32_t from = blockIdx.x * (uint32_t)tile;
  turn_tokens<T, VEC, INTER, NT>(p, q, k, (int)min((uint32_t)tile, total - from), blockIdx.y, gridDim.y, turns, [&](int i) {
    const uint32_t token = from + (uint32_t)i, b = token / (uint32_t)N;
    return make_int2((int)b, (int)(token - b * (uint32_t)N));
  });
}

// Queries q and keys k (H = 0: none) of B rows of N tokens.
static int turn_rows(const TurnPlan& p, const TurnRows& q, const TurnRows& k, int B, int N, int type, hipStream_t st) {
  const uint32_t total = (uint32_t)(B * (int64_t)N);
  const bool vec = p.interleaved || p.dims % 16 == 0;
  const int per = p.D / (vec ? 16 : 2);
  const bool many = total >= kTurnMany;
  const int tile = many ? std::min(kTurnTile, kTurnThreads / per) : 1;
  // Few tokens: heads over more workgroups, a walk of one step each.
  const int heads = q.H + k.H, lanes = kTurnThreads / (tile * per), walk = (heads + lanes - 1) / lanes;
  const dim3 grid((total + tile - 1) / tile, total < kTurnFew ? (unsigned)walk : 1);
  if ((int64_t)grid.x * kTurnThreads > UINT32_MAX) return TKV_EINVAL;
  const size_t lds = sizeof(float2) * tile * (p.dims / 2);
  auto start = [&](auto type) {
    constexpr int T = decltype(type)::value;
    auto kernel = [&](auto inter) {
      constexpr bool I = decltype(inter)::value;
      return many ? rotary_kernel<T, true, I, true> : rotary_kernel<T, true, I, false>;
    };
    return launch(!vec            ? rotary_kernel<T, false, false, false>
                  : p.interleaved ? kernel(std::true_type{})
                                  : kernel(std::false_type{}),
                  grid, dim3(kTurnThreads), lds, st, p, q, k,
                  N, total, tile);
  };
  return type == kF16    ? start(std::integral_constant<int, kF16>{})
         : type == kBf16 ? start(std::integral_constant<int, kBf16>{})
                                 : start(std::integral_constant<int, kF32>{});
}

static bool rows_aligned(const void* p, const int64_t* strides, int align) {
  return !((uintptr_t)p & 15) && !(strides[0] % align) && !(strides[1] % align) && !(strides[2] % align);
}

}  // namespace tkv

extern "C" int tkv_rotary(const tkv_rotary_args* a, tkv_stream_t stream) {
  using namespace tkv;
  if (!a || !a->q || !a->q_out || !a->positions || !a->turns || !a->k != !a->k_out) return TKV_EINVAL;
  if (a->B <= 0 || a->HQ <= 0 || (a->k && a->HKV <= 0) || a->N <= 0 || a->D <= 0 || a->D % 16 || a->D > 256)
    return TKV_EINVAL;
  if (a->dims <= 0 || a->dims % 2 || a->dims > a->D || a->x_type < TKV_F16 || a->x_type > TKV_F32) return TKV_EINVAL;
  if ((int64_t)a->B * a->N > INT32_MAX || a->HQ > 65535 || (a->k && a->HKV > 65535)) return TKV_EINVAL;
  const int align = a->x_type == TKV_F32 ? 4 : 8;
  if (!rows_aligned(a->q, a->q_strides, align) || !rows_aligned(a->q_out, a->q_out_strides, align)) return TKV_EINVAL;
  if (a->k && (!rows_aligned(a->k, a->k_strides, align) || !rows_aligned(a->k_out, a->k_out_strides, align)))
    return TKV_EINVAL;
  const TurnPlan p{a->positions, {a->position_strides[0], a->position_strides[1]}, a->position_step, nullptr, a->turns,
                   a->factor, a->adjoint ? -a->factor : a->factor, a->interleaved, a->dims, a->D};
  auto rows = [&](const void* x, void* out, const int64_t* xs, const int64_t* os, int H) {
    return TurnRows{x, out, {xs[0], xs[1], xs[2]}, {os[0], os[1], os[2]}, H};
  };
  const TurnRows q = rows(a->q, a->q_out, a->q_strides, a->q_out_strides, a->HQ),
                 k = rows(a->k, a->k_out, a->k_strides, a->k_out_strides, a->k ? a->HKV : 0);
  return turn_rows(p, q, k, a->B, a->N, a->x_type, reinterpret_cast<hipStream_t>(stream));
}
