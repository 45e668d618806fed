// The split of paged rows over workgroups, made on the device from the rows' lengths,
// and the join of the rows that were cut (the page-pool decodes).
#pragma once

#include "decode_common.h"
#include "launch.h"

namespace tkv {

// ---------------------------------------------------------------------------
// The split, made on the device from the rows' lengths.
//
// A serving loop's table is as wide as its longest request may get, and the
// lengths live on the device, so a split of the table's capacity would leave
// most pieces empty and the others uneven.  Instead the rows' chunks (32 tokens;
// an empty row counts as one, which writes its zeros) are laid end to end, and the
// W = min(workgroups, ceil(chunks / least_chunks)) workgroups of a KV head
// take equal shares of that line, workgroup i the chunks from Shares::start(i) on.
// (long_workgroups of them where that gives each long_chunks at least, in batches of
// no more rows: fewer, longer streams then read faster; paged16.py has the figures.)
// A share covers the end of one row, whole rows, and the start of another; each
// such segment is attended by itself.  Whole rows are written out; the others
// leave a partial in slot 2i (the row began in an earlier share) or 2i + 1, and
// the join kernel merges a row's partials, which lie in consecutive shares.
// workgroups == 0: one workgroup per row.
//
// Measured on 32 rows of 200-16184 tokens (HKV 8, G 4 / 8, D 128): pieces of one row
// each, cut evenly, 184-194 us; shares 172 / 176; of 1000-16384 (G 8) 193 and 178.  8 rows of 300-4000 take 18.9 us in
// tables of 131072 tokens and of 4032.
// ---------------------------------------------------------------------------
// What finds a workgroup's first segment: scalar arguments of the kernel, which are in
// registers when a wave starts (a struct is not), so that the lengths are asked for at once.
struct SharePlan {
  const int32_t* lens;
  int B, S, workgroups, least_chunks, long_workgroups, long_chunks;
};

__device__ __forceinline__ int clamp_len(int L, int S) { return max(0, min(L, S)); }
__device__ __forceinline__ uint32_t chunks_of(int L) { return max(1u, ((uint32_t)L + 31) / 32); }

// Inclusive sum over the wave's lanes, on the VALU: four shifts within rows of 16
// lanes, then the rows' totals passed on.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t add_dpp(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = add_dpp<0x111, 0xF>(v);  // row_shr:1
  v = add_dpp<0x112, 0xF>(v);
  v = add_dpp<0x114, 0xF>(v);
  v = add_dpp<0x118, 0xF>(v);
  v = add_dpp<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  return add_dpp<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}

struct Shares {
  uint32_t each, more;  // the first `more` shares hold each + 1 chunks
  __device__ __forceinline__ uint32_t start(uint32_t i) const { return i * each + min(i, more); }
  __device__ __forceinline__ uint32_t of(uint32_t chunk) const {
    const uint32_t big = more * (each + 1);
    return chunk < big ? chunk / (each + 1) : more + (chunk - big) / each;
  }
};

// The rows' lengths, 64 of them in a wave's lanes at a time.
struct RowLens {
  const int32_t* lens;
  int B, S, lane, first, L;
  __device__ __forceinline__ void load(int b0) {
    first = b0;
    L = lens ? (b0 + lane < B ? clamp_len(lens[b0 + lane], S) : 0) : S;
  }
  __device__ __forceinline__ int of(int b) {  // b uniform
    if (b >= first + 64) load(b);
    return __builtin_amdgcn_readlane(L, b - first);
  }
};

struct Segment {
  int b, L;             // a row and its length
  uint32_t begin, end;  // its chunks of this segment
  uint32_t at;          // the row's first chunk on the line
};

// Chunks from which on every workgroup has its least (saturated).
__device__ __forceinline__ uint32_t full_at(const SharePlan& a) {
  const uint64_t n = (uint64_t)(uint32_t)a.workgroups * (uint32_t)a.least_chunks;
  return n > 0xffffffffu ? 0xffffffffu : (uint32_t)n;
}

__device__ __forceinline__ Shares make_shares(uint32_t total, const SharePlan& a, uint32_t& W) {
  W = a.workgroups;
  if (a.B <= a.long_workgroups && total >= (uint32_t)a.long_workgroups * (uint32_t)a.long_chunks) W = a.long_workgroups;
  else if (total < full_at(a)) W = min(W, (total + a.least_chunks - 1) / (uint32_t)a.least_chunks);
  Shares s;
  s.each = total / W;
  s.more = total - s.each * W;
  return s;
}

// This workgroup's first segment and the end of its share; false: it has none.
__device__ __forceinline__ bool first_segment(const SharePlan& plan, int i, RowLens& rows, Shares& sh,
                                              Segment& g, uint32_t& share_end) {
  const int B = plan.B, lane = rows.lane;
  if (plan.workgroups == 0) {
    rows.load(i & ~63);
    g.b = i;
    g.L = rows.of(i);
    g.begin = g.at = 0;
    g.end = share_end = chunks_of(g.L);
    sh.each = sh.more = 0;
    return true;
  }
  rows.load(0);
  uint32_t W;
  if (!rows.lens || B == 1) {  // every row alike
    const int L = rows.of(0);
    const uint32_t l = chunks_of(L);
    sh = make_shares(l * B, plan, W);
    if ((uint32_t)i >= W) return false;
    const uint32_t from = sh.start(i);
    share_end = sh.start(i + 1);
    g.b = from / l;
    g.L = L;
    g.at = g.b * l;
    g.begin = from - g.at;
    g.end = min(share_end - g.at, l);
    return true;
  }
  // Up to 64 rows, which is most batches, one scan serves the sum and the search.
  uint32_t l = lane < B ? chunks_of(rows.L) : 0, past = wave_scan(l);
  uint32_t sum = __builtin_amdgcn_readlane((int)past, 63);
  for (int b0 = 64; b0 < B; b0 += 64) {
    rows.load(b0);
    sum += __builtin_amdgcn_readlane((int)wave_scan(b0 + lane < B ? chunks_of(rows.L) : 0), 63);
  }
  sh = make_shares(sum, plan, W);
  if ((uint32_t)i >= W) return false;
  const uint32_t from = sh.start(i);
  share_end = sh.start(i + 1);
  uint32_t before = 0;
  for (int b0 = 0; b0 < B; b0 += 64) {
    if (B > 64) {
      rows.load(b0);
      l = b0 + lane < B ? chunks_of(rows.L) : 0;
      past = wave_scan(l);
    }
    const uint64_t hit = __builtin_amdgcn_ballot_w64(before + past > from);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      const uint32_t n = __builtin_amdgcn_readlane((int)l, at);
      g.b = b0 + at;
      g.L = __builtin_amdgcn_readlane(rows.L, at);
      g.at = before + __builtin_amdgcn_readlane((int)past, at) - n;
      g.begin = from - g.at;
      g.end = min(share_end - g.at, n);
      return true;
    }
    before += __builtin_amdgcn_readlane((int)past, 63);
  }
  return false;  // not reached: from < sum
}

// Where the partial of head h in a slot lives; maxima and sums after all rows.
__device__ __forceinline__ int64_t partial_row(int HQ, uint32_t slot, int h) { return (int64_t)slot * HQ + h; }
__device__ __forceinline__ float* partial_ml(float* partials, int workgroups, int HQ, int D) {
  return partials + (int64_t)2 * workgroups * HQ * D;
}

__device__ __forceinline__ void store_row4(float* out, float* lse, int D, float shift, int64_t row, int d, f4 o,
                                           float m, float l) {
  // A row that saw nothing (no tokens, or scores of -inf alone) is zero.
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  *reinterpret_cast<f4*>(out + row * D + d) = o * inv;
  if (lse && d == 0)
    lse[row] = l == 0.0f ? -INFINITY : (m - shift + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// The join of a call of B rows of HQ (heads, or heads and queries), D 64, 128 or 256.
int join_shares(int D, int B, int HQ, int workgroups, const int32_t* row_pieces, float* partials, float* out, float* lse,
                float shift, hipStream_t st);

// ---------------------------------------------------------------------------
// Host checks that the page-pool entry points share.
// ---------------------------------------------------------------------------
constexpr int kMaxPageTokens = 1 << 24;

// Rows at p are read or written 16 bytes (align elements) at a time.
inline bool rows_ok(const void* p, const int64_t* strides, int n, int align) {
  if ((uintptr_t)p & 15) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] % align) return false;
  return true;
}

// A pool's rows are 16-byte pieces too; a page, head or token stride in them fits 32 bits, and
// so does the span of a tile of rows.
inline bool pool_ok(const void* p, const int64_t* strides, int align) {
  if (!p || !rows_ok(p, strides, 3, align)) return false;
  for (int i = 0; i < 3; ++i)
    if (strides[i] < 0 || strides[i] / align > UINT32_MAX) return false;
  return strides[2] > 0 && strides[2] < (int64_t(1) << 26);
}

// What the split kernels take of a plan and of the rows' room.
inline bool shares_ok(int B, int64_t max_pages, int64_t page_size, int least_chunks, int workgroups, int long_workgroups,
                      int long_chunks, const float* partials, const int32_t* row_pieces) {
  if (max_pages * page_size > INT32_MAX - 65536) return false;
  // the rows' chunks are summed in 32 bits
  if ((int64_t)B * (max_pages * page_size / 32 + 1) > INT32_MAX) return false;
  if (least_chunks <= 0 || workgroups < 0 || workgroups > 65535) return false;
  if (long_workgroups < 0 || long_workgroups > workgroups || long_chunks < 0 ||
      (int64_t)long_workgroups * long_chunks > INT32_MAX || (long_workgroups && !long_chunks))
    return false;
  if (!workgroups && B > 65535) return false;
  return !workgroups || (partials && !((uintptr_t)partials & 15) && row_pieces && !((uintptr_t)row_pieces & 7));
}

}  // namespace tkv
