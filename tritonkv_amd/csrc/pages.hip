// Bookkeeping of page pools on the device, for gfx950: copying pages, forking /
// truncating / growing / freeing rows of a block table over reference-counted
// pages, and moving the live pages to the low end of the pools.
//
// No formula here but the copies' bytes: a page that moves is read and written
// once in every tensor.  The plans are integers; each is made by one workgroup
// in one pass over the rows and one over the reference counts, so that a
// call is two launches and its result does not depend on any order: pages are
// handed out lowest first, in row order, by prefix sums, and the only atomics are
// integer sums, maxima and minima.
#include <hip/hip_runtime.h>

#include "launch.h"
#include "tkv_device.h"
#include "../../include/tkv.h"

namespace tkv {

constexpr int kPlan = 1024;                  // most threads of a plan's workgroup
constexpr int kSmallPlan = 256;              // ... where its rows and pages fit them
constexpr int kCopy = 1024;                  // threads of a copy's workgroup
constexpr int kMaxRows = 8192;               // rows of a fork: three LDS integers each, or four
constexpr int kInlinePairs = 4096;           // pairs that the copy checks by itself
constexpr int kPagesPerThread = 64;          // bits of a thread's mask of pages
constexpr int kMaxPages = 1 << 30;           // of a pool, and pairs of a call: sums of two fit an integer

// A barrier behind which the workgroup's memory operations have been carried out.
__device__ __forceinline__ void settle() {
  __builtin_amdgcn_s_waitcnt(0);  // vmcnt(0) expcnt(0) lgkmcnt(0)
  __syncthreads();
}

// ---------------------------------------------------------------------------
// The copy.  Item = one 16 KiB slice of one tensor's page (the last of a page may be
// less); the items of all pairs lie in a row, and workgroups stride over them RUN at
// a time: they read RUN slices whole before they write any of them.
//
// Bound by HBM, and by how its reads and writes alternate: 4000 scattered pages of 128
// KiB go at 5.9 TB/s in runs of 64 KiB by 1024 threads, at 5.1 in 16 KiB by 256 threads,
// at 5.2 in 64 KiB by 256; torch's copy_ of 2 GiB at 4.9.  Where a call copies less
// than 32 MiB, runs of one slice reach more CUs.  The bytes pass by the caches
// (non-temporal loads and stores: 4% on the large ones), except where a fork's rows
// share what they read: from three copies of a page on its loads keep it, in runs of
// 48 KiB.  126 MB from 16 rows to 15 others each take 38 us, 51 with non-temporal
// loads; 472 MB 89 and 158; with 7 copies of a page 108 and 139; with 3 the two are alike, with 2 the cached ones
// are 4% slower.
// ---------------------------------------------------------------------------
constexpr int kSlice = kCopy * 16;
constexpr int kRun = 4;
constexpr int kSharedRun = 3;
constexpr int64_t kLongCopy = 32 << 20;

// M: the most tensors.  Where a set has no more than kFewTensors the kernels take a
// smaller plan: 1.2 KB less of arguments save 0.3 us of every launch (8 pages of 512 KiB
// 3.6 -> 3.3 us captured, 5.2 -> 4.9 eager; a compaction of 1024 pages 8.8 -> 8.3 eager).
constexpr int kFewTensors = 4;

template <int M>
struct CopyPlan {
  static constexpr int kMost = M;
  const void* src[M];
  void* dst[M];
  int64_t src_stride[M], dst_stride[M], size[M];
  int32_t first[M];       // slices of a page before tensor t
  int32_t count, slices;  // tensors; slices of a page, in all of them
  int64_t bytes;          // of a page, in all tensors
};

// Pair p of the copies as (source, destination); a negative source is no pair.
// pair_of(p) may hold barriers: it is called by all threads alike.  CACHED: the loads
// keep what they read.
template <int RUN, bool CACHED, int M, class PairOf>
__device__ __forceinline__ void copy_run(const CopyPlan<M>& c, int64_t items, int group, int groups, PairOf pair_of) {
  for (int64_t base = (int64_t)group * RUN; base < items; base += (int64_t)groups * RUN) {
    int p = items <= UINT32_MAX ? (int)((uint32_t)base / (uint32_t)c.slices) : (int)(base / c.slices);
    int s = (int)(base - (int64_t)p * c.slices);
    int2 pair = pair_of(p);
    u4 x[RUN];
    u4* to[RUN];
#pragma unroll
    for (int i = 0; i < RUN; ++i) {
      to[i] = nullptr;
      if (base + i >= items) continue;
      if (i) {
        if (++s == c.slices) {
          s = 0;
          pair = pair_of(++p);
        }
      }
      if (pair.x < 0) continue;
      int t = 0;
#pragma unroll
      for (int step = M / 2; step; step /= 2)
        if (t + step < c.count && c.first[t + step] <= s) t += step;
      const int64_t at = (int64_t)(s - c.first[t]) * kSlice + threadIdx.x * 16;
      if (at >= c.size[t]) continue;
      const u4* from =
          reinterpret_cast<const u4*>(static_cast<const char*>(c.src[t]) + pair.x * c.src_stride[t] + at);
      x[i] = CACHED ? *from : __builtin_nontemporal_load(from);
      to[i] = reinterpret_cast<u4*>(static_cast<char*>(c.dst[t]) + pair.y * c.dst_stride[t] + at);
    }
#pragma unroll
    for (int i = 0; i < RUN; ++i)
      if (to[i]) __builtin_nontemporal_store(x[i], to[i]);
  }
}

// The first `count` of a plan's pairs, which read `sources` pages.
template <int M>
__device__ __forceinline__ void copy_pairs(const CopyPlan<M>& c, const int2* pairs, int count, int sources, int group,
                                           int groups) {
  const int64_t items = (int64_t)count * c.slices;
  auto pair_of = [&](int p) { return pairs[p]; };
  const bool shared = count >= 3 * sources;
  if (count * c.bytes < kLongCopy) copy_run<1, false>(c, items, group, groups, pair_of);
  else if (shared) copy_run<kSharedRun, true>(c, items, group, groups, pair_of);
  else copy_run<kRun, false>(c, items, group, groups, pair_of);
}

// tkv_copy_pages_args without its set.
struct PairLists {
  const int32_t *src, *dst;
  int32_t* work;
  int32_t n, src_pages, dst_pages, same;
};

// Whether the lists name a pair at all.
__device__ __forceinline__ bool is_pair(const PairLists& a, int s, int d) {
  return s >= 0 && s < a.src_pages && d >= 0 && d < a.dst_pages && !(a.same && s == d);
}

// A short copy: every workgroup checks its own pair against all of them, which saves
// the launch that checks them beforehand (below) and slows the copies down.  Pages of
// 128 KiB, inline / beforehand: 8 pairs 3.7 / 5.8 us, 64 5.8 / 8.4, 256 17.9 / 19.7, 1024
// 64 / 65; of 512 KiB: 8 4.4 / 6.6, 64 17.2 / 17.1, 256 60 / 56, 1024 213 / 196.  So
// inline below 32 MiB.  A pair is carried out unless an earlier one has its
// destination or, within one set of pools, any one reads it.
template <int M>
__global__ void __launch_bounds__(kCopy) copy_few_kernel(CopyPlan<M> c, PairLists a) {
  copy_run<1, false>(c, (int64_t)a.n * c.slices, blockIdx.x, gridDim.x, [&](int p) {
    const int s = a.src[p], d = a.dst[p];
    bool bad = !is_pair(a, s, d);
    for (int x = threadIdx.x; x < a.n; x += kCopy) {
      const int sx = a.src[x], dx = a.dst[x];
      if (is_pair(a, sx, dx) && ((x < p && dx == d) || (a.same && sx == d))) bad = true;
    }
    return make_int2(__syncthreads_or(bad) ? -1 : s, d);
  });
}

// Many pairs: the same rule in three passes of one workgroup over the pages
// that the pairs name (owner: the first pair of a destination; read: a source).  A
// thread's first pairs stay in registers.
constexpr int kKept = 4;

__global__ void __launch_bounds__(kPlan) copy_check_kernel(PairLists a) {
  int* owner = a.work;
  int* read = owner + a.dst_pages;
  const int64_t pages = (int64_t)a.dst_pages + a.src_pages;
  int2* pairs = reinterpret_cast<int2*>(a.work + pages + (pages & 1));
  int2 kept[kKept];
#pragma unroll
  for (int k = 0; k < kKept; ++k) {
    const int i = threadIdx.x + k * kPlan;
    kept[k] = i < a.n ? make_int2(a.src[i], a.dst[i]) : make_int2(-1, -1);
  }
  auto each = [&](auto take) {
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
      const int i = threadIdx.x + k * kPlan;
      if (i < a.n) take(i, kept[k].x, kept[k].y, is_pair(a, kept[k].x, kept[k].y));
    }
    for (int i = threadIdx.x + kKept * kPlan; i < a.n; i += kPlan) {
      const int s = a.src[i], d = a.dst[i];
      take(i, s, d, is_pair(a, s, d));
    }
  };
  each([&](int, int, int d, bool ok) {
    if (!ok) return;
    owner[d] = a.n;
    if (a.same) read[d] = 0;
  });
  settle();
  each([&](int i, int s, int d, bool ok) {
    if (!ok) return;
    atomicMin(owner + d, i);
    if (a.same) atomicExch(read + s, 1);
  });
  settle();
  each([&](int i, int s, int d, bool ok) {
    if (ok) {
      const int first = __hip_atomic_load(owner + d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const int taken = a.same ? __hip_atomic_load(read + d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
      ok = first == i && taken == 0;
    }
    pairs[i] = make_int2(ok ? s : -1, d);
  });
}

// head: a plan's (below), or null for n pairs of as many pages.
template <int M>
__global__ void __launch_bounds__(kCopy) copy_pairs_kernel(CopyPlan<M> c, const int2* pairs, const int* head, int n) {
  copy_pairs(c, pairs, head ? head[1] : n, head ? head[2] : n, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------------------
// Sums over a plan's workgroup.
// ---------------------------------------------------------------------------
template <int T>
struct ScanLds {
  int2 wave[T / 64];
};

// Exclusive sums of (x, y) over the threads before this one; total of both.
template <int T>
__device__ __forceinline__ int2 block_scan(ScanLds<T>& lds, int x, int y, int2& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int sx = x, sy = y;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int ox = __shfl_up(sx, off, 64), oy = __shfl_up(sy, off, 64);
    if (lane >= off) {
      sx += ox;
      sy += oy;
    }
  }
  __syncthreads();  // the previous scan's sums have been read
  if (lane == 63) lds.wave[w] = make_int2(sx, sy);
  __syncthreads();
  int2 before = make_int2(0, 0);
  total = make_int2(0, 0);
#pragma unroll
  for (int i = 0; i < T / 64; ++i) {
    const int2 v = lds.wave[i];
    if (i < w) {
      before.x += v.x;
      before.y += v.y;
    }
    total.x += v.x;
    total.y += v.y;
  }
  return make_int2(before.x + sx - x, before.y + sy - y);
}

// Bits of the pages p0 .. p0 + per - 1 (per <= 64) that are in use.
__device__ __forceinline__ uint64_t used_mask(const int32_t* __restrict__ refs, int64_t p0, int per, int N) {
  uint64_t m = 0;
  if (p0 + per <= N && per % 4 == 0 && (reinterpret_cast<uintptr_t>(refs + p0) & 15) == 0) {
#pragma unroll 4
    for (int i = 0; i < per; i += 4) {
      const int4 v = *reinterpret_cast<const int4*>(refs + p0 + i);
      m |= (uint64_t)((v.x > 0) | (v.y > 0) << 1 | (v.z > 0) << 2 | (v.w > 0) << 3) << i;
    }
  } else {
    for (int i = 0; i < per; ++i)
      if (p0 + i < N && refs[p0 + i] > 0) m |= uint64_t(1) << i;
  }
  return m;
}
__device__ __forceinline__ uint64_t first_bits(int64_t n) {
  return n <= 0 ? 0 : n >= 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1;
}
// Pages that one of `threads` takes of N in one round of the workgroup.
__host__ __device__ inline int pages_per_thread(int N, int threads) {
  const int per = ((N + threads - 1) / threads + 3) & ~3;
  return per < kPagesPerThread ? per : kPagesPerThread;
}

// ---------------------------------------------------------------------------
// Rows: row b becomes the first min(want_b, L_a) tokens of old row a =
// parents[b], with pages for want_b.  Of these keep = min(want_b, L_a, written_a)
// hold something: f = keep / page full pages, which are shared, and perhaps a
// partial one.  That page, and the room that a has after it, stays with one row
// (`heir`) if nobody else keeps it: it was a's alone, no other child of a keeps it as
// a full page, and of the children that end before it or in it the heir is a itself or
// the lowest; every other child copies the partial page to its first new page.  A page
// of unwritten room is never shared: two rows would write their own tokens into it.
// ---------------------------------------------------------------------------
// tkv_fork_written_args without its set.
struct RowsParams {
  int32_t *block_table, *seq_lens, *refs;
  const int32_t *parents, *new_lens, *written;
  int32_t *status, *work;
  int32_t table_stride, B, max_pages, page_size, num_pages;
};

struct RowsWork {  // a.work, in int32
  int* head;       // status, copies, pages that they read
  int *old_len, *kept, *first, *pages;
  int2* pairs;
  int *fresh, *staged;
};

__host__ __device__ inline int64_t rows_work_ints(int64_t B, int64_t P, int64_t N, bool staged) {
  return 16 + 6 * B + N + (staged ? B * P : 0);
}

__device__ __forceinline__ RowsWork rows_work(const RowsParams& a) {
  RowsWork w;
  int* p = a.work;
  w.head = p;
  w.pairs = reinterpret_cast<int2*>(p + 16);
  w.old_len = p + 16 + 2 * a.B;
  w.kept = w.old_len + a.B;
  w.first = w.kept + a.B;
  w.pages = w.first + a.B;
  w.fresh = w.pages + a.B;
  w.staged = w.fresh + a.num_pages;
  return w;
}

struct Row {
  int a, want, f;  // parent (-1: none), tokens, full pages kept
  int tail, last;  // old pages after them, as far as the row reaches, and the first of them in the pools
  bool rest;       // ... of which some tokens are kept
};

__device__ __forceinline__ int table_tokens(const RowsParams& a) { return a.max_pages * a.page_size; }

// WRITTEN: a.written is given.  (Without it the plan of a beam step is 0.3 us shorter for not
// looking.)
template <bool WRITTEN>
__device__ __forceinline__ Row row_of(const RowsParams& a, int b) {
  Row r;
  r.a = a.parents ? a.parents[b] : b;
  if (r.a < 0 || r.a >= a.B) r.a = -1;
  const int have = r.a < 0 ? 0 : max(0, min(a.seq_lens[r.a], table_tokens(a)));
  r.want = r.a < 0 ? 0 : a.new_lens ? max(0, a.new_lens[b]) : have;
  const int reach = min(have, r.want);
  const int keep = WRITTEN && r.a >= 0 ? min(reach, max(0, a.written[r.a])) : reach;
  r.f = keep / a.page_size;
  r.rest = keep % a.page_size != 0;
  r.tail = r.rest;
  if (WRITTEN) r.tail = reach / a.page_size + (reach % a.page_size != 0) - r.f;
  r.last = r.tail ? a.block_table[(int64_t)r.a * a.table_stride + r.f] : -1;
  return r;
}

// The slot after the pages that the heir of each parent a keeps: end[a], and before it that of
// the first page from first[a] + 1 on (the first one was looked at) that is not a's alone.
// A wave looks at 64 pages of each of kTails parents at a time: 32 rows with 250 pages of room
// each take 13.7 us a call (70.6 with a thread that follows its own row), one row with 8190 73 (1430).
constexpr int kTails = 4;

template <int T>
__device__ __forceinline__ void own_tails(const RowsParams& a, const int* first, int* end) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int p0 = kTails * w; p0 < a.B; p0 += kTails * (T / 64)) {
    int from[kTails], to[kTails];
#pragma unroll
    for (int k = 0; k < kTails; ++k) {
      from[k] = p0 + k < a.B ? first[p0 + k] + 1 : 0;
      to[k] = p0 + k < a.B ? end[p0 + k] : 0;
    }
    for (bool more = true; more;) {
      int page[kTails];
      bool own[kTails];
#pragma unroll
      for (int k = 0; k < kTails; ++k)
        page[k] = from[k] + lane < to[k] ? a.block_table[(int64_t)(p0 + k) * a.table_stride + from[k] + lane] : -1;
#pragma unroll
      for (int k = 0; k < kTails; ++k) own[k] = page[k] >= 0 && page[k] < a.num_pages && a.refs[page[k]] == 1;
      more = false;
#pragma unroll
      for (int k = 0; k < kTails; ++k) {
        const uint64_t other = __builtin_amdgcn_ballot_w64(from[k] + lane < to[k] && !own[k]);
        if (other) {
          to[k] = from[k] + __builtin_ctzll(other);
          if (lane == 0) end[p0 + k] = to[k];
        }
        from[k] += 64;
        more |= from[k] < to[k];
      }
    }
  }
}

template <int T, bool WRITTEN>
__global__ void __launch_bounds__(T) rows_plan_kernel(RowsParams a) {
  extern __shared__ int lds[];
  __shared__ ScanLds<T> scan;
  __shared__ int past;
  const RowsWork w = rows_work(a);
  const int tid = threadIdx.x, B = a.B, P = a.max_pages, N = a.num_pages;
  if (blockIdx.x > 0) {
    // The rows' old pages, which the second launch reads while it writes the table.
    for (int64_t i = (int64_t)(blockIdx.x - 1) * T + tid; i < (int64_t)B * P; i += (int64_t)(gridDim.x - 1) * T) {
      const int b = (int)(i / P);
      w.staged[i] = a.block_table[(int64_t)b * a.table_stride + (i - (int64_t)b * P)];
    }
    return;
  }
  int *most = lds, *best = lds + B, *copied = lds + 2 * B, *end = lds + 3 * B;  // end: if WRITTEN
  for (int b = tid; b < B; b += T) {
    most[b] = -1;
    best[b] = B;
    copied[b] = 0;
    if (WRITTEN) end[b] = 0;
  }
  if (tid == 0) past = 0;
  // This thread's first row and first pages stay in registers: most plans need no others.
  const int per = pages_per_thread(N, T);
  const uint64_t mask0 = used_mask(a.refs, (int64_t)tid * per, per, N);
  Row row0{-1, 0, 0, 0, -1, false};
  int owners0 = 0;  // references of the first page of its tail
  if (tid < B) {
    row0 = row_of<WRITTEN>(a, tid);
    if (row0.last >= 0 && row0.last < N) owners0 = a.refs[row0.last];
  }
  __syncthreads();
  for (int b = tid; b < B; b += T) {
    const Row r = b == tid ? row0 : row_of<WRITTEN>(a, b);
    if (r.a >= 0) atomicMax(most + r.a, r.f);
    if (r.want > table_tokens(a)) past = 1;
  }
  __syncthreads();
  auto may_inherit = [&](const Row& r, int b) {
    if (!r.tail || r.f != most[r.a] || r.last < 0 || r.last >= N) return false;
    return (b == tid ? owners0 : a.refs[r.last]) == 1;
  };
  for (int b = tid; b < B; b += T) {
    const Row r = b == tid ? row0 : row_of<WRITTEN>(a, b);
    if (may_inherit(r, b)) atomicMin(best + r.a, r.a == b ? -1 : b);
  }
  __syncthreads();
  auto is_heir = [&](const Row& r, int b) { return may_inherit(r, b) && best[r.a] == (r.a == b ? -1 : b); };
  if (WRITTEN) {
    bool room = false;
    for (int b = tid; b < B; b += T) {
      const Row r = b == tid ? row0 : row_of<WRITTEN>(a, b);
      if (!is_heir(r, b)) continue;
      end[r.a] = r.f + r.tail;
      room |= r.tail > 1;
    }
    if (__syncthreads_or(room)) {
      own_tails<T>(a, most, end);
      __syncthreads();
    }
  }
  const bool too_long = past != 0;
  // New pages and copies (below 2^16 of them) of the rows taken so far, and in the
  // copies' upper half the parents that they read from.
  int2 done = make_int2(0, 0);
  constexpr int kCopies = 0xffff;
  for (int b0 = 0; b0 < B; b0 += T) {
    const int b = b0 + tid;
    Row r;
    int need = 0, pages = 0, inherited = 0;
    bool copy = false;
    if (b < B) {
      r = b == tid ? row0 : row_of<WRITTEN>(a, b);
      if (is_heir(r, b)) inherited = WRITTEN ? end[r.a] - r.f : 1;
      pages = (int)(((int64_t)r.want + a.page_size - 1) / a.page_size);
      // (a row that does not fit its table asks for nothing: the call fails)
      need = too_long ? 0 : pages - r.f - inherited;
      copy = !too_long && r.rest && !inherited;
    }
    int2 total;
    const int first_copy = copy && atomicExch(copied + r.a, 1) == 0 ? kCopies + 1 : 0;
    const int2 at = block_scan(scan, need, copy ? 1 + first_copy : 0, total);
    if (b < B) {
      w.old_len[b] = max(0, min(a.seq_lens[b], table_tokens(a)));
      w.kept[b] = r.f + inherited;
      w.first[b] = done.x + at.x;
      w.pages[b] = pages;
      if (copy) w.pairs[(done.y + at.y) & kCopies] = make_int2(r.last, done.x + at.x);
    }
    done.x += total.x;
    done.y += total.y;
  }
  // The lowest free pages.
  int found = 0;
  for (int64_t p0 = 0; p0 < N && found < done.x; p0 += (int64_t)per * T) {
    const int64_t mine = p0 + (int64_t)tid * per;
    uint64_t m = ~(p0 ? used_mask(a.refs, mine, per, N) : mask0) & first_bits(N - mine) & first_bits(per);
    int2 total;
    int at = found + block_scan(scan, __popcll(m), 0, total).x;
    for (; m && at < done.x; m &= m - 1) w.fresh[at++] = (int)(mine + __builtin_ctzll(m));
    found += total.x;
  }
  const int status = too_long ? TKV_ROWS_PAST_TABLE : found < done.x ? TKV_ROWS_NO_PAGES : TKV_ROWS_DONE;
  settle();
  const int copies = status ? 0 : done.y & kCopies;
  for (int i = tid; i < copies; i += T) {
    int2 p = w.pairs[i];
    p.y = w.fresh[p.y];
    if (p.x >= N) p.x = -1;  // the table names no page there
    w.pairs[i] = p;
  }
  if (tid == 0) {
    w.head[0] = status;
    w.head[1] = copies;
    w.head[2] = done.y >> 16;
    *a.status = status;
  }
}

// Workgroups [0, tables): the table, lengths and counts; the others: the copies.
template <int M>
__global__ void __launch_bounds__(kCopy) rows_apply_kernel(RowsParams a, CopyPlan<M> c, int tables) {
  const RowsWork w = rows_work(a);
  if (w.head[0] != TKV_ROWS_DONE) return;
  if ((int)blockIdx.x >= tables) {
    copy_pairs(c, w.pairs, w.head[1], w.head[2], blockIdx.x - tables, gridDim.x - tables);
    return;
  }
  const int P = a.max_pages, N = a.num_pages;
  const int64_t entries = (int64_t)a.B * P;
  for (int64_t i = (int64_t)blockIdx.x * kCopy + threadIdx.x; i < entries; i += (int64_t)tables * kCopy) {
    const int b = (int)(i / P), slot = (int)(i - (int64_t)b * P);
    int* at = a.block_table + (int64_t)b * a.table_stride + slot;
    const int old = *at, kept = w.kept[b], pages = w.pages[b];
    int now = -1;
    if (slot < kept) {
      const int from = a.parents ? a.parents[b] : b;
      now = a.parents ? w.staged[(int64_t)from * P + slot] : old;
    } else if (slot < pages) {
      now = w.fresh[w.first[b] + slot - kept];
    }
    const int was = (w.old_len[b] + a.page_size - 1) / a.page_size;
    const int dec = slot < was && old >= 0 && old < N ? old : -1;
    const int inc = slot < pages && now >= 0 && now < N ? now : -1;
    if (dec != inc) {
      if (dec >= 0) atomicSub(a.refs + dec, 1);
      if (inc >= 0) atomicAdd(a.refs + inc, 1);
    }
    if (now != old) *at = now;
    if (slot == 0) {
      const bool none = a.parents && (a.parents[b] < 0 || a.parents[b] >= a.B);
      const int len = a.new_lens ? (none ? 0 : max(0, a.new_lens[b]))
                      : a.parents ? (none ? 0 : w.old_len[a.parents[b]]) : w.old_len[b];
      a.seq_lens[b] = len;
    }
  }
}

// ---------------------------------------------------------------------------
// Compaction: with n live pages (refs > 0), the i-th live page at or past n moves
// to the i-th free page below n.
// ---------------------------------------------------------------------------
// tkv_compact_pages_args without its set.
struct CompactParams {
  const int32_t *block_table, *refs;
  int32_t *out_table, *out_refs, *live, *work;
  int32_t table_stride, out_stride, B, max_pages, num_pages, per;  // per: pages of a thread's block
};

// The plan's blocks: the pages of one thread in one round.
struct PageBlock {
  uint64_t used;  // bit i: page i of the block has references
  int from, to;   // pages before the block that move, and that are moved onto
};

struct CompactWork {
  int* head;          // live pages, moves, pages that they read
  int2* pairs;        // at most N / 2 moves
  int* refs;          // the counts before the call
  PageBlock* blocks;  // of per >= 4 pages each
};

__host__ __device__ inline int64_t compact_refs_at(int64_t N) { return 16 + (N + 4) / 4 * 4; }
__host__ __device__ inline int64_t compact_blocks_at(int64_t N) { return compact_refs_at(N) + (N + 4) / 4 * 4; }
__host__ __device__ inline int64_t compact_work_ints(int64_t N) {
  return compact_blocks_at(N) + 4 * (N / 4 + kPlan);
}

__device__ __forceinline__ CompactWork compact_work(const CompactParams& a) {
  CompactWork w;
  w.head = a.work;
  w.pairs = reinterpret_cast<int2*>(a.work + 16);
  w.refs = a.work + compact_refs_at(a.num_pages);
  w.blocks = reinterpret_cast<PageBlock*>(a.work + compact_blocks_at(a.num_pages));
  return w;
}

template <int T>
__global__ void __launch_bounds__(T) compact_plan_kernel(CompactParams a) {
  __shared__ ScanLds<T> scan;
  const CompactWork w = compact_work(a);
  const int tid = threadIdx.x, N = a.num_pages, per = a.per;
  if (blockIdx.x > 0) {
    // The second launch reads the counts while it writes them.
    for (int64_t i = (int64_t)(blockIdx.x - 1) * T + tid; i < N; i += (int64_t)(gridDim.x - 1) * T) w.refs[i] = a.refs[i];
    return;
  }
  const int64_t round = (int64_t)per * T;
  int live = 0;
  uint64_t m = 0;
  for (int64_t p0 = 0; p0 < N; p0 += round) {
    m = used_mask(a.refs, p0 + (int64_t)tid * per, per, N);
    int2 total;
    block_scan(scan, __popcll(m), 0, total);
    live += total.x;
  }
  int2 done = make_int2(0, 0);
  for (int64_t p0 = 0; p0 < N; p0 += round) {
    const int64_t mine = p0 + (int64_t)tid * per;
    if (N > round) m = used_mask(a.refs, mine, per, N);
    const uint64_t low = first_bits(live - mine), in = first_bits(N - mine) & first_bits(per);
    uint64_t from = m & ~low, to = ~m & low & in;
    int2 total;
    const int2 at = block_scan(scan, __popcll(from), __popcll(to), total);
    int s = done.x + at.x, d = done.y + at.y;
    if (mine < N) w.blocks[p0 / per + tid] = PageBlock{m, s, d};
    for (; from; from &= from - 1, ++s) w.pairs[s].x = (int)mine + __builtin_ctzll(from);
    for (; to; to &= to - 1, ++d) w.pairs[d].y = (int)mine + __builtin_ctzll(to);
    done.x += total.x;
    done.y += total.y;
  }
  if (tid == 0) {
    w.head[0] = live;
    w.head[1] = w.head[2] = done.x;
    if (a.live) *a.live = live;
  }
}

// Which move a page takes part in, -1 for none: as the source of one at or past
// `live` pages, as the destination of one below.
__device__ __forceinline__ int move_of(const CompactWork& w, int page, int per, int live) {
  const int block = page / per, bit = page - block * per;
  const PageBlock b = w.blocks[block];
  const uint64_t below = first_bits(bit), low = first_bits((int64_t)live - (int64_t)block * per);
  const bool used = b.used >> bit & 1;
  if (page >= live) return used ? b.from + __popcll(b.used & ~low & below) : -1;
  return used ? -1 : b.to + __popcll(~b.used & low & below);
}

// Workgroups [0, tables): the table and the counts; the others: the copies.
template <int M>
__global__ void __launch_bounds__(kCopy) compact_apply_kernel(CompactParams a, CopyPlan<M> c, int tables) {
  const CompactWork w = compact_work(a);
  const int live = w.head[0];
  if ((int)blockIdx.x >= tables) {
    copy_pairs(c, w.pairs, w.head[1], w.head[2], blockIdx.x - tables, gridDim.x - tables);
    return;
  }
  const int P = a.max_pages, N = a.num_pages, per = a.per;
  const int64_t entries = (int64_t)a.B * P;
  for (int64_t i = (int64_t)blockIdx.x * kCopy + threadIdx.x; i < entries + N; i += (int64_t)tables * kCopy) {
    if (i < entries) {
      const int b = (int)(i / P), slot = (int)(i - (int64_t)b * P);
      int page = a.block_table[(int64_t)b * a.table_stride + slot];
      const int move = page >= live && page < N ? move_of(w, page, per, live) : -1;
      if (move >= 0) page = w.pairs[move].y;
      a.out_table[(int64_t)b * a.out_stride + slot] = page;
    } else {
      const int p = (int)(i - entries);
      const int move = p < live ? move_of(w, p, per, live) : -1;
      a.out_refs[p] = p >= live ? 0 : w.refs[move >= 0 ? w.pairs[move].x : p];
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
using FullPlan = CopyPlan<TKV_PAGE_TENSORS>;

static int make_plan(const tkv_page_set& s, FullPlan& c) {
  if (s.count < 0 || s.count > TKV_PAGE_TENSORS) return TKV_EINVAL;
  c.count = s.count;
  c.bytes = 0;
  int64_t slices = 0;
  for (int t = 0; t < s.count; ++t) {
    if (!s.src[t] || !s.dst[t] || s.bytes[t] <= 0) return TKV_EINVAL;
    if (((uintptr_t)s.src[t] | (uintptr_t)s.dst[t] | (uint64_t)s.bytes[t] | (uint64_t)s.src_stride[t] |
         (uint64_t)s.dst_stride[t]) & 15)
      return TKV_EINVAL;
    if (s.src_stride[t] < s.bytes[t] || s.dst_stride[t] < s.bytes[t]) return TKV_EINVAL;
    c.src[t] = s.src[t];
    c.dst[t] = s.dst[t];
    c.src_stride[t] = s.src_stride[t];
    c.dst_stride[t] = s.dst_stride[t];
    c.size[t] = s.bytes[t];
    c.first[t] = (int32_t)slices;
    slices += (s.bytes[t] + kSlice - 1) / kSlice;
    if (slices > INT32_MAX) return TKV_EUNSUPPORTED;
    c.bytes += s.bytes[t];
  }
  c.slices = (int32_t)slices;
  return TKV_OK;
}

// start(plan) with the plan that the kernels take.
template <class Start>
static int with_plan(const FullPlan& c, Start start) {
  if (c.count > kFewTensors) return start(c);
  CopyPlan<kFewTensors> few;
  for (int t = 0; t < c.count; ++t) {
    few.src[t] = c.src[t];
    few.dst[t] = c.dst[t];
    few.src_stride[t] = c.src_stride[t];
    few.dst_stride[t] = c.dst_stride[t];
    few.size[t] = c.size[t];
    few.first[t] = c.first[t];
  }
  few.count = c.count;
  few.slices = c.slices;
  few.bytes = c.bytes;
  return start(few);
}

constexpr int kCopyGroups = 8192;  // workgroups that stride over the copies

// Workgroups for at most `pairs` copies.
static unsigned copy_groups(int64_t pairs, const FullPlan& c) {
  const int64_t items = pairs * c.slices;
  return (unsigned)(items < kCopyGroups ? items : kCopyGroups);
}

static int check_copy(const tkv_copy_pages_args* a, FullPlan& c) {
  if (!a || !a->src || !a->dst || a->n <= 0 || a->src_pages <= 0 || a->dst_pages <= 0) return TKV_EINVAL;
  if (a->n > kMaxPages || a->src_pages > kMaxPages || a->dst_pages > kMaxPages) return TKV_EUNSUPPORTED;
  if (a->same && a->src_pages != a->dst_pages) return TKV_EINVAL;
  return make_plan(a->set, c);
}

static bool checked_inline(const tkv_copy_pages_args* a, const FullPlan& c) {
  return a->n <= kInlinePairs && a->n * c.bytes < kLongCopy;
}

}  // namespace tkv

extern "C" int64_t tkv_copy_pages_work(const tkv_copy_pages_args* a) {
  using namespace tkv;
  FullPlan c;
  const int rc = check_copy(a, c);
  if (rc) return rc;
  return checked_inline(a, c) ? 0 : (int64_t)a->src_pages + a->dst_pages + 1 + 2 * (int64_t)a->n;
}

extern "C" int tkv_copy_pages(const tkv_copy_pages_args* a, tkv_stream_t stream) {
  using namespace tkv;
  FullPlan c;
  const int rc = check_copy(a, c);
  if (rc) return rc;
  const bool in_line = checked_inline(a, c);
  if (!in_line && (!a->work || (uintptr_t)a->work & 7)) return TKV_EINVAL;
  if (!c.slices) return TKV_OK;
  const PairLists p{a->src, a->dst, a->work, a->n, a->src_pages, a->dst_pages, a->same};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(copy_groups(a->n, c)), block(kCopy);
  if (in_line)
    return with_plan(c, [&](auto plan) { return launch(copy_few_kernel<plan.kMost>, grid, block, 0, st, plan, p); });
  const int64_t pages = (int64_t)a->dst_pages + a->src_pages;
  const int2* pairs = reinterpret_cast<const int2*>(a->work + pages + (pages & 1));
  const int bad = launch(copy_check_kernel, dim3(1), dim3(kPlan), 0, st, p);
  if (bad) return bad;
  return with_plan(c, [&](auto plan) {
    return launch(copy_pairs_kernel<plan.kMost>, grid, block, 0, st, plan, pairs, (const int*)nullptr, (int)a->n);
  });
}

extern "C" int64_t tkv_fork_rows_work(int32_t B, int32_t max_pages, int32_t num_pages, int32_t parents) {
  if (B <= 0 || max_pages <= 0 || num_pages <= 0) return -1;
  return tkv::rows_work_ints(B, max_pages, num_pages, parents != 0);
}

static int fork_rows(const tkv_fork_rows_args* a, const int32_t* written, tkv_stream_t stream) {
  using namespace tkv;
  if (!a || !a->block_table || !a->seq_lens || !a->refs || !a->status || !a->work || (uintptr_t)a->work & 7)
    return TKV_EINVAL;
  if (a->B <= 0 || a->max_pages <= 0 || a->num_pages <= 0 || a->page_size <= 0 || a->table_stride < a->max_pages)
    return TKV_EINVAL;
  if (a->B > kMaxRows || a->num_pages > kMaxPages) return TKV_EUNSUPPORTED;
  if ((int64_t)a->max_pages * a->page_size > INT32_MAX || (int64_t)a->B * a->max_pages > INT32_MAX) return TKV_EINVAL;
  FullPlan c;
  const int rc = make_plan(a->set, c);
  if (rc) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t entries = (int64_t)a->B * a->max_pages;
  // Small plans take 4 waves: barriers and prefix sums over 16 cost 1 us more.
  const bool small = a->B <= kSmallPlan && a->num_pages <= 16 * kSmallPlan;
  const int threads = small ? kSmallPlan : kPlan;
  const unsigned staging = a->parents ? (unsigned)((entries + 4 * threads - 1) / (4 * threads)) : 0;
  const RowsParams p{a->block_table, a->seq_lens, a->refs, a->parents, a->new_lens, written, a->status, a->work,
                     a->table_stride, a->B, a->max_pages, a->page_size, a->num_pages};
  const auto plan_kernel = small ? (written ? rows_plan_kernel<kSmallPlan, true> : rows_plan_kernel<kSmallPlan, false>)
                                 : (written ? rows_plan_kernel<kPlan, true> : rows_plan_kernel<kPlan, false>);
  const int bad = launch(plan_kernel, dim3(1 + (staging < 512 ? staging : 512)), dim3(threads),
                         (written ? 4 : 3) * sizeof(int) * a->B, st, p);
  if (bad) return bad;
  const int64_t tables = (entries + kCopy - 1) / kCopy;
  const int t = (int)(tables < 512 ? tables : 512);
  return with_plan(c, [&](auto plan) {
    return launch(rows_apply_kernel<plan.kMost>, dim3(t + copy_groups(a->B, c)), dim3(kCopy), 0, st, p, plan, t);
  });
}

extern "C" int tkv_fork_rows(const tkv_fork_rows_args* a, tkv_stream_t stream) { return fork_rows(a, nullptr, stream); }

extern "C" int tkv_fork_rows_written(const tkv_fork_written_args* a, tkv_stream_t stream) {
  return a ? fork_rows(&a->rows, a->written, stream) : TKV_EINVAL;
}

extern "C" int64_t tkv_compact_pages_work(int32_t num_pages) {
  return num_pages <= 0 ? -1 : tkv::compact_work_ints(num_pages);
}

extern "C" int tkv_compact_pages(const tkv_compact_pages_args* a, tkv_stream_t stream) {
  using namespace tkv;
  if (!a || !a->block_table || !a->refs || !a->out_table || !a->out_refs || !a->work || (uintptr_t)a->work & 15)
    return TKV_EINVAL;
  if (a->B <= 0 || a->max_pages <= 0 || a->num_pages <= 0 || a->table_stride < a->max_pages ||
      a->out_stride < a->max_pages)
    return TKV_EINVAL;
  if (a->num_pages > kMaxPages) return TKV_EUNSUPPORTED;
  FullPlan c;
  const int rc = make_plan(a->set, c);
  if (rc) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool small = a->num_pages <= 16 * kSmallPlan;  // (more pages: more threads to share them)
  const int threads = small ? kSmallPlan : kPlan;
  const CompactParams p{a->block_table, a->refs, a->out_table, a->out_refs, a->live, a->work,
                        a->table_stride, a->out_stride, a->B, a->max_pages, a->num_pages,
                        pages_per_thread(a->num_pages, threads)};
  const int staging = (a->num_pages + 4 * threads - 1) / (4 * threads);
  const int bad = launch(small ? compact_plan_kernel<kSmallPlan> : compact_plan_kernel<kPlan>,
                         dim3(1 + (staging < 512 ? staging : 512)), dim3(threads), 0, st, p);
  if (bad) return bad;
  const int64_t tables = ((int64_t)a->B * a->max_pages + a->num_pages + kCopy - 1) / kCopy;
  const int t = (int)(tables < 512 ? tables : 512);
  return with_plan(c, [&](auto plan) {
    return launch(compact_apply_kernel<plan.kMost>, dim3(t + copy_groups(a->num_pages / 2, c)), dim3(kCopy), 0, st, p,
                  plan, t);
  });
}

// The copies of a plan in further tensors: pairs and their count as the plan left them.
extern "C" int tkv_copy_planned(const tkv_page_set* set, const int32_t* work, int32_t most, tkv_stream_t stream) {
  using namespace tkv;
  if (!set || !work || (uintptr_t)work & 7 || most < 0) return TKV_EINVAL;
  FullPlan c;
  const int rc = make_plan(*set, c);
  if (rc) return rc;
  const unsigned groups = copy_groups(most, c);
  if (!groups) return TKV_OK;
  return with_plan(c, [&](auto plan) {
    return launch(copy_pairs_kernel<plan.kMost>, dim3(groups), dim3(kCopy), 0, reinterpret_cast<hipStream_t>(stream),
                  plan, reinterpret_cast<const int2*>(work + 16), (const int*)work, 0);
  });
}
