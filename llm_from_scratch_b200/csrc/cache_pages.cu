// Pages of a paged cache: copies (forks, moves) and compaction.
//
// A cache is a set of pools, one per layer and kind of row, that share page ids: page i of every pool belongs to the same tokens.
// Copy: page target[j] of every pool becomes page source[j]; pairs with a negative id are left out.  The copies of a call run in no order, so
// a pair whose target is also a source of the call, or the target of an earlier pair, is not carried out and reported: every CTA looks
// through the pairs for its own one's, or, beyond kLookedThrough of them, a kernel in front marks the pages.
// Compaction: with L pages in use (named in a block table), the pages in use from id L on move, in ascending order, to the unused ids
// below L, in ascending order.  What moves is never a target and the old places keep their contents, so all copies may run at once.
//
// Bound by the bytes: every page is read and written once (a compaction that moves 975 pages of 32 KB in
// 16 pools, 1.02 GB: 166 us, 6.2 TB/s).  A CTA copies 32 KB of a page, all loads of a thread ahead of its stores; the CTAs of
// a pool start before those of the next, so that a page which goes to several targets is mostly read from L2 after the first time.
#include "common.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256;
// Measured (us, every CTA looks / marks in front): 64 pairs of a pool with pages of 32 KB 3.2 / 5.2, 1,024 8.7 / 10.9, 8,192 87 / 84; 48 pools with
// pages of 8 KB, 64 pairs 10 / 12, 1,024 171 / 158, 4,096 906 / 631; 2 pools with pages of 4 KB, 1,024 pairs 7.8 / 9.4, 2,048 16 / 14.
constexpr int kLookedThrough = 1024;

struct CopyArgs {
  const int64_t* pools;      // [num_pools] addresses
  const int64_t* bytes;      // [num_pools] bytes of a page
  const int32_t* source;
  const int32_t* target;
  const int32_t* count;      // pairs, or null: all
  int n, num_pools;
  int pieces;                // of a page, in the pool with the largest
  bool look;                 // through all pairs for conflicts
  const int32_t* first;      // or in what mark_pairs_kernel left; null: there are none
  int64_t num_pages;
  int32_t* status;
};

__device__ __forceinline__ bool in_pool(int id, int64_t num_pages) {
  return static_cast<uint64_t>(static_cast<int64_t>(id)) < static_cast<uint64_t>(num_pages);
}

// Pair j against all pairs, by the CTA.
__device__ __forceinline__ bool conflicts(int to, int j, const int32_t* source, const int32_t* target, int n) {
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int other_from = source[i], other = target[i];
    if (other_from < 0 || other < 0) continue;
    bad |= (other_from == to && other != to) || (other == to && i < j);
  }
  return __syncthreads_or(bad);
}

constexpr int kNoPair = 0x7f7f7f7f;

// first (kNoPair before): per page the first pair that it is the target of, -1 for sources.  Pair j may go on if first[target] == j.
__global__ void __launch_bounds__(kThreads) mark_pairs_kernel(const int32_t* source, const int32_t* target, int n, int64_t num_pages, int32_t* first) {
  const int j = blockIdx.x * kThreads + threadIdx.x;
  if (j >= n) return;
  const int from = source[j], to = target[j];
  if (from < 0 || to < 0) return;
  if (in_pool(to, num_pages)) atomicMin(&first[to], j);
  if (from != to && in_pool(from, num_pages)) atomicMin(&first[from], -1);
}

constexpr int kPiece = 32768, kDeep = kPiece / (kThreads * 16);      // bytes of a CTA, 16-byte loads of a thread

// Items are pieces of pairs; blockIdx.y: the pool.
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const CopyArgs a) {
  const int pool = blockIdx.y, n = a.count ? min(*a.count, a.n) : a.n;
  const int64_t bytes = a.bytes[pool];
  uint8_t* base = reinterpret_cast<uint8_t*>(a.pools[pool]);
  const uintptr_t grain = reinterpret_cast<uintptr_t>(base) | static_cast<uintptr_t>(bytes);
  const int pieces = a.pieces;
  for (int64_t item = blockIdx.x; item < static_cast<int64_t>(n) * pieces; item += gridDim.x) {
    const int j = static_cast<int>(item / pieces);
    const int64_t at = item % pieces * kPiece, left = bytes - at;
    const int from = a.source[j], to = a.target[j];
    if (from < 0 || to < 0 || from == to) continue;
    if (!in_pool(from, a.num_pages) || !in_pool(to, a.num_pages)) {
      if (threadIdx.x == 0) report(a.status, B200_ERR_BOUNDS);
      continue;
    }
    if (a.look ? conflicts(to, j, a.source, a.target, n) : a.first != nullptr && a.first[to] != j) {
      if (threadIdx.x == 0) report(a.status, B200_ERR_ARG);
      continue;
    }
    if (left <= 0) continue;
    const uint8_t* src = base + from * bytes + at;
    uint8_t* dst = base + to * bytes + at;
    const int size = static_cast<int>(left < kPiece ? left : kPiece);
    if (grain % 16 == 0) {
      uint4 v[kDeep];
#pragma unroll
      for (int c = 0; c < kDeep; ++c) {
        const int i = (threadIdx.x + c * kThreads) * 16;
        if (i < size) v[c] = *reinterpret_cast<const uint4*>(src + i);
      }
#pragma unroll
      for (int c = 0; c < kDeep; ++c) {
        const int i = (threadIdx.x + c * kThreads) * 16;
        if (i < size) __stcs(reinterpret_cast<uint4*>(dst + i), v[c]);
      }
    } else if (grain % 4 == 0) {
      for (int i = threadIdx.x * 4; i < size; i += kThreads * 4) *reinterpret_cast<uint32_t*>(dst + i) = *reinterpret_cast<const uint32_t*>(src + i);
    } else {
      for (int i = threadIdx.x; i < size; i += kThreads) dst[i] = src[i];
    }
  }
}

// page_map (zeros before): 1 for the pages in use
__global__ void __launch_bounds__(kThreads) mark_pages_kernel(const int32_t* tables, int64_t row_stride, int64_t rows, int width,
                                                              int64_t num_pages, int32_t* page_map, int32_t* status) {
  const int64_t total = rows * width;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int id = tables[i / width * row_stride + i % width];
    if (in_pool(id, num_pages)) page_map[id] = 1;
    else if (id >= 0) report(status, B200_ERR_BOUNDS);
  }
}

constexpr int kPlanThreads = 1024;

// Inclusive sum over the CTA.
__device__ __forceinline__ int block_sum_upto(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    before += w < warp ? s_warp[w] : 0;
    all += s_warp[w];
  }
  *total = all;
  return v + before;
}

// page_map: marks -> new ids (-1: unused); source / target: the moves; counts: pages in use, moves.  One CTA, a run of pages per thread.
__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(int32_t* page_map, int num_pages, int32_t* source, int32_t* target,
                                                                  int32_t* counts) {
  __shared__ int s_warp[kPlanThreads / 32];
  // in 64 bits: pools may have up to 2^31 - 1 pages
  const int64_t pages = num_pages, per = (pages + kPlanThreads - 1) / kPlanThreads, begin = threadIdx.x * per;
  const int lo = static_cast<int>(min(begin, pages)), hi = static_cast<int>(min(begin + per, pages));
  int mine = 0, live, moves;
  for (int i = lo; i < hi; ++i) mine += page_map[i];
  block_sum_upto(mine, s_warp, &live);
  int holes = 0, movers = 0;
  for (int i = lo; i < hi; ++i) (i < live ? holes : movers) += i < live ? !page_map[i] : page_map[i];
  int hole = block_sum_upto(holes, s_warp, &moves) - holes, mover = block_sum_upto(movers, s_warp, &moves) - movers;
  for (int i = lo; i < hi; ++i) {
    const bool used = page_map[i];
    if (i < live && !used) target[hole++] = i;
    if (i >= live && used) source[mover++] = i;
    page_map[i] = used && i < live ? i : -1;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < moves; j += kPlanThreads) page_map[source[j]] = target[j];
  if (threadIdx.x == 0) counts[0] = live, counts[1] = moves;
}

__global__ void __launch_bounds__(kThreads) rename_pages_kernel(const int32_t* tables, int64_t row_stride, int64_t rows, int width,
                                                                int64_t num_pages, const int32_t* page_map, int32_t* out) {
  const int64_t total = rows * width;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int id = tables[i / width * row_stride + i % width];
    out[i] = in_pool(id, num_pages) ? page_map[id] : -1;
  }
}

// The whole plan in one CTA, for pools of up to kOnePages pages and up to kOneEntries table entries: the pages in use as bits of shared memory.
constexpr int kOnePages = 65536, kOneEntries = 65536;

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const int32_t* tables, int64_t row_stride, int entries, int width,
                                                                    int num_pages, int32_t* out, int32_t* page_map, int32_t* source,
                                                                    int32_t* target, int32_t* counts, int32_t* status) {
  __shared__ uint32_t used[kOnePages / 32];
  __shared__ int s_warp[kPlanThreads / 32];
  const int words = (num_pages + 31) / 32;
  for (int i = threadIdx.x; i < words; i += kPlanThreads) used[i] = 0;
  __syncthreads();
  auto entry = [&](int i) { return tables[static_cast<int64_t>(i / width) * row_stride + i % width]; };
  for (int i = threadIdx.x; i < entries; i += kPlanThreads) {
    const int id = entry(i);
    if (in_pool(id, num_pages)) atomicOr(&used[id >> 5], 1u << (id & 31));
    else if (id >= 0) report(status, B200_ERR_BOUNDS);
  }
  __syncthreads();
  // a run of words per thread
  const int per = (words + kPlanThreads - 1) / kPlanThreads, lo = min(static_cast<int>(threadIdx.x) * per, words), hi = min(lo + per, words);
  int mine = 0, live, moves;
  for (int i = lo; i < hi; ++i) mine += __popc(used[i]);
  block_sum_upto(mine, s_warp, &live);
  auto front = [&](int i) -> uint32_t {                  // the pages of word i below `live`
    const int n = live - i * 32;
    return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
  };
  int holes = 0, movers = 0;
  for (int i = lo; i < hi; ++i) holes += __popc(~used[i] & front(i)), movers += __popc(used[i] & ~front(i));
  int hole = block_sum_upto(holes, s_warp, &moves) - holes, mover = block_sum_upto(movers, s_warp, &moves) - movers;
  for (int i = lo; i < hi; ++i) {
    for (uint32_t m = ~used[i] & front(i); m; m &= m - 1) target[hole++] = i * 32 + __ffs(m) - 1;
    for (uint32_t m = used[i] & ~front(i); m; m &= m - 1) source[mover++] = i * 32 + __ffs(m) - 1;
  }
  for (int i = threadIdx.x; i < num_pages; i += kPlanThreads) page_map[i] = i < live && (used[i >> 5] >> (i & 31) & 1) ? i : -1;
  __syncthreads();
  for (int j = threadIdx.x; j < moves; j += kPlanThreads) page_map[source[j]] = target[j];
  if (threadIdx.x == 0) counts[0] = live, counts[1] = moves;
  __syncthreads();
  for (int i = threadIdx.x; i < entries; i += kPlanThreads) {
    const int id = entry(i);
    out[i] = in_pool(id, num_pages) ? page_map[id] : -1;
  }
}

int grid_for(int64_t items) {
  const int64_t ctas = (items + kThreads - 1) / kThreads;
  return static_cast<int>(ctas < 1184 ? ctas : 1184);
}

int copy(const CopyArgs& a, cudaStream_t s) {
  if (a.n == 0 || a.num_pools == 0) return B200_OK;
  if (a.num_pools > 65535) return B200_ERR_TOO_LARGE;
  // a CTA per piece; where the number of pairs is known on the device only, CTAs for one wave of them per pool, which walk
  const int64_t items = static_cast<int64_t>(a.n) * a.pieces, most = a.count ? 1184 : 2147483647;
  copy_pages_kernel<<<dim3(static_cast<unsigned>(items < most ? items : most), a.num_pools), kThreads, 0, s>>>(a);
  return launch_result();
}

int pieces_of(int64_t largest_page) { return static_cast<int>(largest_page > 0 ? (largest_page + kPiece - 1) / kPiece : 1); }

}  // namespace
}  // namespace b200

extern "C" size_t b200_copy_pages_workspace_bytes(int32_t num_pairs, int64_t num_pages) {
  return num_pairs > b200::kLookedThrough && num_pages > 0 ? static_cast<size_t>(num_pages) * sizeof(int32_t) : 0;
}

extern "C" int b200_copy_pages(const int64_t* pools, const int64_t* page_bytes, int64_t largest_page, int32_t num_pools, int64_t num_pages,
                               const int32_t* source, const int32_t* target, int32_t num_pairs, void* workspace,
                               size_t workspace_bytes, int32_t* status, void* stream) {
  using namespace b200;
  if (num_pools < 0 || num_pages < 0 || num_pairs < 0 || largest_page < 0) return B200_ERR_ARG;
  if (num_pairs == 0 || num_pools == 0) return B200_OK;
  if (!pools || !page_bytes || !source || !target) return B200_ERR_ARG;
  if (num_pages > 2147483647 || num_pairs >= kNoPair) return B200_ERR_TOO_LARGE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CopyArgs a{pools, page_bytes, source, target, nullptr, num_pairs, num_pools, pieces_of(largest_page),
             num_pairs <= kLookedThrough, nullptr, num_pages, status};
  const size_t need = b200_copy_pages_workspace_bytes(num_pairs, num_pages);
  if (need > 0) {
    if (!workspace || workspace_bytes < need) return B200_ERR_WORKSPACE;
    int32_t* first = static_cast<int32_t*>(workspace);
    if (cudaMemsetAsync(first, 0x7f, need, s) != cudaSuccess) return launch_result(cudaErrorUnknown);
    mark_pairs_kernel<<<(num_pairs - 1) / kThreads + 1, kThreads, 0, s>>>(source, target, num_pairs, num_pages, first);
    a.first = first;
  }
  return copy(a, s);
}

extern "C" int b200_compact_pages(const int64_t* pools, const int64_t* page_bytes, int64_t largest_page, int32_t num_pools, int64_t num_pages,
                                  const int32_t* block_tables, int64_t bt_stride, int64_t rows, int32_t width, int32_t* out_tables,
                                  int32_t* page_map, int32_t* source, int32_t* target, int32_t* counts, int32_t* status, void* stream) {
  using namespace b200;
  if (num_pools < 0 || num_pages < 0 || rows < 0 || width < 0 || bt_stride < width || largest_page < 0) return B200_ERR_ARG;
  if (num_pages > 2147483647) return B200_ERR_TOO_LARGE;
  if (!counts || (num_pages > 0 && (!page_map || !source || !target)) || (rows * width > 0 && (!block_tables || !out_tables)) ||
      (num_pools > 0 && (!pools || !page_bytes)))
    return B200_ERR_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t entries = rows * width;
  // One launch where its CTA can hold the pages as bits (us, one CTA / the four launches, copies without moves included): 500 pages with 208
  // entries 6.5 / 12.6, 8,192 with as many 12 / 17, 65,536 with 8,192 17 / 159, with 65,536 60 / 160.
  if (num_pages <= kOnePages && entries <= kOneEntries) {
    compact_plan_kernel<<<1, kPlanThreads, 0, s>>>(block_tables, bt_stride, static_cast<int>(entries), width > 0 ? width : 1,
                                                   static_cast<int>(num_pages), out_tables, page_map, source, target, counts, status);
  } else {
    if (cudaMemsetAsync(page_map, 0, num_pages * sizeof(int32_t), s) != cudaSuccess) return launch_result(cudaErrorUnknown);
    if (entries > 0)
      mark_pages_kernel<<<grid_for(entries), kThreads, 0, s>>>(block_tables, bt_stride, rows, width, num_pages, page_map, status);
    plan_pages_kernel<<<1, kPlanThreads, 0, s>>>(page_map, static_cast<int>(num_pages), source, target, counts);
    if (entries > 0)
      rename_pages_kernel<<<grid_for(entries), kThreads, 0, s>>>(block_tables, bt_stride, rows, width, num_pages, page_map, out_tables);
  }
  const int rc = launch_result();
  if (rc != B200_OK || num_pages == 0) return rc;
  return copy({pools, page_bytes, source, target, counts + 1, static_cast<int>(num_pages), num_pools, pieces_of(largest_page), false, nullptr, num_pages,
               status}, s);
}
