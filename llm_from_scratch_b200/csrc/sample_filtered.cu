// The next token under temperature, top-k, top-p and min-p, drawn with a given random number per row.
//
// The tokens of a row are ordered by logit, highest first, and by number among equal logits.  With w_i = exp((x_i - max x) / T):
//   top-k   keeps the first k of the order;
//   top-p   of those the shortest run from the front whose weights reach p of their sum (at least one token);
//   min-p   of those the tokens with w_i >= min_p;
//   draw    the first token, by number, at which the running sum of the kept weights exceeds u times their sum.
// Rows with T <= 0 and rows without any weight (no logit above -inf) take the first of the highest logits.  NaN counts as -inf.
//
// Weights are computed in 64 bits and held as whole numbers of 2^-S, S as large as their sum allows (45 bits at 131,072
// tokens): sums of whole numbers do not depend on their order, so the borders fall at the same token whatever the launch looks like.
//
// A cluster of CTAs shares a row, whose logits stay in shared memory: a thread owns a run of neighbouring tokens.  Borders by value (top-k with
// ones as masses, top-p with the weights) are found with a histogram over the distance from the maximum, in steps of T / 64, and, if the
// border's bin holds more than a few tokens, over ever finer ranges of the logits' bits; what is left is sorted.  The border of the draw is
// found by sums over the threads' runs.  Histograms hold a weight in three parts of 16 bits or more, each a 32-bit counter: shared memory adds
// 32 bits at a time.
//
// Bound by the reads for large rows in principle; in fact by the weights (ten 64-bit operations each) and the histogram's additions.
#include <cooperative_groups.h>

#include "common.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 512;

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int vocab;
  const float* uniforms;
  const float* temperatures;
  const int32_t* top_k;      // or null
  const float* top_p;        // or null
  const float* min_p;        // or null
  int64_t* out;
  int bits;                  // S
};

// Unsigned number with the order of the floats; NaN as -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) x = -INFINITY;
  if (x == 0.f) x = 0.f;     // -0 and 0 are equal
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// ---------------------------------------------------------------------------------------------
// rows that fit the shared memory of a cluster
// ---------------------------------------------------------------------------------------------
constexpr int kRowThreads = 512, kRowWarps = kRowThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 512;           // tokens that are sorted at most
constexpr double kMagic = 6755399441055744.0;      // 1.5 * 2^52: added, it leaves the nearest whole number in the low bits

struct RowShared {
  double table[64];                  // 2^(i / 64)
  uint32_t hist[3][kBins];
  unsigned long long list_key[kList], list_mass[kList];
  unsigned long long parts[8];       // of the CTAs of the cluster
  unsigned long long scan[kRowWarps];
  unsigned long long found_key, found_left;
  uint32_t list_size, lo_key, hi_key;
};

// Shape of a row in the cluster: tokens of a CTA, of a thread, and the stride of the threads' runs (an odd number of 16-byte pieces, so that
// the lanes of a warp read different banks).
struct RowShape {
  int slice, run, stride;
};
__host__ __device__ inline RowShape row_shape(int vocab, int ranks) {
  RowShape r;
  r.slice = ((vocab + ranks - 1) / ranks + 7) / 8 * 8;
  r.run = ((r.slice + kRowThreads - 1) / kRowThreads + 3) / 4 * 4;
  r.stride = 4 * (r.run / 4 | 1);
  return r;
}
inline size_t row_smem(int vocab, int ranks) { return sizeof(RowShared) + static_cast<size_t>(kRowThreads) * row_shape(vocab, ranks).stride * 4; }

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2) sample_row_kernel(const SampleArgs a) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t smem[];
  RowShared& sh = *reinterpret_cast<RowShared*>(smem);
  float* data = reinterpret_cast<float*>(smem + sizeof(RowShared));
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int row = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.vocab;
  const RowShape shape = row_shape(V, ranks);
  const int begin = rank * shape.slice;                  // first token of the CTA
  const int mine = begin + tid * shape.run;              // of the thread
  float* own = data + tid * shape.stride;
  auto sync = [&]() {
    if (ranks > 1) cluster.sync();
    else __syncthreads();
  };

  // ---- the CTA's logits; NaN and what lies behind the row as -inf
  {
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride + begin;
    const int n = min(shape.slice, V - begin);           // may be negative
    auto clean = [](float v) { return v != v ? -INFINITY : v; };
    const int all = kRowThreads * shape.run;
    constexpr int W = 16 / sizeof(T);
    const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0;
    for (int i = tid * W; i < all; i += kRowThreads * W) {
      float v[W];
      if (wide && i + W <= n) {
        const uint4 raw = __ldg(reinterpret_cast<const uint4*>(x + i));
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = clean(to_float<T>(e[j]));
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = i + j < n ? clean(to_float<T>(x[i + j])) : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < W; j += 4) {
        const int owner = (i + j) / shape.run, at = (i + j) % shape.run;
        if (owner < kRowThreads) *reinterpret_cast<float4*>(data + owner * shape.stride + at) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      }
    }
    if (tid < 64) sh.table[tid] = exp2(tid / 64.0);
    if (tid == 0) sh.list_size = 0;
  }
  __syncthreads();
  auto each = [&](auto f) {                              // f(logit, token) over the thread's run
    for (int i = 0; i < shape.run; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(own + i);
      f(v.x, mine + i), f(v.y, mine + i + 1), f(v.z, mine + i + 2), f(v.w, mine + i + 3);
    }
  };
  auto composite = [](float x, int i) -> unsigned long long {
    return static_cast<unsigned long long>(order_key(x)) << 32 | static_cast<uint32_t>(~i);
  };
  // over the cluster, the same in all threads; what parts held is lost
  auto combine = [&](unsigned long long v, bool max) -> unsigned long long {
    auto join = [&](unsigned long long x, unsigned long long y) { return max ? (x > y ? x : y) : x + y; };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0) sh.scan[warp] = v;
    __syncthreads();
    v = sh.scan[0];
    for (int w = 1; w < kRowWarps; ++w) v = join(v, sh.scan[w]);
    if (ranks > 1) {
      if (tid < ranks) *cluster.map_shared_rank(&sh.parts[rank], tid) = v;
      cluster.sync();
      v = sh.parts[0];
      for (int r = 1; r < ranks; ++r) v = join(v, sh.parts[r]);
    }
    sync();                                              // scan and parts may be written again
    return v;
  };

  unsigned long long best = 0;
  each([&](float x, int i) {
    const unsigned long long c = composite(x, i);
    best = c > best ? c : best;
  });
  best = combine(best, true);
  const float temperature = a.temperatures[row], top = key_value(static_cast<uint32_t>(best >> 32));
  if (!(temperature > 0.f) || top == -INFINITY) {
    if (rank == 0 && tid == 0) a.out[row] = static_cast<int>(~static_cast<uint32_t>(best));
    return;
  }
  const double max = top, factor = 64.0 * 1.4426950408889634 / temperature;
  const int S = a.bits;
  double floor_w = a.min_p ? static_cast<double>(a.min_p[row]) : 0.0;
  floor_w = (floor_w > 1.0 ? 1.0 : floor_w) * static_cast<double>(1ull << S);
  // the weight in units of 2^-S: 2^(k / 64) 2^(r / 64) with |r| <= 1/2, the second factor by its series up to r^4 (error 4e-14)
  auto weight = [&](float x) -> double {
    if (x == top) return static_cast<double>(1ull << S);
    const double y = (static_cast<double>(x) - max) * factor;
    if (!(y > -64.0 * 55)) return 0.0;                   // below 2^-55, or the NaN of infinities
    const double t = y + kMagic, r = y - (t - kMagic);
    const int k = __double2loint(t);
    constexpr double b = 0.010830424696249145;           // ln 2 / 64
    const double p = fma(r, fma(r, fma(r, fma(r, b * b * b * b / 24, b * b * b / 6), b * b / 2), b), 1.0);
    const double v = sh.table[k & 63] * p;
    return __hiloint2double(__double2hiint(v) + (((k >> 6) + S) << 20), __double2loint(v));
  };
  auto whole = [&](float x) -> unsigned long long {      // rounded: below 2^51
    return static_cast<unsigned long long>(__double_as_longlong(weight(x) + 4503599627370496.0)) & 0xfffffffffffffull;
  };
  unsigned long long bound = 0;                          // tokens at or above it are kept

  // ---- border by value: the first kept token, from the front of the order, at which the running mass reaches `target`
  const float step = 64.f / temperature;
  auto select = [&](auto mass_of, const bool weighted, unsigned long long target) -> unsigned long long {
    // candidates: tokens of bin `bin` of the last division; of keys lo .. hi from the second one on
    int level = 0, bin = 0, shift = 0;
    uint32_t lo_key = 0, hi_key = 0xffffffffu;
    auto first_bin = [&](float x) -> int {
      const int b = static_cast<int>((top - x) * step);  // saturates; the NaN of infinities gives 0
      return b < kBins - 1 ? b : kBins - 1;
    };
    auto candidate = [&](float x, uint32_t key) -> bool {        // before the division of this level
      return level == 0 || (key >= lo_key && key <= hi_key && (level > 1 || first_bin(x) == bin));
    };
    for (;;) {
      // divide
      for (int i = tid; i < 3 * kBins; i += kRowThreads) (&sh.hist[0][0])[i] = 0;
      __syncthreads();
      each([&](float x, int i) {
        const unsigned long long c = composite(x, i);
        const uint32_t key = static_cast<uint32_t>(c >> 32);
        if (c < bound || !candidate(x, key)) return;
        const int b = level == 0 ? first_bin(x) : static_cast<int>((hi_key - key) >> shift);
        if (!weighted) {
          atomicAdd(&sh.hist[0][b], 1u);
          return;
        }
        const unsigned long long m = mass_of(x);
        const uint32_t m0 = m & 0xffff, m1 = (m >> 16) & 0xffff, m2 = static_cast<uint32_t>(m >> 32);
        if (m0) atomicAdd(&sh.hist[0][b], m0);
        if (m1) atomicAdd(&sh.hist[1][b], m1);
        if (m2) atomicAdd(&sh.hist[2][b], m2);
      });
      sync();
      // a CTA sums its share of the bins over the cluster, a thread a run of them
      const int share = kBins / ranks, each_thread = (share + kRowThreads - 1) / kRowThreads;
      unsigned long long h[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[j] = 0;
        const int b = tid * each_thread + j;
        if (j < each_thread && b < share)
          for (int r = 0; r < ranks; ++r) {
            const uint32_t* from = ranks > 1 ? cluster.map_shared_rank(&sh.hist[0][0], r) : &sh.hist[0][0];
            const int at = rank * share + b;
            h[j] += from[at];
            if (weighted) h[j] += (static_cast<unsigned long long>(from[kBins + at]) << 16) + (static_cast<unsigned long long>(from[2 * kBins + at]) << 32);
          }
        sum += h[j];
      }
      unsigned long long upto = sum;                     // inclusive over the CTA's threads
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (lane == 31) sh.scan[warp] = upto;
      __syncthreads();
      unsigned long long all = 0;
      for (int w = 0; w < kRowWarps; ++w) {
        if (w == warp) upto += all;
        all += sh.scan[w];
      }
      if (tid < ranks) *cluster.map_shared_rank(&sh.parts[rank], tid) = all;
      sync();
      unsigned long long before = 0;
      for (int r = 0; r < rank; ++r) before += sh.parts[r];
      upto += before;
      if (upto >= target && upto - sum < target) {       // one thread of the cluster
        unsigned long long left = target - (upto - sum);
        int b = rank * share + tid * each_thread;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j + 1 < each_thread && left > h[j]) {
            left -= h[j];
            ++b;
          } else {
            break;
          }
        }
        for (int r = 0; r < ranks; ++r) {
          RowShared* to = cluster.map_shared_rank(&sh, r);
          to->found_key = b;
          to->found_left = left;
          to->list_size = 0;
          to->lo_key = 0xffffffffu;
          to->hi_key = 0;
        }
      }
      sync();
      const int next_bin = static_cast<int>(sh.found_key);
      target = sh.found_left;
      // gather the bin
      RowShared* lead = ranks > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
      uint32_t least = 0xffffffffu, most = 0;
      each([&](float x, int i) {
        const unsigned long long c = composite(x, i);
        const uint32_t key = static_cast<uint32_t>(c >> 32);
        if (c < bound || !candidate(x, key) || (level == 0 ? first_bin(x) : static_cast<int>((hi_key - key) >> shift)) != next_bin) return;
        const unsigned long long m = mass_of(x);
        if (m == 0) return;
        least = min(least, key);
        most = key > most ? key : most;
        const uint32_t at = atomicAdd(&lead->list_size, 1u);
        if (at < kList) lead->list_key[at] = c, lead->list_mass[at] = m;
      });
      least = __reduce_min_sync(0xffffffffu, least);
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0 && most != 0) atomicMin(&lead->lo_key, least), atomicMax(&lead->hi_key, most);
      sync();
      const uint32_t size = lead->list_size;
      if (size <= kList) {
        if (rank == 0) {
          // sort, then the first place at which the running mass reaches the target
          int n = 32;
          while (n < static_cast<int>(size)) n *= 2;
          for (int i = size + tid; i < n; i += kRowThreads) sh.list_key[i] = 0, sh.list_mass[i] = 0;
          __syncthreads();
          for (int k = 2; k <= n; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
              const int other = tid ^ j;
              if (tid < n && other > tid) {
                const unsigned long long x = sh.list_key[tid], y = sh.list_key[other];
                if ((tid & k) == 0 ? x < y : x > y) {
                  const unsigned long long mx = sh.list_mass[tid], my = sh.list_mass[other];
                  sh.list_key[tid] = y, sh.list_key[other] = x;
                  sh.list_mass[tid] = my, sh.list_mass[other] = mx;
                }
              }
              __syncthreads();
            }
          unsigned long long m = tid < n ? sh.list_mass[tid] : 0, up = m;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long y = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += y;
          }
          if (lane == 31) sh.scan[warp] = up;
          __syncthreads();
          for (int w = 0; w < warp; ++w) up += sh.scan[w];
          if (up >= target && up - m < target)
            for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(&sh, r)->found_key = sh.list_key[tid];
        }
        sync();
        return sh.found_key;
      }
      const uint32_t least_all = lead->lo_key, most_all = lead->hi_key;
      if (least_all == most_all) {                       // equal logits: so many of them, by token
        const unsigned long long one = mass_of(key_value(least_all));
        sh.found_left = (target + one - 1) / one;        // the same in all threads
        lo_key = hi_key = least_all;
        sync();                                          // nobody reads the list's words any more
        return static_cast<unsigned long long>(least_all) << 32;
      }
      sync();
      bin = next_bin;
      lo_key = least_all, hi_key = most_all;
      const int width = 32 - __clz(hi_key - lo_key);     // bits of the range
      shift = width > 11 ? width - 11 : 0;
      ++level;
    }
  };
  // ---- border by token: the first token at which the running mass reaches `target`; -1 in all threads but the one that owns it
  auto locate = [&](auto mass_at, auto target_of) -> int {
    unsigned long long sum = 0;
    each([&](float x, int i) { sum += mass_at(x, i); });
    unsigned long long upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) sh.scan[warp] = upto;
    __syncthreads();
    unsigned long long all = 0;
    for (int w = 0; w < kRowWarps; ++w) {
      if (w == warp) upto += all;
      all += sh.scan[w];
    }
    if (tid < ranks) *cluster.map_shared_rank(&sh.parts[rank], tid) = all;
    sync();
    unsigned long long before = 0, total = 0;
    for (int r = 0; r < ranks; ++r) {
      if (r < rank) before += sh.parts[r];
      total += sh.parts[r];
    }
    const unsigned long long target = target_of(total);
    upto += before;
    if (!(upto >= target && upto - sum < target)) return -1;
    unsigned long long left = target - (upto - sum);
    for (int i = 0; i < shape.run; ++i) {
      const unsigned long long m = mass_at(own[i], mine + i);
      if (m >= left) return mine + i;
      left -= m;
    }
    return -1;
  };
  // a border by value with its place among equal logits
  auto cut = [&](auto mass_of, const bool weighted, unsigned long long target) {
    const unsigned long long at = select(mass_of, weighted, target);
    if (static_cast<uint32_t>(at) != 0) {                // a token's number is never 2^32 - 1
      bound = at;
      return;
    }
    const unsigned long long ties = sh.found_left;
    __syncthreads();
    const int token = locate(
        [&](float x, int i) -> unsigned long long {
          const unsigned long long c = composite(x, i);
          return c >= bound && (c >> 32) == (at >> 32) ? 1ull : 0ull;
        },
        [&](unsigned long long total) { return ties < total ? ties : total; });
    if (token >= 0)
      for (int r = 0; r < ranks; ++r) cluster.map_shared_rank(&sh, r)->found_key = at | static_cast<uint32_t>(~token);
    sync();
    bound = sh.found_key;
    sync();
  };
  const int k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && k < V) cut([](float) -> unsigned long long { return 1; }, false, static_cast<unsigned long long>(k));
  const float p = a.top_p ? a.top_p[row] : 1.f;
  if (p < 1.f) {
    unsigned long long sum = 0;
    each([&](float x, int i) {
      if (composite(x, i) >= bound) sum += whole(x);
    });
    const double want = ceil(static_cast<double>(p) * static_cast<double>(combine(sum, false)));
    cut(whole, true, want > 1.0 ? static_cast<unsigned long long>(want) : 1ull);
  }
  const float u = a.uniforms[row];
  const bool any = !(u > 0.f);                           // the first kept token of any weight, however small
  const int token = locate(
      [&](float x, int i) -> unsigned long long {
        if (composite(x, i) < bound) return 0;
        if (any && floor_w <= 0.0) return x == top || (static_cast<double>(x) - max) / temperature > -745.13 ? 1 : 0;
        const double w = weight(x);
        if (!(w >= floor_w)) return 0;
        return any ? 1 : static_cast<unsigned long long>(__double_as_longlong(w + 4503599627370496.0)) & 0xfffffffffffffull;
      },
      [&](unsigned long long total) -> unsigned long long {
        const unsigned long long t = any ? 1ull : static_cast<unsigned long long>(static_cast<double>(u) * static_cast<double>(total)) + 1;
        return t < total ? t : total;
      });
  if (token >= 0) a.out[row] = token;
}

template <typename T>
int launch_rows(const SampleArgs& a, int64_t rows, int ranks, cudaStream_t s) {
  static bool configured[64] = {};                       // racing threads set the same attribute
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return B200_ERR_UNSUPPORTED;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(sample_row_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess) {
      cudaGetLastError();
      return B200_ERR_LAUNCH;
    }
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * ranks));
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = row_smem(a.vocab, ranks);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launch_result(cudaLaunchKernelEx(&cfg, sample_row_kernel<T>, a));
}

// ---------------------------------------------------------------------------------------------
// rows beyond that: a CTA per row that reads the logits for every step of a radix selection over the bytes of the order
// ---------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_filtered_kernel(const SampleArgs a) {
  __shared__ uint32_t h_lo[256], h_hi[256];
  __shared__ unsigned long long s_key, s_left;
  __shared__ unsigned long long s_red[kThreads / 32];
  const int row = blockIdx.x, tid = threadIdx.x, V = a.vocab;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  auto reduce = [&](unsigned long long v, bool max) {
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long w = __shfl_xor_sync(0xffffffffu, v, o);
      v = max ? (w > v ? w : v) : v + w;
    }
    __syncthreads();
    if ((tid & 31) == 0) s_red[tid >> 5] = v;
    __syncthreads();
    v = s_red[0];
    for (int w = 1; w < kThreads / 32; ++w) v = max ? (s_red[w] > v ? s_red[w] : v) : v + s_red[w];
    return v;
  };
  // order of the tokens: larger is earlier
  auto composite = [&](int i) {
    return static_cast<unsigned long long>(order_key(to_float<T>(x[i]))) << 32 | static_cast<uint32_t>(~i);
  };
  unsigned long long best = 0;
  for (int i = tid; i < V; i += kThreads) {
    const unsigned long long c = composite(i);
    best = c > best ? c : best;
  }
  best = reduce(best, true);
  const uint32_t top = static_cast<uint32_t>(best >> 32);
  const float temperature = a.temperatures[row];
  if (!(temperature > 0.f) || top == order_key(-INFINITY)) {
    if (tid == 0) a.out[row] = static_cast<int>(~static_cast<uint32_t>(best));
    return;
  }
  const double max = key_value(top), t = temperature, unit = static_cast<double>(1ull << a.bits);
  double floor_w = a.min_p ? static_cast<double>(a.min_p[row]) : 0.0;
  if (floor_w > 1.0) floor_w = 1.0;
  auto weight = [&](uint32_t key) -> double {
    if (key == top) return 1.0;
    const double e = (static_cast<double>(key_value(key)) - max) / t;
    return e > -746.0 ? exp(e) : 0.0;                // also 0 for the NaN of infinities
  };
  unsigned long long bound = 0;                      // tokens at or above it are kept
  // the first element, by descending `key`, at which the running mass of the kept elements reaches `target`; bytes from `top_byte` down
  auto select = [&](auto key_of, auto mass_of, unsigned long long target, int top_byte) {
    unsigned long long prefix = 0;
    for (int shift = top_byte * 8; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = tid; i < 256; i += kThreads) h_lo[i] = h_hi[i] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const unsigned long long c = composite(i);
        if (c < bound) continue;
        const unsigned long long k = key_of(c);
        if (shift + 8 < 64 && (k >> (shift + 8)) != prefix) continue;
        const unsigned long long m = mass_of(c);
        if (m == 0) continue;
        const int bin = static_cast<int>(k >> shift) & 255;
        const uint32_t lo = static_cast<uint32_t>(m), old = atomicAdd(&h_lo[bin], lo);
        const uint32_t hi = static_cast<uint32_t>(m >> 32) + (old + lo < old ? 1u : 0u);
        if (hi) atomicAdd(&h_hi[bin], hi);
      }
      __syncthreads();
      if (tid == 0) {
        unsigned long long left = target;
        int bin = 255;
        for (; bin > 0; --bin) {
          const unsigned long long h = static_cast<unsigned long long>(h_hi[bin]) << 32 | h_lo[bin];
          if (h >= left) break;
          left -= h;
        }
        s_key = prefix << 8 | static_cast<unsigned>(bin);
        s_left = left;
      }
      __syncthreads();
      prefix = s_key;
      target = s_left;
    }
    return prefix;
  };
  auto whole = [&](unsigned long long c) { return static_cast<unsigned long long>(__double2ull_rn(weight(static_cast<uint32_t>(c >> 32)) * unit)); };
  auto itself = [](unsigned long long c) { return c; };
  auto total = [&](auto mass_of) {
    unsigned long long sum = 0;
    for (int i = tid; i < V; i += kThreads) {
      const unsigned long long c = composite(i);
      if (c >= bound) sum += mass_of(c);
    }
    return reduce(sum, false);
  };
  const int k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && k < V) bound = select(itself, [](unsigned long long) { return 1ull; }, static_cast<unsigned long long>(k), 7);
  const float p = a.top_p ? a.top_p[row] : 1.f;
  if (p < 1.f) {
    const double want = ceil(static_cast<double>(p) * static_cast<double>(total(whole)));
    bound = select(itself, whole, want > 1.0 ? static_cast<unsigned long long>(want) : 1ull, 7);
  }
  auto kept = [&](unsigned long long c) {
    const double w = weight(static_cast<uint32_t>(c >> 32));
    return w >= floor_w ? static_cast<unsigned long long>(__double2ull_rn(w * unit)) : 0ull;
  };
  const unsigned long long sum = total(kept);
  const float u = a.uniforms[row];
  if (!(u > 0.f)) {                                  // the first kept token of any weight, however small
    unsigned long long first = 0;
    for (int i = tid; i < V; i += kThreads) {
      const unsigned long long c = composite(i);
      const double w = weight(static_cast<uint32_t>(c >> 32));
      if (c >= bound && w >= floor_w && w > 0.0) first = (c & 0xffffffffull) > first ? c & 0xffffffffull : first;
    }
    first = reduce(first, true);
    if (tid == 0) a.out[row] = static_cast<int>(~static_cast<uint32_t>(first));
    return;
  }
  unsigned long long target = static_cast<unsigned long long>(static_cast<double>(u) * static_cast<double>(sum)) + 1;
  if (target > sum) target = sum;
  const unsigned long long at = select([](unsigned long long c) { return c & 0xffffffffull; }, kept, target, 3);
  if (tid == 0) a.out[row] = static_cast<int>(~static_cast<uint32_t>(at));
}

}  // namespace
}  // namespace b200

extern "C" int b200_sample_filtered(const void* logits, int64_t row_stride, int64_t num_rows, int32_t vocab_size,
                                    const float* uniforms, const float* temperatures, const int32_t* top_k, const float* top_p,
                                    const float* min_p, int64_t* out_tokens, int32_t dtype, void* stream) {
  using namespace b200;
  if (num_rows < 0 || vocab_size <= 0 || row_stride < vocab_size) return B200_ERR_ARG;
  if (dtype != B200_DTYPE_F32 && dtype != B200_DTYPE_BF16) return B200_ERR_UNSUPPORTED;
  if (num_rows == 0) return B200_OK;
  if (!logits || !uniforms || !temperatures || !out_tokens) return B200_ERR_ARG;
  if (num_rows > 2147483647 || vocab_size > (1 << 24)) return B200_ERR_TOO_LARGE;
  SampleArgs a{logits, row_stride, vocab_size, uniforms, temperatures, top_k, top_p, min_p, out_tokens, 62};
  while ((1ll << (62 - a.bits)) < vocab_size) --a.bits;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int ranks = 1;
  while (ranks < 8 && row_smem(vocab_size, ranks) > 110 * 1024) ranks *= 2;
  while (ranks < 8 && num_rows * ranks * 2 <= 296 && vocab_size / ranks > 4096) ranks *= 2;
  if (row_smem(vocab_size, ranks) <= 226 * 1024 && row_shape(vocab_size, ranks).slice < 65536 && num_rows * ranks <= 2147483647) {
    if (a.bits > 50) a.bits = 50;
    return dtype == B200_DTYPE_F32 ? launch_rows<float>(a, num_rows, ranks, s) : launch_rows<__nv_bfloat16>(a, num_rows, ranks, s);
  }
  const int grid = static_cast<int>(num_rows);
  if (dtype == B200_DTYPE_F32) sample_filtered_kernel<float><<<grid, kThreads, 0, s>>>(a);
  else sample_filtered_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
  return launch_result();
}
