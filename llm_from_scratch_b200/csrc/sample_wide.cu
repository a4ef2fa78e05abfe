// Filtered sampling of many long rows (sample_filtered.cu has the definition and the form for few or short ones): passes over the logits by CTAs
// that share nothing but small sums, one launch each.
//
//   top      highest logit of every slice of 8,192
//   count    histogram of the distances from the row's maximum, in steps of T / 256
//   bracket  a CTA per row: the bin of the k-th token, and the bins among which the nucleus ends (as there, at twice the resolution)
//   sum      weights in front of those bins and of all, per 1,024 tokens; the tokens in the bins go to the row's list
//   draw     a CTA per row: the list in order, the borders, the 1,024 tokens in which the draw falls, the token
//
// The form in shared memory reads the logits once but passes six barriers of a cluster, with two CTAs on an SM to fill the waits: 256 rows of
// 131,072 take it 251 us.  Here they are read three times and nothing waits inside a pass: 141 us, mean of 20 (a read alone takes 21).  Launched
// one by one with cold caches, which takes 152 in all: top 27, count 34, bracket 9, sum 69, draw 13.  Bound by the weights of the sum: ten 64-bit operations for a token that has one, of which an SM
// does few at a time.  In bf16 140 .. 150 us (with the bins' middles for where their tokens lie the lists overflow and rows go to the other form: 280).
// Rows that this form does not take (greedy ones, infinite logits, u <= 0, lists that overflow, a bracket that does not hold the border) are
// named in a list, and the other form's kernel runs over that list at the end.
#include "sampling.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kChunk = 1024, kSlice = kWarps * kChunk;    // tokens of a warp and of a CTA
constexpr int kBins = 8192;
constexpr float kPerUnit = 256.f;                         // bins per distance T: 32 T and the last bin
constexpr int kList = 2048;
constexpr int kRowThreads = 512, kOwnBins = kBins / kRowThreads, kOwnList = kList / kRowThreads;
constexpr int kMaxChunks = 1024;                          // vocabularies up to 1,048,576

struct alignas(16) RowState {
  int bin_k, left_k, bin_hi;
  int list_size, skip;                                    // skip: the row is in the list of the others
  // what the pass over the weights needs.  With y the distance from the maximum in bins: the bracket holds y_lo < y <= y_hi, the k-th token's bin
  // y_k < y <= y_k1, and up to y_near a token may lie in front of the bracket or in a bin of the list.
  float top, step, deep, y_lo, y_hi, y_k, y_k1, y_near;   // deep: logits below it weigh e^-64, which rounds to 0
  int nucleus, at_k;
  double factor, floor_w;
};

struct Wide {
  SampleArgs a;
  int rows, slices, chunks;
  int count_tokens, sum_slices;                           // of a CTA of the two long passes
  uint32_t* slice_top;                                    // [rows, slices] order keys
  uint32_t* hist;                                         // [rows, kBins]
  RowState* state;                                        // [rows]
  unsigned long long* list_key;                           // [rows, kList]
  unsigned long long* list_mass;
  unsigned long long* sums;                               // [rows, chunks, 3]: weights in front of the bracket, all, kept in front
  int32_t* others;                                        // [1 + rows]: number of them, rows
};

template <typename T>
__device__ __forceinline__ void load4_raw(const T* x, int i, int n, bool wide, float (&v)[4]) {
  if (wide && i + 4 <= n) {
    if constexpr (sizeof(T) == 4) {
      const float4 t = *reinterpret_cast<const float4*>(x + i);
      v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    } else {
      const uint2 t = *reinterpret_cast<const uint2*>(x + i);
      v[0] = __uint_as_float(t.x << 16), v[1] = __uint_as_float(t.x & 0xffff0000u);
      v[2] = __uint_as_float(t.y << 16), v[3] = __uint_as_float(t.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < n ? to_float<T>(x[i + j]) : -INFINITY;
  }
}
template <typename T>
__device__ __forceinline__ void load4(const T* x, int i, int n, bool wide, float (&v)[4]) {       // NaN as -inf
  load4_raw(x, i, n, wide, v);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = v[j] != v[j] ? -INFINITY : v[j];
}
template <typename T>
__device__ __forceinline__ bool wide_loads(const T* x) { return reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0; }

template <typename T>
__global__ void __launch_bounds__(kThreads) wide_top_kernel(const Wide w) {
  __shared__ uint32_t s_top[kWarps];
  const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, V = w.a.vocab;
  const T* x = static_cast<const T*>(w.a.logits) + row * w.a.row_stride;
  const bool wide = wide_loads(x);
  float top = -INFINITY;
#pragma unroll 8
  for (int c = 0; c < kSlice / (kThreads * 4); ++c) {
    float v[4];
    load4(x, slice * kSlice + (c * kThreads + tid) * 4, V, wide, v);
    top = fmaxf(fmaxf(top, fmaxf(v[0], v[1])), fmaxf(v[2], v[3]));
  }
  const uint32_t key = __reduce_max_sync(0xffffffffu, order_key(top));
  if ((tid & 31) == 0) s_top[tid >> 5] = key;
  __syncthreads();
  if (tid < 32) {
    const uint32_t all = __reduce_max_sync(0xffffffffu, tid < kWarps ? s_top[tid] : 0u);
    if (tid == 0) w.slice_top[row * w.slices + slice] = all;
  }
  // what the next passes add to
  for (int i = slice * kThreads + tid; i < kBins / 4; i += w.slices * kThreads)
    reinterpret_cast<uint4*>(w.hist + static_cast<int64_t>(row) * kBins)[i] = make_uint4(0, 0, 0, 0);
  if (slice == 0 && tid == 0) {
    w.state[row].list_size = w.state[row].skip = 0;
    if (row == 0) w.others[0] = 0;
  }
}

// The row's parameters, the same in all threads; false: a row for the other form, or without filters where these are asked for.  Every thread
// of the CTA calls it.
struct RowParams {
  float top, temperature, p, u, step, reach;
  int k;
  double factor, floor_w;
  bool taken, filtered;
};
__device__ __forceinline__ RowParams row_params(const Wide& w, int row) {
  __shared__ uint32_t s_row_top;
  const SampleArgs& a = w.a;
  if (threadIdx.x < 32) {
    uint32_t key = 0;
    for (int i = threadIdx.x; i < w.slices; i += 32) key = max_key(key, w.slice_top[row * w.slices + i]);
    key = __reduce_max_sync(0xffffffffu, key);
    if (threadIdx.x == 0) s_row_top = key;
  }
  __syncthreads();
  RowParams r;
  r.top = key_value(s_row_top);
  r.temperature = fminf(a.temperatures[row], 1e30f);
  r.p = a.top_p ? a.top_p[row] : 1.f;
  r.u = fminf(a.uniforms[row], 1.f);
  r.k = a.top_k ? a.top_k[row] : 0;
  if (r.k >= a.vocab || r.k < 0) r.k = 0;
  const float floor_w = a.min_p ? a.min_p[row] : 0.f;
  r.floor_w = (floor_w > 1.f ? 1.0 : floor_w > 0.f ? static_cast<double>(floor_w) : 0.0) * static_cast<double>(1ull << a.bits);
  // (the pass over the weights cuts distances at 64 T in 32 bits, which needs a T that is not lost beside the maximum)
  r.taken = r.temperature > 0.f && fabsf(r.top) < INFINITY && r.u > 0.f && fabsf(r.top) < 1e6f * r.temperature;
  r.filtered = r.k > 0 || r.p < 1.f;
  r.factor = 64.0 * 1.4426950408889634 / r.temperature;
  r.reach = 660.f * r.temperature;
  r.step = fminf(kPerUnit / r.temperature, 3e38f);
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) wide_count_kernel(const Wide w) {
  __shared__ uint32_t hist[kBins / 2];                    // two counts to a word: a CTA has fewer than 65,536 tokens
  const int row = blockIdx.y, tid = threadIdx.x, V = w.a.vocab;
  const RowParams r = row_params(w, row);
  if (!r.taken || !r.filtered) return;
  const T* x = static_cast<const T*>(w.a.logits) + row * w.a.row_stride;
  const bool wide = wide_loads(x);
  for (int i = tid; i < kBins / 2; i += kThreads) hist[i] = 0;
  __syncthreads();
  const int last = r.k > 0 ? kBins : kBins - 1;           // what is in the last bin has no weight
  const int end = min_of((blockIdx.x + 1) * w.count_tokens, V);
#pragma unroll 4
  for (int i = blockIdx.x * w.count_tokens + tid * 4; i < end; i += kThreads * 4) {
    float v[4];
    load4_raw(x, i, V, wide, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = __float2int_ru(fminf((r.top - v[j]) * r.step, kBins - 1.f));       // NaN goes to the last bin, as do places behind the row
      if (b < last) atomicAdd(&hist[b & (kBins / 2 - 1)], b >= kBins / 2 ? 0x10000u : 1u);
    }
  }
  __syncthreads();
  uint32_t* out = w.hist + static_cast<int64_t>(row) * kBins;
  for (int i = tid; i < kBins / 2; i += kThreads) {
    const uint32_t y = hist[i];
    if (y & 0xffff) atomicAdd(out + i, y & 0xffff);
    if (y >> 16) atomicAdd(out + kBins / 2 + i, y >> 16);
  }
}

__device__ __forceinline__ void leave_to_others(const Wide& w, int row) {
  w.state[row].skip = 1;
  w.others[1 + atomicAdd(&w.others[0], 1)] = row;
}

// Running sums over the CTA's threads, inclusive, and the whole.
template <typename U>
__device__ __forceinline__ U block_upto(U v, U* s_warp, U& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_upto(v);
  __syncthreads();
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  const U upto = warp_upto(lane < kRowThreads / 32 ? s_warp[lane] : U(0));
  const U before = __shfl_sync(0xffffffffu, upto, warp > 0 ? warp - 1 : 0);
  all = __shfl_sync(0xffffffffu, upto, kRowThreads / 32 - 1);
  return warp > 0 ? v + before : v;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) wide_bracket_kernel(const Wide w) {
  __shared__ int s_int[kRowThreads / 32];
  __shared__ float s_float[kRowThreads / 32];
  __shared__ int bin_k, left_k, bin_lo, bin_hi;
  __shared__ float mass_k, spread_k;
  const int row = blockIdx.x, tid = threadIdx.x;
  const RowParams r = row_params(w, row);
  if (!r.taken) {
    if (tid == 0) leave_to_others(w, row);
    return;
  }
  if (tid == 0) bin_k = bin_lo = bin_hi = kBins, left_k = 0;
  if (r.filtered) {
    uint32_t count[kOwnBins];
    const uint4* from = reinterpret_cast<const uint4*>(w.hist + static_cast<int64_t>(row) * kBins) + tid * (kOwnBins / 4);
#pragma unroll
    for (int c = 0; c < kOwnBins / 4; ++c) {
      const uint4 y = from[c];
      count[4 * c] = y.x, count[4 * c + 1] = y.y, count[4 * c + 2] = y.z, count[4 * c + 3] = y.w;
    }
    // a bin's weight where its tokens lie on the average, and the variance of that
    const BinPlaces<sizeof(T) == 2> places(r.top, r.step);
    auto weight_of_bin = [&](int b, float& variance) {
      variance = 0.f;                                    // of the last bin, which weighs nothing
      const float g = b < kBins - 1 ? fast_exp2(-1.4426950408889634f / kPerUnit * places.of(b, variance)) : 0.f;
      variance *= g * g * (1.f / (kPerUnit * kPerUnit));
      return g;
    };
    // 1.2 standard deviations (the other form takes one, where a border outside costs less): a border outside costs its row the other form (75 us), as does a bracket of more tokens than the list
    // takes.  Means of 20 calls of 256 rows of 131,072, p up to 0.99: 142 us; with two 147, with 3.5 159
    auto off = [&](float m, float e) {
      float root;
      asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(e));
      return 1.2f * root + 1e-5f * m;
    };
    int counted = 0;
    float mass = 0.f, spread = 0.f;
#pragma unroll
    for (int c = 0; c < kOwnBins; ++c) {
      const int b = tid * kOwnBins + c;
      float variance;
      const float g = weight_of_bin(b, variance);
      counted += count[c], mass += count[c] * g, spread += count[c] * variance;
    }
    int all;
    float mass_all, spread_all;
    const int upto = block_upto(counted, s_int, all);
    const float mass_up = block_upto(mass, s_float, mass_all), spread_up = block_upto(spread, s_float, spread_all);
    if (r.k > 0) {
      if (upto >= r.k && upto - counted < r.k) {
        int n = upto - counted;
        float m = mass_up - mass, e = spread_up - spread;
#pragma unroll
        for (int c = 0; c < kOwnBins; ++c) {
          const int b = tid * kOwnBins + c, here = count[c];
          float variance;
          const float g = weight_of_bin(b, variance);
          if (n < r.k && n + here >= r.k) bin_k = b, left_k = r.k - n, mass_k = m + (r.k - n) * g, spread_k = e + (r.k - n) * variance;
          n += here, m += here * g, e += here * variance;
        }
      }
      __syncthreads();
      mass_all = mass_k, spread_all = spread_k;
    }
    if (r.p < 1.f) {
      const float goal = r.p * mass_all, wide = r.p * off(mass_all, spread_all);
      if (mass_up + off(mass_up, spread_up) + wide >= goal && !(mass_up - mass - off(mass_up - mass, spread_up - spread) - wide >= goal)) {
        float m = mass_up - mass, e = spread_up - spread;
#pragma unroll
        for (int c = 0; c < kOwnBins; ++c) {
          const int b = tid * kOwnBins + c;
          float variance;
          const float g = weight_of_bin(b, variance);
          m += count[c] * g, e += count[c] * variance;
          if (m + off(m, e) + wide >= goal) atomicMin(&bin_lo, b);
          if (m - off(m, e) - wide >= goal) atomicMin(&bin_hi, b);
        }
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    if (r.p < 1.f && bin_lo >= kBins - 1) {
      leave_to_others(w, row);
    } else {
      const bool nucleus = r.p < 1.f, at_k = bin_k < kBins;
      const int hi = min_of(min_of(bin_hi, bin_k), kBins - 2);
      RowState& s = w.state[row];
      s.bin_k = bin_k, s.left_k = left_k, s.bin_hi = hi;
      s.top = r.top, s.step = r.step, s.factor = r.factor, s.floor_w = r.floor_w;
      // a bin's tokens are told by ceil(y) <= b where y <= b
      s.y_k = at_k ? bin_k - 1.f : INFINITY;
      s.y_k1 = !at_k ? -1.f : bin_k < kBins - 1 ? bin_k : INFINITY;
      s.y_lo = nucleus ? bin_lo - 1.f : s.y_k;
      s.y_hi = nucleus ? hi : -1.f;
      s.deep = r.top - 64.f * r.temperature;
      s.y_near = fmaxf(fmaxf(s.y_lo, s.y_hi), s.y_k1);
      s.nucleus = nucleus, s.at_k = at_k;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) wide_sum_kernel(const Wide w) {
  __shared__ double table[64];
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = w.a.vocab;
  RowState& s = w.state[row];
  if (s.skip) return;
  if (tid < 64) table[tid] = kTable[tid];
  __syncthreads();
  const float top = s.top, step = s.step, deep = s.deep, y_lo = s.y_lo, y_hi = s.y_hi, y_k = s.y_k, y_k1 = s.y_k1, y_near = s.y_near;
  const bool nucleus = s.nucleus, at_k = s.at_k;
  const double max = top, factor = s.factor, least = s.floor_w;
  const int S = w.a.bits;
  const T* x = static_cast<const T*>(w.a.logits) + row * w.a.row_stride;
  const bool wide = wide_loads(x);
#pragma unroll 1
  for (int part = 0; part < w.sum_slices; ++part) {
    const int chunk = (blockIdx.x * w.sum_slices + part) * kWarps + warp, base = chunk * kChunk;
    if (chunk >= w.chunks) break;
    unsigned long long front = 0, all = 0, kept = 0;
    uint32_t noted = 0;                                   // four bits a trip
#pragma unroll 2
    for (int c = 0; c < kChunk / 128; ++c) {
      float v[4], y[4];
      load4_raw(x, base + (c * 32 + lane) * 4, V, wide, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = (top - v[j]) * step;                       // NaN stays: no comparison holds for it
        v[j] = fmaxf(v[j], deep);
      }
      const bool near = fminf(fminf(y[0], y[1]), fminf(y[2], y[3])) <= y_near;
      if (!near && !nucleus) continue;
      double g[4];
      unsigned long long m[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = weight_within(v[j], max, factor, S, table), m[j] = rounded(g[j]);
      if (at_k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = y[j] <= y_k1 ? m[j] : 0;
      }
      all += (m[0] + m[1]) + (m[2] + m[3]);
      if (!near) continue;
      if (!at_k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool before = y[j] <= y_lo;
          if (before) front += m[j];
          if (!before && y[j] <= y_hi) noted |= 1u << (c * 4 + j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool before = y[j] <= y_lo;
          if (before) front += m[j];
          if (!before && (y[j] <= y_hi || (y[j] > y_k && y[j] <= y_k1))) noted |= 1u << (c * 4 + j);
        }
      }
      if (least > 0.0) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (y[j] <= y_lo && g[j] >= least) kept += m[j];
      }
    }
    if (__any_sync(0xffffffffu, noted)) {                 // one addition to the list's size per warp
      const int n = __popc(noted), upto = warp_upto(n);
      int at = 0;
      if (lane == 31) at = atomicAdd(&s.list_size, upto);
      at = __shfl_sync(0xffffffffu, at, 31) + upto - n;
      for (; noted; noted &= noted - 1, ++at) {
        const int bit = __ffs(noted) - 1, i = base + ((bit >> 2) * 32 + lane) * 4 + (bit & 3);
        const float v = i < V ? to_float<T>(x[i]) : -INFINITY;         // no NaN is in the list
        if (at < kList) {
          w.list_key[static_cast<int64_t>(row) * kList + at] = composite(v, i);
          w.list_mass[static_cast<int64_t>(row) * kList + at] = rounded(weight_within(fmaxf(v, deep), max, factor, S, table));
        }
      }
    }
    front = warp_total(front), all = warp_total(all), kept = least > 0.0 ? warp_total(kept) : front;
    if (lane == 0) {
      unsigned long long* out = w.sums + (static_cast<int64_t>(row) * w.chunks + chunk) * 3;
      out[0] = front, out[1] = all, out[2] = kept;
    }
  }
}

constexpr int kBuckets = 4096, kOwnBuckets = kBuckets / kRowThreads;

struct DrawShared {
  unsigned long long key[kList], mass[kList], chunk[kMaxChunks], scan[kRowThreads / 32];
  int bucket[kBuckets];                                   // tokens, then the place of the first one, of a step of the list's bins
  double table[64];
  int place, chunk_at;
  unsigned long long left;
};

template <typename T>
__global__ void __launch_bounds__(kRowThreads) wide_draw_kernel(const Wide w) {
  extern __shared__ __align__(16) uint8_t smem[];
  DrawShared& sh = *reinterpret_cast<DrawShared*>(smem);
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, V = w.a.vocab;
  const RowState s = w.state[row];
  if (s.skip) return;
  if (tid < 64) sh.table[tid] = kTable[tid];
  const RowParams r = row_params(w, row);
  if (s.list_size > kList) {
    if (tid == 0) leave_to_others(w, row);
    return;
  }
  const bool nucleus = r.p < 1.f;
  const int size = s.list_size, S = w.a.bits;
  const double max = r.top;
  auto weight = [&](float x) { return weight_of(x, r.top, max, r.factor, r.reach, S, sh.table); };
  auto bin_of = [&](unsigned long long key) {
    return min_of(__float2int_ru((r.top - key_value(static_cast<uint32_t>(key >> 32))) * r.step), kBins - 1);
  };
  // ---- the list in order: tokens are counted and placed by fine steps of the bracket and of the k-th token's bin (0 .. 2,047 and behind them),
  // then by the number of those before them in their step
  unsigned long long listed_all = 0;
  {
    unsigned long long key[kOwnList], mass[kOwnList];
    int bucket[kOwnList], count[kOwnBuckets], own = 0, all;
    const float near = 2047.f / (s.y_hi - s.y_lo), far = 2047.f / (s.y_k1 - s.y_k);
    for (int i = tid; i < kBuckets; i += kRowThreads) sh.bucket[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOwnList; ++j) {
      const int i = tid + j * kRowThreads;
      if (i >= size) break;
      key[j] = w.list_key[static_cast<int64_t>(row) * kList + i];
      mass[j] = w.list_mass[static_cast<int64_t>(row) * kList + i];
      listed_all += mass[j];
      const float y = (r.top - key_value(static_cast<uint32_t>(key[j] >> 32))) * r.step;
      bucket[j] = y <= s.y_hi ? __float2int_ru(fminf(fmaxf((y - s.y_lo) * near, 0.f), 2047.f))
                              : 2048 + __float2int_ru(fmaxf(fminf((y - s.y_k) * far, 2047.f), 0.f));        // NaN, of infinities, to the end
      atomicAdd(&sh.bucket[bucket[j]], 1);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kOwnBuckets; ++c) count[c] = sh.bucket[tid * kOwnBuckets + c], own += count[c];
    int first = block_upto(own, reinterpret_cast<int*>(sh.scan), all) - own;
#pragma unroll
    for (int c = 0; c < kOwnBuckets; ++c) sh.bucket[tid * kOwnBuckets + c] = first, first += count[c];
    __syncthreads();
    int slot[kOwnList];
#pragma unroll
    for (int j = 0; j < kOwnList; ++j) {
      if (tid + j * kRowThreads >= size) break;
      slot[j] = atomicAdd(&sh.bucket[bucket[j]], 1);      // afterwards the place behind the bucket
      sh.key[slot[j]] = key[j];
    }
    __syncthreads();
    int place[kOwnList];
#pragma unroll
    for (int j = 0; j < kOwnList; ++j) {
      if (tid + j * kRowThreads >= size) break;
      const int begin = bucket[j] > 0 ? sh.bucket[bucket[j] - 1] : 0, end = sh.bucket[bucket[j]];
      place[j] = begin;
      for (int i = begin; i < end; ++i) place[j] += sh.key[i] > key[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOwnList; ++j) {
      if (tid + j * kRowThreads >= size) break;
      sh.key[place[j]] = key[j], sh.mass[place[j]] = mass[j];
    }
  }
  // ---- sums in front of the list and behind it
  unsigned long long front = 0, rest = 0, ignored;
  const unsigned long long* sums = w.sums + static_cast<int64_t>(row) * w.chunks * 3;
  for (int c = tid; c < w.chunks; c += kRowThreads) {
    front += sums[c * 3], rest += sums[c * 3 + 1];
    sh.chunk[c] = sums[c * 3 + 2];
  }
  block_upto(front, sh.scan, front);
  block_upto(rest, sh.scan, rest);
  block_upto(listed_all, sh.scan, listed_all);
  rest -= front + listed_all;                             // what lies between the bracket and the k-th token's bin
  // ---- the borders: of the k-th token's bin the first left_k stay
  unsigned long long g[kOwnList], key[kOwnList], sum = 0;
  int at_k[kOwnList], before_k = 0, place = -1;           // place of the last token that is kept of the list
#pragma unroll
  for (int j = 0; j < kOwnList; ++j) {
    const int i = tid * kOwnList + j;
    key[j] = i < size ? sh.key[i] : 0;
    g[j] = i < size ? sh.mass[i] : 0;
    at_k[j] = i < size && bin_of(key[j]) == s.bin_k;
    before_k += at_k[j];
  }
  if (tid == 0) sh.place = -1;
  if (r.k > 0) {
    int upk = static_cast<int>(block_upto(static_cast<unsigned long long>(before_k), sh.scan, ignored)) - before_k;
#pragma unroll
    for (int j = 0; j < kOwnList; ++j) {
      upk += at_k[j];
      if (at_k[j] && upk == s.left_k) sh.place = tid * kOwnList + j;
      if (at_k[j] && upk > s.left_k) g[j] = 0;
    }
    __syncthreads();
    place = sh.place;
    __syncthreads();
  }
  if (nucleus) {
#pragma unroll
    for (int j = 0; j < kOwnList; ++j) sum += g[j];
    unsigned long long listed;
    unsigned long long up = block_upto(sum, sh.scan, listed);
    const double want = ceil(static_cast<double>(r.p) * static_cast<double>(front + rest + listed));
    const unsigned long long target = want > 1.0 ? static_cast<unsigned long long>(want) : 1ull;
    if (tid == 0) sh.place = kList;
    __syncthreads();
    up += front - sum;
    // the border lies behind the front and among the list's first bins, or the bins were wrong
#pragma unroll
    for (int j = 0; j < kOwnList; ++j) {
      if (up < target && up + g[j] >= target && (rest == 0 || bin_of(key[j]) <= s.bin_hi)) sh.place = tid * kOwnList + j;
      up += g[j];
    }
    __syncthreads();
    place = sh.place;
    if (place == kList || front >= target) {
      if (tid == 0) leave_to_others(w, row);
      return;
    }
  }
  // kept: tokens above the border, and of those at it the ones up to a token; without a list all
  const float edge = place >= 0 ? key_value(static_cast<uint32_t>(sh.key[place] >> 32)) : -INFINITY;
  const int edge_token = place >= 0 ? static_cast<int>(~static_cast<uint32_t>(sh.key[place])) : 0x7fffffff;
  for (int i = tid; i <= place; i += kRowThreads) {
    const unsigned long long m = sh.mass[i];
    if (m > 0 && weight(key_value(static_cast<uint32_t>(sh.key[i] >> 32))) >= r.floor_w)
      atomicAdd(&sh.chunk[static_cast<int>(~static_cast<uint32_t>(sh.key[i])) / kChunk], m);
  }
  __syncthreads();
  // ---- the chunk of the draw
  const int per = (w.chunks + kRowThreads - 1) / kRowThreads;
  unsigned long long own = 0, total;
  for (int c = tid * per; c < min_of((tid + 1) * per, w.chunks); ++c) own += sh.chunk[c];
  unsigned long long up = block_upto(own, sh.scan, total);
  unsigned long long target = static_cast<unsigned long long>(static_cast<double>(r.u) * static_cast<double>(total)) + 1;
  if (target > total) target = total;
  if (up >= target && up - own < target) {                // one thread
    unsigned long long left = target - (up - own);
    int c = tid * per;
    while (sh.chunk[c] < left) left -= sh.chunk[c++];
    sh.chunk_at = c, sh.left = left;
  }
  __syncthreads();
  // ---- its tokens, four to a thread
  const T* x = static_cast<const T*>(w.a.logits) + row * w.a.row_stride;
  const int i0 = sh.chunk_at * kChunk + tid * 4;
  unsigned long long m[4] = {0, 0, 0, 0}, four = 0;
  if (tid < kChunk / 4) {
    float v[4];
    load4(x, i0, V, false, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double gj = weight(v[j]);
      const bool in = v[j] > edge || (v[j] == edge && i0 + j <= edge_token);
      m[j] = in && gj >= r.floor_w ? rounded(gj) : 0ull;
      four += m[j];
    }
  }
  up = block_upto(four, sh.scan, ignored);
  if (up >= sh.left && up - four < sh.left) {
    unsigned long long left = sh.left - (up - four);
    int j = 0;
#pragma unroll
    for (int c = 0; c < 3; ++c)
      if (j == c && left > m[c]) left -= m[c], ++j;
    w.a.out[row] = i0 + j;
  }
}

template <typename T>
int launch_wide(const Wide& w, cudaStream_t s) {
  static bool configured[64] = {};                        // racing threads set the same attribute
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return B200_ERR_UNSUPPORTED;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(wide_draw_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(DrawShared)) != cudaSuccess) {
      cudaGetLastError();
      return B200_ERR_LAUNCH;
    }
    configured[dev] = true;
  }
  wide_top_kernel<T><<<dim3(w.slices, w.rows), kThreads, 0, s>>>(w);
  if (w.a.top_k != nullptr || w.a.top_p != nullptr)
    wide_count_kernel<T><<<dim3((w.a.vocab + w.count_tokens - 1) / w.count_tokens, w.rows), kThreads, 0, s>>>(w);
  wide_bracket_kernel<T><<<w.rows, kRowThreads, 0, s>>>(w);
  wide_sum_kernel<T><<<dim3((w.slices + w.sum_slices - 1) / w.sum_slices, w.rows), kThreads, 0, s>>>(w);
  wide_draw_kernel<T><<<w.rows, kRowThreads, sizeof(DrawShared), s>>>(w);
  return launch_result();
}

size_t aligned(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace

size_t sample_wide_workspace_bytes(int64_t rows, int vocab) {
  const size_t n = rows, slices = (vocab + kSlice - 1) / kSlice, chunks = (vocab + kChunk - 1) / kChunk;
  return aligned(n * slices * 4) + aligned(n * kBins * 4) + aligned(n * sizeof(RowState)) + 2 * aligned(n * kList * 8) + aligned(n * chunks * 24) +
         aligned((n + 1) * 4);
}

bool sample_wide_takes(int64_t rows, int vocab) { return rows <= 65535 && vocab <= kMaxChunks * kChunk; }

// `others`: where the list of the rows that are left lies in the workspace
int sample_wide_launch(const SampleArgs& a, int64_t rows, int32_t dtype, void* workspace, const int32_t** others, cudaStream_t s) {
  Wide w{};
  w.a = a;
  w.rows = static_cast<int>(rows);
  w.slices = (a.vocab + kSlice - 1) / kSlice;
  w.chunks = (a.vocab + kChunk - 1) / kChunk;
  // longer shares for less work around them, while there are CTAs for every SM several times over
  int sms = sm_count_cached();
  if (sms <= 0) sms = 148;
  w.count_tokens = kSlice;
  while (w.count_tokens < 32768 && rows * (a.vocab / (2 * w.count_tokens)) >= 4 * sms) w.count_tokens *= 2;
  w.sum_slices = 1;
  while (w.sum_slices < 4 && rows * (w.slices / (2 * w.sum_slices)) >= 8 * sms) w.sum_slices *= 2;
  const size_t n = rows;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  auto take = [&](size_t bytes) {
    uint8_t* p = at;
    at += aligned(bytes);
    return p;
  };
  w.slice_top = reinterpret_cast<uint32_t*>(take(n * w.slices * 4));
  w.hist = reinterpret_cast<uint32_t*>(take(n * kBins * 4));
  w.state = reinterpret_cast<RowState*>(take(n * sizeof(RowState)));
  w.list_key = reinterpret_cast<unsigned long long*>(take(n * kList * 8));
  w.list_mass = reinterpret_cast<unsigned long long*>(take(n * kList * 8));
  w.sums = reinterpret_cast<unsigned long long*>(take(n * w.chunks * 24));
  w.others = reinterpret_cast<int32_t*>(take((n + 1) * 4));
  *others = w.others;
  return dtype == B200_DTYPE_F32 ? launch_wide<float>(w, s) : launch_wide<__nv_bfloat16>(w, s);
}

}  // namespace b200
