// Pieces of filtered sampling that its kernels share (sample_filtered.cu, sample_wide.cu): the order of the tokens and their weights.
#pragma once

#include "common.cuh"

namespace b200 {

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

__device__ __forceinline__ int min_of(int x, int y) { return x < y ? x : y; }
__device__ __forceinline__ int max_of(int x, int y) { return x > y ? x : y; }
__device__ __forceinline__ uint32_t max_key(uint32_t x, uint32_t y) { return x > y ? x : y; }

constexpr double kMagic = 6755399441055744.0;            // 1.5 * 2^52: added, it leaves the nearest whole number in the low bits

// 2^(i / 64)
__device__ const double kTable[64] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951};

// The weight in units of 2^-S by reduction to a table and a short series: 2^(n / 64) 2^(r / 64) with |r| <= 1/2, the second factor by its series up to r^4 (error 4e-14).
// For logits no further from the maximum than 600 T.
__device__ __forceinline__ double weight_within(float x, double max, double factor, int S, const double* table) {
  const double y = (static_cast<double>(x) - max) * factor;
  const double t = y + kMagic, r = y - (t - kMagic);
  const int n = __double2loint(t);
  constexpr double b = 0.010830424696249145;             // ln 2 / 64
  const double q = fma(r, fma(r, fma(r, fma(r, b * b * b * b / 24, b * b * b / 6), b * b / 2), b), 1.0);
  const double v = table[n & 63] * q;
  return __hiloint2double(__double2hiint(v) + (((n >> 6) + S) << 20), __double2loint(v));
}
// For any: 0 beyond `reach`.
__device__ __forceinline__ double weight_of(float x, float top, double max, double factor, float reach, int S, const double* table) {
  const double w = weight_within(x, max, factor, S, table);
  return top - x > reach ? 0.0 : w;
}

// A weight as a whole number, below 2^51; 0 for weights below e^-32 where the unit is 2^-45.
__device__ __forceinline__ unsigned long long rounded(double w) {
  return static_cast<unsigned long long>(__double_as_longlong(w + 4503599627370496.0)) & 0xfffffffffffffull;
}

// Order of the tokens: larger is earlier.
__device__ __forceinline__ unsigned long long composite(float x, int i) {
  return static_cast<unsigned long long>(order_key(x)) << 32 | static_cast<uint32_t>(~i);
}

// Sum over the warp, in all lanes: three parts of 24 bits, whose sums fit 32.
__device__ __forceinline__ unsigned long long warp_total(unsigned long long v) {
  const uint32_t lo = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v) & 0xffffffu);
  const uint32_t mid = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v >> 24) & 0xffffffu);
  const uint32_t hi = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v >> 48));
  return lo + (static_cast<unsigned long long>(mid) << 24) + (static_cast<unsigned long long>(hi) << 48);
}
template <typename U>
__device__ __forceinline__ U warp_upto(U v) {            // inclusive running sum over the lanes
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const U y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// Sorts n keys, highest first, and the masses with them.  Up to THREADS / 4 keys by the number of those before each, more by a bitonic network (in the
// tail that makes a power of two of n: keys 0), for which the arrays have room.  Every thread of the CTA calls it; a barrier in front and behind.
template <int THREADS>
__device__ __forceinline__ void sort_by_key(unsigned long long* key, unsigned long long* mass, int n) {
  __syncthreads();
  if (n <= THREADS / 4) {
    const int i = threadIdx.x;
    unsigned long long k = 0, m = 0;
    int place = 0;
    if (i < n) {
      k = key[i], m = mass[i];
#pragma unroll 4
      for (int j = 0; j < n; ++j) place += key[j] > k;
    }
    __syncthreads();
    if (i < n) key[place] = k, mass[place] = m;
    __syncthreads();
    return;
  }
  int all = 2;
  while (all < n) all *= 2;
  for (int i = n + threadIdx.x; i < all; i += THREADS) key[i] = 0, mass[i] = 0;
  __syncthreads();
#pragma unroll 1
  for (int size = 2; size <= all; size *= 2)
#pragma unroll 1
    for (int step = size / 2; step > 0; step /= 2) {
#pragma unroll 1
      for (int i = threadIdx.x; i < all / 2; i += THREADS) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;           // the i-th pair at this distance
        const unsigned long long x = key[lo], y = key[hi];
        if ((lo & size) == 0 ? x < y : x > y) {
          const unsigned long long mx = mass[lo], my = mass[hi];
          key[lo] = y, key[hi] = x;
          mass[lo] = my, mass[hi] = mx;
        }
      }
      __syncthreads();
    }
}

// Where the tokens of a bin lie that is told by b = ceil((top - x) step): their mean distance from the maximum in bins and its variance, if
// all logits that the bin can hold are equally likely.  fp32: anywhere in it.  bf16 (GRID): on a grid, which meets the bins anywhere and is often
// coarser than they are; with their middles instead, sums of weights would be off by half a bin to one side.  An estimate only: it narrows down
// where borders lie, and what rests on it is checked with the weights.
template <bool GRID>
struct BinPlaces {
  float top, step, width;
  __device__ __forceinline__ BinPlaces(float top, float step) : top(top), step(step), width(1.f / step) {}
  __device__ __forceinline__ float of(int b, float& variance) const {
    variance = b == 0 ? 0.f : 1.f / 12.f;
    if (!GRID || b == 0) return b == 0 ? 0.f : b - 0.5f;
    const float middle = top - (b - 0.5f) * width;
    const uint32_t exponent = max(__float_as_uint(middle) & 0x7f800000u, 0x10000000u) - (7u << 23);      // eight bits of a number
    const float grain = __uint_as_float(exponent), per = __uint_as_float(0x7f000000u - exponent);        // a power of two and its reciprocal
    auto bin = [&](float x) { return ceilf((top - x) * step); };
    float high = floorf((top - (b - 1) * width) * per) * grain, low = ceilf((top - b * width) * per) * grain;
    if (bin(high) < b) high -= grain;
    else if (bin(high + grain) == b) high += grain;
    if (bin(low) > b) low += grain;
    else if (bin(low - grain) == b) low -= grain;
    if (!(low <= high)) low = high = rintf(middle * per) * grain;          // none: the next one
    const float n = (high - low) * per + 1.f, apart = grain * step;
    variance = apart * apart * (n * n - 1.f) * (1.f / 12.f);
    return fminf(fmaxf((top - 0.5f * (high + low)) * step, b - 1.f), static_cast<float>(b));
  }
};

// Many long rows (sample_wide.cu): rows that it leaves to the other form are named in `others`, their number first.
size_t sample_wide_workspace_bytes(int64_t rows, int vocab);
bool sample_wide_takes(int64_t rows, int vocab);
int sample_wide_launch(const SampleArgs& a, int64_t rows, int32_t dtype, void* workspace, const int32_t** others, cudaStream_t s);

}  // namespace b200
