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
// Every border is found by one routine, a radix selection over bytes with the weights (or ones) as masses.
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
  const int grid = static_cast<int>(num_rows);
  if (dtype == B200_DTYPE_F32) sample_filtered_kernel<float><<<grid, kThreads, 0, s>>>(a);
  else sample_filtered_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
  return launch_result();
}
