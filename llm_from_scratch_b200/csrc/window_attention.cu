// Attention over a paged cache in which a query sees a sliding window and a few first tokens, for ragged portions of prompts and
// for single tokens.  The query at position p of its sequence sees key j when 0 <= p - j and (p - j < window or j < first):
//
//   out[i, h] = sum_j softmax_j(scale q[i, h] . k[j, h / G]) v[j, h / G],     zeros where no key is visible.
//
// General kernel: a warp per (query token, query head), every element type, head size and page size.  A lane owns the head-dim
// elements lane, lane + 32, ...; the visible keys are visited in order with an fp32 online softmax.  Rows that are not visible are
// never read, nor are the table entries of pages without a visible row, so freed pages may be anything.  It is for shapes that the tiled
// kernels do not take, and bound by reading every row once per query and head: 256 single tokens with a window of 4,096 at 32/8 x 128 in bf16
// 12,301 us (clusters: 315), 64 with 500 at 16/4 x 64 in fp32 672 (14.3).
#include "window_attention.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4;

template <typename T, int kPerLane>
__global__ void __launch_bounds__(kWarps * 32) window_general_kernel(const WindowArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = blockIdx.z, head = blockIdx.y;
  int64_t row, pos;                            // of the query: its row and its position in the sequence
  if (a.cu_q != nullptr) {
    const int i = blockIdx.x * kWarps + warp, q0 = a.cu_q[s], q_len = a.cu_q[s + 1] - q0;
    if (i >= q_len) return;
    row = static_cast<int64_t>(q0) + i;
    pos = static_cast<int64_t>(a.cu_k[s + 1]) - a.cu_k[s] - q_len + i;
  } else {
    row = static_cast<int64_t>(s) * kWarps + warp;
    if (row >= a.num_seqs) return;
    pos = a.lens[row] - 1;
  }
  const int64_t seq = a.cu_q != nullptr ? s : row;
  const int kvh = head / (a.Hq / a.Hkv);
  const int64_t cap = static_cast<int64_t>(a.bt_width) * a.bs;
  if (pos >= cap) {
    if (lane == 0) report(a.status, B200_ERR_BOUNDS);       // the table is too short for the context
    if (a.cu_q == nullptr) pos = cap - 1;
  }
  const T* qp = static_cast<const T*>(a.q) + row * a.q_stride + static_cast<int64_t>(head) * a.D;
  float qv[kPerLane], acc[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int d = lane + 32 * i;
    qv[i] = d < a.D ? to_float<T>(qp[d]) : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int64_t low = pos - a.window + 1, end = (pos < cap ? pos : cap - 1) + 1;
  const int32_t* table = a.bt + seq * a.bt_stride;
  for (int64_t j = low <= 0 || a.first > 0 ? 0 : low; j < end; ++j) {
    if (j < low && j >= a.first) j = low;
    if (j >= end) break;
    const int64_t id = table[j / a.bs];
    if (static_cast<uint64_t>(id) >= static_cast<uint64_t>(a.num_blocks)) {
      if (lane == 0) report(a.status, B200_ERR_BOUNDS);
      continue;
    }
    const int64_t at = (id * a.bs + j % a.bs) * a.Hkv + kvh;
    const T* kp = static_cast<const T*>(a.kc) + at * a.D;
    const T* vp = static_cast<const T*>(a.vc) + at * a.Dv;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int d = lane + 32 * i;
      if (d < a.D) dot += qv[i] * to_float<T>(kp[d]);
    }
    dot = warp_sum(dot) * a.scale_log2;
    const float mn = fmaxf(m, dot), ref = mn == -INFINITY ? 0.f : mn;      // scores of -inf alone: weights 0
    const float al = exp2f(m - ref), pw = exp2f(dot - ref);
    l = l * al + pw;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int d = lane + 32 * i;
      if (d < a.Dv) acc[i] = acc[i] * al + pw * to_float<T>(vp[d]);
    }
    m = mn;
  }
  T* op = static_cast<T*>(a.out) + (row * a.Hq + head) * a.Dv;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int d = lane + 32 * i;
    if (d < a.Dv) op[d] = from_float<T>(l == 0.f ? 0.f : acc[i] / l);      // 0: no key; a NaN stays one
  }
}

template <typename T>
int launch_general(const WindowArgs& a, int max_seqlen_q, cudaStream_t s) {
  const int wide = a.D > a.Dv ? a.D : a.Dv;
  const int z = a.cu_q != nullptr ? a.num_seqs : (a.num_seqs + kWarps - 1) / kWarps;
  if (z > 65535 || a.Hq > 65535) return B200_ERR_TOO_LARGE;
  const dim3 grid(a.cu_q != nullptr ? (max_seqlen_q + kWarps - 1) / kWarps : 1, a.Hq, z);
  if (wide <= 256) window_general_kernel<T, 8><<<grid, kWarps * 32, 0, s>>>(a);
  else window_general_kernel<T, 32><<<grid, kWarps * 32, 0, s>>>(a);
  return launch_result();
}

int check(const WindowArgs& a, int32_t dtype) {
  if (a.num_seqs < 0 || a.Hq <= 0 || a.Hkv <= 0 || a.Hq % a.Hkv != 0 || a.D <= 0 || a.Dv <= 0 || a.bs <= 0 || a.num_blocks < 0 ||
      (a.num_seqs > 0 && a.bt_width <= 0) || a.bt_stride < 0 || a.window < 1 || a.first < 0)
    return B200_ERR_ARG;
  if (dtype != B200_DTYPE_F32 && dtype != B200_DTYPE_BF16) return B200_ERR_UNSUPPORTED;
  if (a.D > 1024 || a.Dv > 1024) return B200_ERR_UNSUPPORTED;
  return B200_OK;
}

bool given(const WindowArgs& a) { return a.q && a.kc && a.vc && a.out && a.bt && (a.cu_q ? a.cu_k != nullptr : a.lens != nullptr); }

int general(const WindowArgs& a, int max_seqlen_q, int32_t dtype, cudaStream_t s) {
  return dtype == B200_DTYPE_F32 ? launch_general<float>(a, max_seqlen_q, s) : launch_general<__nv_bfloat16>(a, max_seqlen_q, s);
}

int dispatch(const WindowArgs& given_args, int64_t total_q, int max_seqlen_q, int32_t dtype, cudaStream_t s) {
  WindowArgs a = given_args;
  int rc = B200_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(a.bt_width) * a.bs <= kMaxPosition) {
    if (a.window > kMaxPosition) a.window = kMaxPosition;
    if (a.first > kMaxPosition) a.first = kMaxPosition;
    if (dtype == B200_DTYPE_BF16) rc = a.cu_q != nullptr ? window_prefill_launch(a, total_q, s) : window_decode_launch(a, s);
    else rc = a.cu_q != nullptr ? window_prefill_f32_launch(a, total_q, max_seqlen_q, s) : window_decode_f32_launch(a, s);
  }
  return rc == B200_ERR_UNSUPPORTED ? general(given_args, max_seqlen_q, dtype, s) : rc;
}

}  // namespace
}  // namespace b200

extern "C" int b200_window_attention(const void* q, int64_t q_token_stride, const void* k_cache, const void* v_cache, void* out,
                                     int64_t total_q, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t num_seqs,
                                     int32_t max_seqlen_q, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim_qk,
                                     int32_t head_dim_v, float scale, const int32_t* block_tables, int64_t bt_stride,
                                     int32_t bt_width, int32_t block_size, int64_t num_blocks, int32_t window, int32_t first, int32_t dtype,
                                     int32_t* status, void* stream) {
  using namespace b200;
  WindowArgs a{};
  a.q = q, a.kc = k_cache, a.vc = v_cache, a.out = out;
  a.q_stride = q_token_stride;
  a.cu_q = cu_seqlens_q, a.cu_k = cu_seqlens_k;
  a.num_seqs = num_seqs, a.Hq = num_q_heads, a.Hkv = num_kv_heads, a.D = head_dim_qk, a.Dv = head_dim_v, a.bs = block_size;
  a.bt = block_tables, a.bt_stride = bt_stride, a.bt_width = bt_width, a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.window = window, a.first = first;
  a.status = status;
  const int rc = check(a, dtype);
  if (rc != B200_OK) return rc;
  if (total_q < 0 || max_seqlen_q < 0) return B200_ERR_ARG;
  if (num_seqs == 0 || total_q == 0 || max_seqlen_q == 0) return B200_OK;
  if (!cu_seqlens_q || !given(a)) return B200_ERR_ARG;
  return dispatch(a, total_q, max_seqlen_q, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int b200_window_decode(const void* q, const void* k_cache, const void* v_cache, void* out, const int32_t* block_tables,
                                  int64_t bt_stride, int32_t bt_width, const int64_t* context_lens, int32_t batch, int32_t num_q_heads,
                                  int32_t num_kv_heads, int32_t head_dim_qk, int32_t head_dim_v, int32_t block_size,
                                  int64_t num_blocks, float scale, int32_t window, int32_t first, int32_t dtype, int32_t* status,
                                  void* stream) {
  using namespace b200;
  WindowArgs a{};
  a.q = q, a.kc = k_cache, a.vc = v_cache, a.out = out;
  a.q_stride = static_cast<int64_t>(num_q_heads) * head_dim_qk;
  a.lens = context_lens;
  a.num_seqs = batch, a.Hq = num_q_heads, a.Hkv = num_kv_heads, a.D = head_dim_qk, a.Dv = head_dim_v, a.bs = block_size;
  a.bt = block_tables, a.bt_stride = bt_stride, a.bt_width = bt_width, a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.window = window, a.first = first;
  a.status = status;
  const int rc = check(a, dtype);
  if (rc != B200_OK) return rc;
  if (batch == 0) return B200_OK;
  if (!given(a)) return B200_ERR_ARG;
  return dispatch(a, batch, 1, dtype, static_cast<cudaStream_t>(stream));
}
