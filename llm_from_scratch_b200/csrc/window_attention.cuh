// Arguments shared by the kernels of attention with a sliding window and visible first tokens (window_attention.cu).
#pragma once

#include "common.cuh"

namespace b200 {

struct WindowArgs {
  const void* q;             // [tokens, Hq, D], token stride q_stride
  const void* kc;            // [num_blocks, bs, Hkv, D]
  const void* vc;            // [num_blocks, bs, Hkv, Dv]
  void* out;                 // [tokens, Hq, Dv]
  int64_t q_stride;
  const int32_t* cu_q;       // portions: [num_seqs + 1]; null: one token per sequence
  const int32_t* cu_k;
  const int64_t* lens;       // single tokens: [num_seqs]
  int num_seqs, Hq, Hkv, D, Dv, bs;
  const int32_t* bt;         // [num_seqs, bt_width], row stride bt_stride
  int64_t bt_stride, num_blocks;
  int bt_width;
  float scale_log2;
  int window, first;
  int32_t* status;
};

// The tiled kernels count positions in 32 bits: a window or a number of first tokens beyond every position is cut to this one.
constexpr int kMaxPosition = 1 << 30;

// Launches of the tiled kernels; B200_ERR_UNSUPPORTED: a shape, page size or alignment that the general kernel takes.
int window_prefill_launch(const WindowArgs& a, int64_t total_q, cudaStream_t s);                       // bf16, head sizes 64 and 128
int window_decode_launch(const WindowArgs& a, cudaStream_t s);                                         // bf16, head sizes 64 and 128
int window_prefill_f32_launch(const WindowArgs& a, int64_t total_q, int max_seqlen_q, cudaStream_t s); // head sizes 32, 64 and 128
int window_decode_f32_launch(const WindowArgs& a, cudaStream_t s);                                     // head sizes 32, 64 and 128

}  // namespace b200
