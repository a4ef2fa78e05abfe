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

}  // namespace b200
