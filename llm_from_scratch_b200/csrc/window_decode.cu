// Attention over a sliding window and the first tokens for single tokens in bf16, head sizes 64 and 128, pages of a multiple of 16 tokens.
//
// Bound by reading every visible K and V row once.  A cluster of CTAs shares the visible keys of a (sequence, KV head), a CTA takes up to
// sixteen query heads; a warp takes every fourth 16-token block of its CTA's share, and the pieces meet in shared memory, then in the
// cluster's distributed shared memory.  The window bounds the work of a sequence, and the host knows it, so no pass over the lengths is needed
// and there is no scratch in global memory.  Products and softmax are those of decode_cluster.cu: the query heads are the N dimension
// of mma.sync m16n8k16 (a decode step has too few rows for tcgen05, and the tensor pipe idles either way), S^T = K Q^T and O^T = V^T P^T,
// scores and sums in fp32, weights rounded to bf16 for the second product (2^-8 of a weight, and the tensor cores take nothing wider beside
// bf16 values).  Rows arrive by cp.async, swizzled, blocks ahead; a row that is not visible is not read, zeros take its place.
//
// Measured at 32/8 x 128: a sequence with a window of 1,024 and 4 first tokens 6.2 us, of which a launch is half and the rest a chain of dependent
// reads (length, table, rows) and the two merges; 256 sequences with a window of 4,096, 2.08 GB of rows, 315 us, 6.6 TB/s.
#include <cooperative_groups.h>

#include "window_attention.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = kWarps * 32, kTok = 16;

template <int D, int NT>
struct Lay {
  static constexpr int tile = kTok * D * 2;                           // K or V rows of a block
  static constexpr int stages = D == 128 ? 3 : 4;                     // blocks of a warp in flight
  static constexpr int ring = kWarps * stages * 2 * tile;
  static constexpr int LDO = D + 4;
  static constexpr int pieces = kWarps * NT * 8 * LDO * 4;            // over the ring
  static constexpr int bytes = ring > pieces ? ring : pieces;
};

struct StepArgs {
  WindowArgs w;
  int sub;                   // 16-token blocks of a page
  int chunks;                // of up to 16 query heads per KV head
  int least;                 // blocks of a CTA at least
};

template <int D, int NT>
__global__ void __launch_bounds__(kThreads) window_decode_kernel(const StepArgs p) {
  using L = Lay<D, NT>;
  constexpr int ROWB = D * 2, CPR = D / 8, KS = D / 16, LOADS = kTok * CPR / 32, kStages = L::stages;
  const WindowArgs& a = p.w;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][NT * 8], s_l[kWarps][NT * 8];
  __shared__ __align__(16) float c_o[NT * 8][D];       // of the CTA, read by the cluster
  __shared__ float c_m[NT * 8], c_l[NT * 8];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ranks = cluster.num_blocks();
  const int seq = blockIdx.z, h = blockIdx.y / p.chunks, all = a.Hq / a.Hkv, head0 = h * all + blockIdx.y % p.chunks * (NT * 8);
  const int G = min(all - blockIdx.y % p.chunks * (NT * 8), NT * 8);   // query heads of this CTA
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
  auto swizzle = [](int c, int t) { return c ^ (t & 7); };

  uint32_t qf[NT][KS][2];                              // in flight with the length
  const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(a.q) + (static_cast<int64_t>(seq) * a.Hq + head0) * D;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int head = nt * 8 + g;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(qp + head * D + ks * 16 + tq * 2);
      qf[nt][ks][0] = head < G ? __ldg(src) : 0u;
      qf[nt][ks][1] = head < G ? __ldg(src + 4) : 0u;
    }
  int64_t len64 = a.lens[seq];
  const int64_t cap = static_cast<int64_t>(a.bt_width) * a.bs;
  if (len64 > cap) {
    if (tid == 0) report(a.status, B200_ERR_BOUNDS);   // table row too short for the context
    len64 = cap;
  }
  const int len = len64 > 0 ? static_cast<int>(len64) : 0;
  // ---- visible blocks: 0 .. nf - 1 with first tokens, then those from `start` on
  const int low = max(len - a.window, 0), first = min(a.first, low), start = low / kTok, nf = min((first + kTok - 1) / kTok, start);
  const int blocks = nf + (len + kTok - 1) / kTok - start;
  // this CTA's share, of it every kWarps-th block for a warp.  CTAs without one leave: a barrier of the cluster counts the threads that are
  // still there, and nobody reads what they hold.
  const int per = max((blocks + ranks - 1) / ranks, p.least), used = max((blocks + per - 1) / per, 1);
  if (rank >= used) return;
  const int lo = min(rank * per, blocks) + warp, hi = min((rank + 1) * per, blocks);
  const int mine = lo < hi ? (hi - lo + kWarps - 1) / kWarps : 0;
  const int32_t* table = a.bt + static_cast<int64_t>(seq) * a.bt_stride;
  const uint32_t ring = smem_u32(smem) + warp * (kStages * 2 * L::tile);
  const int64_t row_stride = static_cast<int64_t>(a.Hkv) * ROWB;
  const uint8_t* kbase = static_cast<const uint8_t*>(a.kc) + static_cast<int64_t>(h) * ROWB;
  const uint8_t* vbase = static_cast<const uint8_t*>(a.vc) + static_cast<int64_t>(h) * ROWB;
  auto block_of = [&](int i) -> int {                  // number of the warp's i-th block in the context
    const int b = lo + i * kWarps;
    return b < nf ? b : b - nf + start;
  };
  int id_lane = -1;                                    // page of this lane's block of the current 32
  uint32_t found = 0;                                  // of the current 32: pages in the pool
  uint32_t found_before = 0;                           // of the 32 before them, some of which are still in flight
  auto issue = [&](int i) {
    if (i % 32 == 0) {
      id_lane = -1;
      if (i + lane < mine) {
        const int blk = block_of(i + lane);
        id_lane = __ldg(table + (p.sub == 1 ? blk : blk / p.sub));
        if (static_cast<uint64_t>(static_cast<int64_t>(id_lane)) >= static_cast<uint64_t>(a.num_blocks)) {
          report(a.status, B200_ERR_BOUNDS);
          id_lane = -1;
        }
      }
      found_before = found;
      found = __ballot_sync(0xffffffffu, id_lane >= 0);
    }
    const int id = __shfl_sync(0xffffffffu, id_lane, i % 32), blk = block_of(i);
    const int64_t at = id >= 0 ? (static_cast<int64_t>(id) * p.sub + (p.sub == 1 ? 0 : blk % p.sub)) * kTok * row_stride : 0;
    const uint32_t kdst = ring + i % kStages * (2 * L::tile), vdst = kdst + L::tile;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int idx = lane + 32 * j, t = idx / CPR, c = idx % CPR, key = blk * kTok + t;
      const int bytes = id >= 0 && key < len && (key >= low || key < first) ? 16 : 0;
      const int64_t from = at + (bytes ? t * row_stride + c * 16 : 0);
      const uint32_t d = t * ROWB + swizzle(c, t) * 16;
      cp_async16(kdst + d, kbase + from, bytes);
      cp_async16(vdst + d, vbase + from, bytes);
    }
  };
  float o[NT][KS][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
  }
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (s < mine) issue(s);
    cp_async_commit();
  }
  for (int i = 0; i < mine; ++i) {
    if (i + kStages - 1 < mine) issue(i + kStages - 1);
    cp_async_commit();
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t kt = ring + i % kStages * (2 * L::tile), vt = kt + L::tile;
    const int key = block_of(i) * kTok + g;            // of this lane's first token; the second is 8 behind it
    // the block's page: among the 32 of the last issue, or of those before them
    const int ahead = min(i + kStages - 1, mine - 1);
    const bool in_pool = ((ahead / 32 == i / 32 ? found : found_before) >> (i % 32)) & 1;
    const bool seen[2] = {in_pool && key < len && (key >= low || key < first), in_pool && key + 8 < len && (key + 8 >= low || key + 8 < first)};
    // ---- S^T[token, head] = K Q^T
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
    {
      const int t = (lane & 7) + ((lane >> 3) & 1) * 8, ch = lane >> 4;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t af[4];
        ldmatrix_x4(af, kt + t * ROWB + swizzle(2 * ks + ch, t) * 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(s[nt], af, qf[nt][ks]);
      }
    }
    // ---- online softmax over the tokens g, g + 8
    uint32_t pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = seen[e >> 1] ? s[nt][e] * a.scale_log2 : -INFINITY;
      float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
      }
      float w[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float mn = fmaxf(m[nt][e], mx[e]), ref = mn == -INFINITY ? 0.f : mn;     // scores of -inf alone: weights 0
        const float al = fast_exp2(m[nt][e] - ref);
        m[nt][e] = mn;
        w[e] = fast_exp2(x[e] - ref);
        w[e + 2] = fast_exp2(x[e + 2] - ref);
        l[nt][e] = l[nt][e] * al + w[e] + w[e + 2];
#pragma unroll
        for (int mt = 0; mt < KS; ++mt) {
          o[nt][mt][e] *= al;
          o[nt][mt][e + 2] *= al;
        }
      }
      pb[nt][0] = movmatrix_trans(pack_bf16x2(w[0], w[1]));
      pb[nt][1] = movmatrix_trans(pack_bf16x2(w[2], w[3]));
    }
    // ---- O^T[d, head] += V^T P^T
    {
      const int t = (lane & 7) + (lane >> 4) * 8, ch = (lane >> 3) & 1;
#pragma unroll
      for (int mt = 0; mt < KS; ++mt) {
        uint32_t af[4];
        ldmatrix_x4_trans(af, vt + t * ROWB + swizzle(2 * mt + ch, t) * 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(o[nt][mt], af, pb[nt]);
      }
    }
    __syncwarp();                                      // the stage may be refilled
  }
  cp_async_wait<0>();
  __syncthreads();                                     // the ring becomes the warps' pieces
  // ---- warps of the CTA
  float* pieces = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int head = nt * 8 + tq * 2 + e;
      float sum = l[nt][e];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      float* row = pieces + (warp * NT * 8 + head) * L::LDO + g;
#pragma unroll
      for (int mt = 0; mt < KS; ++mt) {
        row[mt * 16] = o[nt][mt][e];
        row[mt * 16 + 8] = o[nt][mt][e + 2];
      }
      if (g == 0) s_m[warp][head] = m[nt][e], s_l[warp][head] = sum;
    }
  __syncthreads();
  for (int i = tid; i < G * (D / 4); i += kThreads) {
    const int head = i / (D / 4), d = i % (D / 4) * 4;
    float M = s_m[0][head];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[w][head]);
    float sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_m[w][head] == -INFINITY ? 0.f : exp2f(s_m[w][head] - M);
      const float4 y = *reinterpret_cast<const float4*>(pieces + (w * NT * 8 + head) * L::LDO + d);
      x.x += f * y.x, x.y += f * y.y, x.z += f * y.z, x.w += f * y.w;
      sum += f * s_l[w][head];
    }
    *reinterpret_cast<float4*>(&c_o[head][d]) = x;
    if (d == 0) c_m[head] = M, c_l[head] = sum;
  }
  if (used > 1) cluster.sync();
  else __syncthreads();
  // ---- CTAs of the cluster: every one finishes its share of the columns
  for (int i = rank * kThreads + tid; i < G * (D / 2); i += used * kThreads) {
    const int head = i / (D / 2), d = i % (D / 2) * 2;
    float mr[8], lr[8], M = -INFINITY;
    float2 y[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < used) {
        mr[r] = *cluster.map_shared_rank(&c_m[head], r);
        lr[r] = *cluster.map_shared_rank(&c_l[head], r);
        y[r] = *reinterpret_cast<const float2*>(cluster.map_shared_rank(&c_o[head][d], r));
        M = fmaxf(M, mr[r]);
      }
    float sum = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < used) {
        const float f = mr[r] == -INFINITY ? 0.f : exp2f(mr[r] - M);
        sum += f * lr[r];
        x0 += f * y[r].x;
        x1 += f * y[r].y;
      }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;    // an empty context gives zeros; a NaN stays one
    *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + (static_cast<int64_t>(seq) * a.Hq + head0 + head) * D + d) =
        pack_bf16x2(x0 * inv, x1 * inv);
  }
  if (used > 1) cluster.sync();                        // nobody leaves while another CTA reads its shared memory
}

template <int D, int NT>
int launch(const StepArgs& p, int ranks, cudaStream_t s) {
  constexpr int smem = Lay<D, NT>::bytes;
  static bool configured[64] = {false};                // racing threads set the same attribute
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    if (cudaFuncSetAttribute(window_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
      cudaGetLastError();
      return B200_ERR_LAUNCH;
    }
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, p.w.Hkv * p.chunks, p.w.num_seqs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launch_result(cudaLaunchKernelEx(&cfg, window_decode_kernel<D, NT>, p));
}

}  // namespace

int window_decode_launch(const WindowArgs& a, cudaStream_t s) {
  const int G = a.Hq / a.Hkv;
  if (a.D != a.Dv || (a.D != 64 && a.D != 128) || a.bs % kTok != 0 || a.num_seqs > 65535 || !aligned16(a.q) || !aligned16(a.kc) ||
      !aligned16(a.vc) || !aligned16(a.out))
    return B200_ERR_UNSUPPORTED;
  int sms = sm_count_cached();
  if (sms <= 0) sms = 148;
  StepArgs p{a, a.bs / kTok, (G + 15) / 16, kWarps};
  if (static_cast<int64_t>(a.Hkv) * p.chunks > 65535) return B200_ERR_UNSUPPORTED;
  const int64_t units = static_cast<int64_t>(a.num_seqs) * a.Hkv * p.chunks, wave = 2 * static_cast<int64_t>(sms);
  int64_t keys = static_cast<int64_t>(a.bt_width) * a.bs;               // that a sequence may see
  if (keys > static_cast<int64_t>(a.window) + a.first) keys = static_cast<int64_t>(a.window) + a.first;
  // CTAs per (sequence, KV head): doubled up to two an SM, none with fewer than four blocks of its own (one, two, four, eight, 32/8 x 128: 1 sequence
  // with 512 visible keys 9.3, 7.2, 6.0, 5.6 us, with 16,384 173, 89, 47, 26; 16 with 1,024 15.6, 15.4, 19.9, 29.1, with 16,384 175, 161,
  // 161, 169; 64 with 512 28, 38, 51, 88, with 4,096 158, 163, 172, 201)
  int ranks = 1;
  while (ranks < 8 && static_cast<int64_t>(ranks) * kWarps * kTok < keys && units * ranks * 2 <= wave) ranks *= 2;
  if (G > 8) return a.D == 128 ? launch<128, 2>(p, ranks, s) : launch<64, 2>(p, ranks, s);
  return a.D == 128 ? launch<128, 1>(p, ranks, s) : launch<64, 1>(p, ranks, s);
}

}  // namespace b200
