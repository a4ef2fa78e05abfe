// Attention over a sliding window and the first tokens for portions of prompts in bf16, head sizes 64 and 128, on the Blackwell tensor cores:
// keys and values are read from the pages of the cache.
//
// A row of a tile is a (query token, query head) pair, the heads of one KV head beside each other, so that a staged K / V tile serves all of
// them and a tile of 128 rows spans 128 / G tokens only: the window of its first row and that of its last differ by as little.  A CTA owns
// two such tiles, problems A and B, that walk the same tiles of 64 keys: those with first tokens, then those from the start of A's window
// on.  The warps' parts are those of prefill_umma2.cu:
//
//   warp 0      K producer (+ both Q tiles): a lane per box, a box being 64 columns of the keys of one page (at most 64)
//   warp 1      V producer
//   warp 2      tensor-memory allocation; lane 0 issues the tcgen05.mma of problem A
//   warp 3      lane 0 issues the tcgen05.mma of problem B
//   warps 4-7   softmax of A: a thread per row, the 64 scores of a tile in registers
//   warps 8-11  softmax of B
//
// Tensor memory per problem: two score buffers of 64 columns (bf16 P overwrites the first half of its buffer and is the A operand of
// O += P.V) and O.  Scores are issued a tile ahead, O is rescaled lazily, and the exponentials of the two problems take turns (see there).
//
// At head size 64 a problem has a CTA of its own, and two CTAs share an SM (portions below: 45 us; two problems in one CTA 48).
//
// Measured: 4 prompts of 8,192 at 32/8 x 128, window 4,096, 1.65 TFLOP: 1,570 .. 1,820 us, 0.91 .. 1.05 PFLOP/s with the clock under the power cap.
// Bound by the exponentials, 16 a clock and SM.  Without the turns 1,747 us against 1,618 in the same minute; a quarter of the exponentials by
// polynomial 1,765, half 2,064.  24 portions of 1 .. 1,000 tokens, 3,930 in all, behind up to 8,000, 16/4 x 64, window 1,024: 45 us (a warp per
// row: 10,886), two rounds of CTAs whose rows pass 18 tiles one after the other: 1,400 cycles a tile (wait 250, scores and maximum 360,
// exponentials 650, of which the unit needs 512), 5,000 before the first and 2,000 behind the last.
//
// P is rounded to bf16, the type that the tensor cores take beside bf16 values: 2^-8 of a weight.  Sums of weights are taken before that, in fp32.
//
// Boxes whose keys no row of the CTA sees are not read: their coordinate lies behind the pool, where a copy delivers zeros.  What is
// left are keys that some rows see and others do not.  Their scores become -inf in the other rows, but a weight of 0 would still turn an
// infinity or NaN of the value row into a NaN: tiles in which some row is cut are searched for one, and a CTA that finds one
// computes all its rows again, key by key, at its end.  The same way it leaves out keys of pages outside the pool.  That costs: the portions
// above with NaN behind the ends of 20 of the contexts, where pools that were not filled can hold some, take 10.7 ms instead of 45 us (the 32
// tokens of a CTA times 4 heads read their keys one by one).  The engine's pools start as zeros.
#include <cuda.h>

#include "umma.cuh"
#include "window_attention.cuh"

namespace b200 {
namespace {

constexpr int BM = 128, BN = 64;
constexpr int Q_SLAB = BM * 128;           // 64 columns of 128 rows
constexpr int K_SLAB = BN * 128;           // 64 columns of 64 keys
constexpr float kRescaleThreshold = 8.f;   // log2 units

// NP: problems of a CTA
template <int D, int NP>
struct Lay {
  static constexpr int kThreads = 128 + NP * 128;
  static constexpr int S = D / 64;
  static constexpr int Q_BYTES = S * Q_SLAB, K_BYTES = S * K_SLAB, STAGE = 2 * K_BYTES;
  static constexpr int NST = 4;
  static constexpr int OFF_KV = NP * Q_BYTES, OFF_BAR = OFF_KV + NST * STAGE;
  // as in prefill_umma2.cu
  static constexpr int Q_FULL = 0, K_FULL = 1, V_FULL = 1 + NST, QK_DONE = 1 + 2 * NST, PV_DONE = 1 + 4 * NST, P_READY = 1 + 6 * NST,
                       TURN = P_READY + 4, LEFT = TURN + 8, NUM_BARS = LEFT + NP;
  static constexpr int SMEM = OFF_BAR + NUM_BARS * 8 + 32 + 1024;
  static constexpr int TCOLS = NP * (128 + D) > 256 ? 512 : 256;
};

struct PromptArgs {
  WindowArgs w;
  int G, tokens;             // query heads of a KV head; tokens of a problem
  int box;                   // keys of a box
};

// The tile of query tokens of a CTA: tile number -> (sequence, tile within it); false: there are fewer tiles.  One warp calls it.
__device__ __forceinline__ bool find_tile(const int32_t* cu_q, int n, int per, int number, int* seq, int* tile) {
  const int lane = threadIdx.x & 31;
  int left = number;
  for (int base = 0; base < n; base += 32) {
    const int s = base + lane;
    const int t = s < n ? (cu_q[s + 1] - cu_q[s] + per - 1) / per : 0;
    int upto = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, left < upto);
    if (hit) {
      const int src = __ffs(hit) - 1;
      *seq = base + src;
      *tile = left - __shfl_sync(0xffffffffu, upto - t, src);
      return true;
    }
    left -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

// One row, key by key: what the tensor cores do, without a key that the row does not see.  A warp calls it.
template <int D>
__device__ __noinline__ void plain_row(const WindowArgs& a, int seq, int64_t row, int head, int pos) {
  const int lane = threadIdx.x & 31, kvh = head / (a.Hq / a.Hkv);
  constexpr int N = D / 32;
  const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(a.q) + row * a.q_stride + static_cast<int64_t>(head) * D + lane * N;
  float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = __bfloat162float(qp[i]), o[i] = 0.f;
  const int low = pos - a.window + 1;
  const int32_t* table = a.bt + seq * a.bt_stride;
  for (int j = a.first > 0 ? 0 : max(low, 0); j <= pos; ++j) {
    if (j < low && j >= a.first) j = low;
    const int page = j / a.bs;
    const int64_t id = page < a.bt_width ? table[page] : -1;
    if (static_cast<uint64_t>(id) >= static_cast<uint64_t>(a.num_blocks)) continue;       // the producer has reported it
    const int64_t at = ((id * a.bs + j % a.bs) * a.Hkv + kvh) * D + lane * N;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) dot += q[i] * __bfloat162float(static_cast<const __nv_bfloat16*>(a.kc)[at + i]);
    dot = warp_sum(dot) * a.scale_log2;
    const float mn = fmaxf(m, dot), ref = mn == -INFINITY ? 0.f : mn;
    const float al = exp2f(m - ref), p = exp2f(dot - ref);
    l = l * al + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * al + p * __bfloat162float(static_cast<const __nv_bfloat16*>(a.vc)[at + i]);
    m = mn;
  }
  __nv_bfloat16* op = static_cast<__nv_bfloat16*>(a.out) + (row * a.Hq + head) * D + lane * N;
#pragma unroll
  for (int i = 0; i < N; ++i) op[i] = __float2bfloat16_rn(l == 0.f ? 0.f : o[i] / l);
}

template <int D, int NP>
__global__ void __launch_bounds__(Lay<D, NP>::kThreads, NP == 1 ? 2 : 1)
window_prefill_kernel(const PromptArgs p, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v) {
  using L = Lay<D, NP>;
  constexpr int NST = L::NST, kThreads = L::kThreads;
  const WindowArgs& a = p.w;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_tile[2];
  __shared__ int s_again;                    // the rows have to be computed key by key
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sb = smem_u32(smem);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L::OFF_BAR + L::NUM_BARS * 8);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::OFF_BAR + L::NUM_BARS * 8 + 8);
  auto bar = [&](int i) -> uint32_t { return sb + L::OFF_BAR + i * 8; };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x % a.Hkv;

  if (warp == 0) {
    int seq = -1, tile = 0;
    find_tile(a.cu_q, a.num_seqs, NP * p.tokens, blockIdx.x / a.Hkv, &seq, &tile);
    if (lane == 0) s_tile[0] = seq, s_tile[1] = tile, s_again = 0;
  } else if (tid == 32) {
    umma::mbar_init(bar(L::Q_FULL), 1);
    for (int s = 0; s < NST; ++s) {
      umma::mbar_init(bar(L::K_FULL + s), 1);
      umma::mbar_init(bar(L::V_FULL + s), 1);
      for (int x = 0; x < 2; ++x) {
        umma::mbar_init(bar(L::QK_DONE + 2 * s + x), 1);
        umma::mbar_init(bar(L::PV_DONE + 2 * s + x), 1);
      }
    }
    for (int i = 0; i < 4; ++i) umma::mbar_init(bar(L::P_READY + i), 128);
    for (int i = 0; i < 8; ++i) umma::mbar_init(bar(L::TURN + i), 32);
    for (int x = 0; x < NP; ++x) umma::mbar_init(bar(L::LEFT + x), 1);
    *s_abort = 0;
    umma::mbar_init_fence();
  }
  __syncthreads();
  const int seq = s_tile[0];
  if (seq < 0) return;                       // uniform over the CTA, before any allocation
  const int q0 = a.cu_q[seq], q_len = a.cu_q[seq + 1] - q0, k_len = a.cu_k[seq + 1] - a.cu_k[seq];
  const int off = k_len - q_len;             // position of the first query (negative: queries without a key)
  const int m0 = s_tile[1] * NP * p.tokens;
  // tokens of the two problems; B may be empty
  const int toks[2] = {min(p.tokens, q_len - m0), NP == 2 ? max(0, min(p.tokens, q_len - m0 - p.tokens)) : 0};
  const bool has_b = toks[1] > 0;
  const int pos0 = off + m0, last = pos0 + toks[0] + toks[1] - 1;     // positions of the CTA's first and last row
  // the walk: key tiles 0 .. nf - 1 (first tokens), then those from `start` on
  const int low0 = max(pos0 - a.window + 1, 0);                       // first key of the first window
  const int start = low0 / BN, nf = min((a.first + BN - 1) / BN, start);
  int nt[2];
  for (int x = 0; x < 2; ++x) {
    const int end = max(pos0 + x * p.tokens + toks[x] - 1, 0);
    nt[x] = toks[x] > 0 ? nf + end / BN - start + 1 : 0;
  }
  const int n = max(nt[0], nt[1]);           // A's windows end first
  auto key0 = [&](int j) -> int { return (j < nf ? j : j - nf + start) * BN; };

  if (warp == 2) umma::tmem_alloc(sb + L::OFF_BAR + L::NUM_BARS * 8, L::TCOLS);
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = *s_tmem;

  auto give_up = [&]() {
    *s_abort = 1;
    report(a.status, B200_ERR_TIMEOUT);
  };
#define WAIT_OR_ABORT(idx, parity)                                   \
  if (!umma::mbar_wait(bar(idx), (parity), s_abort)) {               \
    give_up();                                                       \
    break;                                                           \
  }

  int issued = 0;                            // key tiles that this producer has asked for
  if (warp < 2) {
    // =============================== TMA producers ===============================
    const bool is_k = warp == 0;
    if (is_k && lane == 0) {
      const int bytes = L::S * p.tokens * p.G * 128;
      umma::mbar_expect_tx(bar(L::Q_FULL), (has_b ? 2 : 1) * bytes);
      for (int x = 0; x < (has_b ? 2 : 1); ++x)
        for (int h = 0; h < L::S; ++h)
          umma::tma_load_3d(sb + x * L::Q_BYTES + h * Q_SLAB, &tm_q, h * 64, kvh * p.G, q0 + m0 + x * p.tokens, bar(L::Q_FULL));
    }
    const int boxes = BN / p.box;            // of a tile and slab; one lane each, at most 16
    const int part = lane % boxes, slab = lane / boxes;
    const bool mine = slab < L::S;
    const int32_t* table = a.bt + seq * a.bt_stride;
    const int64_t nothing = a.num_blocks * a.bs;                       // a row behind the pool: zeros
    const int full0 = is_k ? L::K_FULL : L::V_FULL, empty0 = is_k ? L::QK_DONE : L::PV_DONE;
    for (int j = 0; j < n; ++j) {
      const int st = j % NST;
      const int key = key0(j) + part * p.box;
      // does any row of the CTA see a key of this box?
      const bool seen = key <= last && (key < a.first || key + p.box > low0);
      int64_t row = nothing;
      if (mine && seen) {
        const int page = key / a.bs;
        const int64_t id = page < a.bt_width ? table[page] : -1;
        if (static_cast<uint64_t>(id) < static_cast<uint64_t>(a.num_blocks)) {
          row = id * a.bs + key % a.bs;
        } else {
          report(a.status, B200_ERR_BOUNDS);
          s_again = 1;
        }
      }
      if (j >= NST) {   // both problems must have released the tile that occupied this stage
        bool ok = true;
        for (int x = 0; x < 2; ++x)
          if (j - NST < nt[x]) ok = ok && umma::mbar_wait(bar(empty0 + 2 * st + x), ((j / NST) - 1) & 1, s_abort);
        if (!__all_sync(0xffffffffu, ok)) {
          give_up();
          break;
        }
      }
      if (lane == 0) umma::mbar_expect_tx(bar(full0 + st), L::K_BYTES);
      __syncwarp();
      if (mine)
        umma::tma_load_3d(sb + L::OFF_KV + st * L::STAGE + (is_k ? 0 : L::K_BYTES) + slab * K_SLAB + part * p.box * 128, is_k ? &tm_k : &tm_v,
                          slab * 64, kvh, static_cast<int>(row), bar(full0 + st));
      issued = j + 1;
    }
  } else if (warp < 4) {
    // =============================== MMA issuers ===============================
    const int x = warp - 2;
    if (x < NP && lane == 0 && nt[x] > 0) {
      const uint32_t idesc_qk = umma::instr_desc_bf16(BM, BN, false, false);
      const uint32_t idesc_pv = umma::instr_desc_bf16(BM, D, false, true);
      const int nx = nt[x];
      const uint64_t qd = umma::smem_desc(sb + x * L::Q_BYTES, 0, 1024);
      const uint64_t kd = umma::smem_desc(sb + L::OFF_KV, 0, 1024);
      const uint64_t vd = umma::smem_desc(sb + L::OFF_KV + L::K_BYTES, K_SLAB, 1024);
      const uint32_t tSx = tmem + x * (128 + D), tOx = tSx + 128;
      auto qk = [&](int st, int buf) {              // S[buf] = Q . K^T of the tile in stage st, contraction in steps of 16
        const uint32_t so = st * (L::STAGE >> 4);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          umma::mma_ss(tSx + buf * 64, umma::desc_advance(qd, ((ks >> 2) * Q_SLAB + (ks & 3) * 32) >> 4),
                       umma::desc_advance(kd, so + (((ks >> 2) * K_SLAB + (ks & 3) * 32) >> 4)), idesc_qk, ks > 0);
        umma::commit(bar(L::QK_DONE + x) + st * 16);
      };
      bool ok = umma::mbar_wait(bar(L::Q_FULL), 0, s_abort) && umma::mbar_wait(bar(L::K_FULL + 0), 0, s_abort);
      if (!ok) give_up();
      if (ok) {
        umma::fence_after_sync();
        qk(0, 0);
      }
      int st = 0, ph = 0;                      // stage and phase of tile j
      for (int j = 0; ok && j < nx; ++j) {
        int st1 = st + 1, ph1 = ph;
        if (st1 == NST) {
          st1 = 0;
          ph1 ^= 1;
        }
        if (j + 1 < nx) {
          WAIT_OR_ABORT(L::K_FULL + st1, ph1)
          umma::fence_after_sync();
          qk(st1, (j + 1) & 1);
        }
        WAIT_OR_ABORT(L::P_READY + 2 * x + (j & 1), (j >> 1) & 1)
        WAIT_OR_ABORT(L::V_FULL + st, ph)
        umma::fence_after_sync();
        const uint32_t so = st * (L::STAGE >> 4);
#pragma unroll
        for (int ks = 0; ks < BN / 16; ++ks)        // O += P[j & 1] . V_j : contraction over the 64 keys
          umma::mma_ts(tOx, tSx + (j & 1) * 64 + ks * 8, umma::desc_advance(vd, so + ks * (2048 >> 4)), idesc_pv, !(j == 0 && ks == 0));
        umma::commit(bar(L::PV_DONE + x) + st * 16);
        st = st1;
        ph = ph1;
      }
    }
  } else {
    // =============================== softmax / epilogue ===============================
    const int x = warp >= 8 ? 1 : 0;                        // problem A or B
    const int row = (warp & 3) * 32 + lane;                 // row of the problem == tensor-memory lane
    const uint32_t lane_sel = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS0 = tmem + x * (128 + D) + lane_sel, tOx = tS0 + 128;
    const int tok = row / p.G;
    const bool live = tok < toks[x];
    const int lim = pos0 + x * p.tokens + min(tok, max(toks[x] - 1, 0));     // position of the row's query: its last visible key
    const int low = lim - a.window + 1;                     // first key of its window (may be negative)
    const int nx = nt[x];
    const uint32_t qk_done = bar(L::QK_DONE + x), pv_done = bar(L::PV_DONE + x);
    const uint32_t my_turn = bar(L::TURN + (x == 0 ? 0 : 4) + (warp & 3));
    const uint32_t their_turn = bar(L::TURN + (x == 0 ? 4 : 0) + (warp & 3));
    // positions of the problem's first and last row: tiles that all rows see need no mask and no search
    const int pos_x = pos0 + x * p.tokens, last_x = pos_x + max(toks[x] - 1, 0);
    float m_ref = -INFINITY, l = 0.f;
    bool alive = true;
    int st = 0, ph = 0, stp = 0, php = 0;                   // stage and phase of tile j and of tile j - 1
    for (int j = 0; j < nx; ++j) {
      // tensor-memory loads / stores are warp-collective: the whole warp continues or stops together
      const uint32_t tSx = tS0 + (j & 1) * 64;                // score buffer of this tile
      const int n0 = key0(j);
      const bool masked = n0 + BN - 1 > pos_x || (n0 <= last_x - a.window && n0 + BN > a.first);
      if (masked) {                                           // uniform over the problem's warps
        // 16-byte pieces of the value tile with an exponent of ones
        const bool ok = umma::mbar_wait(bar(L::V_FULL + st), ph, s_abort);
        uint32_t odd = 0;
        const uint4* v = reinterpret_cast<const uint4*>(smem + L::OFF_KV + st * L::STAGE + L::K_BYTES) + row;
        auto look = [&](uint32_t w) { odd |= ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; };
#pragma unroll
        for (int i = 0; i < L::K_BYTES / 2048; ++i) {
          const uint4 w = v[i * 128];
          look(w.x), look(w.y), look(w.z), look(w.w);
        }
        if (ok && odd) s_again = 1;
      }
      if (!__all_sync(0xffffffffu, umma::mbar_wait(qk_done + st * 16, ph, s_abort))) {
        give_up();
        alive = false;
        break;
      }
      umma::fence_after_sync();
      // the 64 raw scores of the row stay in registers for both passes
      uint32_t ra[32], rb[32];
      umma::tmem_ld32(tSx, ra);
      umma::tmem_ld32_issue(tSx + 32, rb);
      float mx0 = -INFINITY, mx1 = -INFINITY;
      uint64_t seen = 0;                                      // bit e set: the row sees key n0 + e
      if (masked) {
        auto below = [](int k) -> uint64_t { return k >= 64 ? ~0ull : k <= 0 ? 0ull : (1ull << k) - 1ull; };     // keys n0 .. n0 + k - 1
        seen = below(lim - n0 + 1) & (~below(low - n0) | below(a.first - n0));
        const uint32_t m = static_cast<uint32_t>(seen);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(m & (1u << e))) ra[e] = 0xff800000u;          // -inf
      }
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        mx0 = fmaxf(mx0, __uint_as_float(ra[e]));
        mx1 = fmaxf(mx1, __uint_as_float(ra[e + 1]));
      }
      umma::tmem_ld32_wait(rb);
      if (masked) {
        const uint32_t m = static_cast<uint32_t>(seen >> 32);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!(m & (1u << e))) rb[e] = 0xff800000u;
      }
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        mx0 = fmaxf(mx0, __uint_as_float(rb[e]));
        mx1 = fmaxf(mx1, __uint_as_float(rb[e + 1]));
      }
      const float mx = fmaxf(mx0, mx1) * a.scale_log2;      // the scale is positive: it commutes with max
      // lazy rescale: move the reference maximum only when it grows by more than the threshold
      const bool need = mx > m_ref + kRescaleThreshold || (m_ref == -INFINITY && mx > -INFINITY);
      if (__any_sync(0xffffffffu, need)) {
        const float m_new = need ? mx : m_ref;
        const float alpha = (m_ref == -INFINITY) ? (need ? 0.f : 1.f) : fast_exp2(m_ref - m_new);
        l *= alpha;
        if (j > 0) {
          // O still receives P(j-1).V(j-1): the scores of this tile were issued ahead of that product
          if (!__all_sync(0xffffffffu, umma::mbar_wait(pv_done + stp * 16, php, s_abort))) {
            give_up();
            alive = false;
            break;
          }
          umma::fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t r[32];
            umma::tmem_ld32(tOx + c * 32, r);
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
            umma::tmem_st32(tOx + c * 32, r);
          }
          umma::tmem_wait_st();
        }
        m_ref = m_new;
      }
      // whose exponentials run now: A(j) follows B(j - 1), B(j) follows A(j) while A has tiles left
      if (x == 0 ? (has_b && j >= 1) : (j < nt[0])) {
        if (!__all_sync(0xffffffffu, umma::mbar_wait(my_turn, (x == 0 ? j - 1 : j) & 1, s_abort))) {
          give_up();
          alive = false;
          break;
        }
      }
      // P = 2^(s * scale - m_ref) as bf16 into the first 32 columns of S, row sum in fp32
      const float sub = m_ref == -INFINITY ? 0.f : m_ref;
      const uint64_t scale2 = umma::pack_f32x2(a.scale_log2, a.scale_log2);
      const uint64_t nsub2 = umma::pack_f32x2(-sub, -sub);
      uint64_t lsum2 = umma::pack_f32x2(0.f, 0.f);
      auto emit = [&](const uint32_t (&r)[32], int c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float s0, s1;
          umma::unpack_f32x2(
              umma::fma_f32x2(umma::pack_f32x2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), scale2, nsub2),
              s0, s1);
          const float p0 = fast_exp2(s0), p1 = fast_exp2(s1);   // 2^-inf = 0 for masked keys
          lsum2 = umma::add_f32x2(lsum2, umma::pack_f32x2(p0, p1));
          pk[e >> 1] = pack_bf16x2(p0, p1);
        }
        umma::tmem_st16(tSx + c * 16, pk);
      };
      emit(ra, 0);
      emit(rb, 1);
      umma::mbar_arrive(their_turn);
      {
        float la, lb;
        umma::unpack_f32x2(lsum2, la, lb);
        l += la + lb;
      }
      umma::tmem_wait_st();
      umma::fence_before_sync();
      umma::mbar_arrive(bar(L::P_READY + 2 * x + (j & 1)));
      stp = st;
      php = ph;
      if (++st == NST) {
        st = 0;
        ph ^= 1;
      }
    }
    if (nx > 0) {
      // the last product: stp / php are the stage and phase of tile nx - 1
      if (alive && __all_sync(0xffffffffu, umma::mbar_wait(pv_done + stp * 16, php, s_abort))) {
        umma::fence_after_sync();
        const float inv = l == 0.f ? 0.f : 1.f / l;          // 0: no key; a NaN stays one
        __nv_bfloat16* op = static_cast<__nv_bfloat16*>(a.out) +
                            (static_cast<int64_t>(q0 + m0 + x * p.tokens + tok) * a.Hq + kvh * p.G + row % p.G) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          umma::tmem_ld32(tOx + c * 32, r);     // warp-collective: every lane loads, live rows store
          if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 v;
              v.x = pack_bf16x2(__uint_as_float(r[e]) * inv, __uint_as_float(r[e + 1]) * inv);
              v.y = pack_bf16x2(__uint_as_float(r[e + 2]) * inv, __uint_as_float(r[e + 3]) * inv);
              v.z = pack_bf16x2(__uint_as_float(r[e + 4]) * inv, __uint_as_float(r[e + 5]) * inv);
              v.w = pack_bf16x2(__uint_as_float(r[e + 6]) * inv, __uint_as_float(r[e + 7]) * inv);
              *reinterpret_cast<uint4*>(op + c * 32 + e) = v;
            }
          }
        }
      } else if (alive) {
        give_up();
      }
    }
  }
#undef WAIT_OR_ABORT
  umma::fence_before_sync();
  __syncthreads();
  if (*s_abort) {                            // uniform: nobody sets it any more.  Copies and products under way end before the CTA does
    volatile int never = 0;
    if (warp < 2 && lane == 0) {
      for (int t = max(issued - NST, 0); t < issued; ++t)
        umma::mbar_wait(bar((warp == 0 ? L::K_FULL : L::V_FULL) + t % NST), (t / NST) & 1, &never);
      if (warp == 0) umma::mbar_wait(bar(L::Q_FULL), 0, &never);
    } else if (warp < 2 + NP && lane == 0) {
      umma::commit(bar(L::LEFT + warp - 2));
      umma::mbar_wait(bar(L::LEFT + warp - 2), 0, &never);
    }
    __syncthreads();
  }
  if (warp == 2) umma::tmem_dealloc(tmem, L::TCOLS);
  if (s_again && !*s_abort) {
    const int all = (toks[0] + toks[1]) * p.G;
    for (int r = warp; r < all; r += kThreads / 32)
      plain_row<D>(a, seq, static_cast<int64_t>(q0) + m0 + r / p.G, kvh * p.G + r % p.G, pos0 + r / p.G);
  }
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn tensor_map_encoder() {
  static EncodeFn fn = nullptr;                // racing threads store the same address
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeFn>(p);
    else
      cudaGetLastError();
  }
  return fn;
}

// [rows, heads, D] bf16 with a row stride in elements, as (d, head, row); a box is 64 columns of `box_heads` heads of `box_rows` rows.
bool make_map(CUtensorMap* m, const void* base, int64_t rows, int heads, int D, int64_t stride, int box_heads, int box_rows) {
  const EncodeFn encode = tensor_map_encoder();
  if (encode == nullptr || rows <= 0) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t steps[3] = {1, 1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NP>
int launch(const PromptArgs& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, int64_t ctas, cudaStream_t s) {
  using L = Lay<D, NP>;
  static_assert(L::SMEM <= 227 * 1024, "shared memory budget");
  static bool configured[64] = {};             // racing threads set the same attribute
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return B200_ERR_UNSUPPORTED;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(window_prefill_kernel<D, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM) != cudaSuccess) {
      cudaGetLastError();
      return B200_ERR_LAUNCH;
    }
    configured[dev] = true;
  }
  window_prefill_kernel<D, NP><<<static_cast<unsigned>(ctas), L::kThreads, L::SMEM, s>>>(p, tq, tk, tv);
  return launch_result();
}

}  // namespace

// B200_ERR_UNSUPPORTED: a shape, page size or alignment that the general kernel takes
int window_prefill_launch(const WindowArgs& a, int64_t total_q, cudaStream_t s) {
  const int G = a.Hq / a.Hkv;
  if (a.D != a.Dv || (a.D != 64 && a.D != 128) || G > BM || !(a.scale_log2 > 0.f)) return B200_ERR_UNSUPPORTED;
  if (a.bs < 8 || (a.bs % BN != 0 && BN % a.bs != 0)) return B200_ERR_UNSUPPORTED;
  const int64_t rows = a.num_blocks * a.bs;
  if (rows <= 0 || rows > 2147483647LL) return B200_ERR_UNSUPPORTED;       // coordinates of a copy are 32-bit
  if (!aligned16(a.q) || a.q_stride % 8 != 0 || (total_q > 1 && a.q_stride < static_cast<int64_t>(a.Hq) * a.D) || !aligned16(a.kc) || !aligned16(a.vc) || !aligned16(a.out)) return B200_ERR_UNSUPPORTED;
  PromptArgs p{a, G, BM / G, a.bs < BN ? a.bs : BN};
  const int problems = a.D == 64 ? 1 : 2;
  const int64_t ctas = (total_q / (problems * p.tokens) + a.num_seqs) * a.Hkv;     // tiles of all portions, the last of each perhaps short
  if (ctas > 2147483647LL || a.num_seqs > (1 << 20)) return B200_ERR_UNSUPPORTED;
  CUtensorMap tq, tk, tv;
  if (!make_map(&tq, a.q, total_q, a.Hq, a.D, a.q_stride, G, p.tokens) ||
      !make_map(&tk, a.kc, rows, a.Hkv, a.D, static_cast<int64_t>(a.Hkv) * a.D, 1, p.box) ||
      !make_map(&tv, a.vc, rows, a.Hkv, a.D, static_cast<int64_t>(a.Hkv) * a.D, 1, p.box))
    return B200_ERR_UNSUPPORTED;
  return a.D == 128 ? launch<128, 2>(p, tq, tk, tv, ctas, s) : launch<64, 1>(p, tq, tk, tv, ctas, s);
}

}  // namespace b200
