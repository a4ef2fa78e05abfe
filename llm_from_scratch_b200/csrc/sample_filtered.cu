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
// tokens, no more in the clustered kernel): sums of whole numbers do not depend on their order, so the borders fall at the same token whatever
// the launch looks like.
//
// A cluster of CTAs shares a row, whose logits stay in shared memory: a thread owns a run of neighbouring tokens.  Borders by value (top-k with
// ones as masses, top-p with the weights) are found with a histogram over the distance from the maximum, in steps of T / 128, and, if the
// border's bin holds more than a few tokens, over ever finer ranges of the logits' bits; what is left is sorted.  The border of the draw is
// found by sums over the threads' runs.  Many long rows go through sample_wide.cu.  Histograms hold a weight in three parts of 16 bits or more,
// each a 32-bit counter: shared memory adds 32 bits at a time.
//
// Bound by the reads for large rows in principle; in fact by latency, a chain of short steps with barriers between them: a row of 32,000 under
// all filters 16.5 us, 64 rows 25 us (means of 20; the first kernel, a CTA per row that read the logits for every byte of a border: 199 and 270).
// No unit is busy: 33 % of the issue slots at 64 rows.  Of the stalls there 19 % are for instructions, 17 % at barriers of the CTA, 14 % fixed
// latency, 9 % at fences; of one row's 49 % for instructions and 15 % at barriers.
#include <cooperative_groups.h>

#include "sampling.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 512;

// ---------------------------------------------------------------------------------------------
// rows that fit the shared memory of a cluster
// ---------------------------------------------------------------------------------------------
constexpr int kRowThreads = 512, kRowWarps = kRowThreads / 32;
constexpr int kBins = 4096, kOwnBins = kBins / kRowThreads;        // of the histogram of counts, two to a word
constexpr int kSteps = 2048, kOwnSteps = kSteps / kRowThreads;     // of the histograms of weights
constexpr int kList = 1024, kOwnList = kList / kRowThreads;        // tokens that are sorted at most
constexpr float kPerUnit = 128.f;                                   // bins per distance T from the maximum: 32 T and the last bin

struct alignas(16) RowShared {      // the logits lie behind it in 16-byte pieces
  double table[64];                  // 2^(i / 64)
  union {
    uint32_t hist[kSteps];           // counts: bins 2 i and 2 i + 1; weights: their bits 0 .. 15
    unsigned long long sorted_key[kList];
  };
  union {                            // never in use together
    uint32_t upper[2][kSteps];       // weights: their bits 16 .. 31 and from 32 on
    struct {
      unsigned long long key[kList], mass[kList];
    } list;
  };
  unsigned long long sorted_mass[kList];
  unsigned long long drawn[kRowThreads];   // kept weights of the list, by the thread that owns the token
  unsigned long long parts[2][8][3]; // of the CTAs of the cluster, in turns
  unsigned long long scan[kRowWarps][3];
  unsigned long long found_key, found_left;
  uint32_t list_size, lo_key, hi_key;
  uint32_t bin_lo, before_lo, bin_hi, upto_hi;       // the bracket, the tokens in front of it and up to its end
  int bin_k, left_k, count_k, step_at;
  float mass_k, spread_k;
};

static_assert(sizeof(RowShared) % 16 == 0, "the logits behind it are read in 16-byte pieces");

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

// What the kernel's parts know of a row.
struct Row {
  RowShared* sh;
  float* own;                        // the thread's logits
  RowShape shape;
  int rank, ranks, mine;             // place in the cluster, first token of the thread
  int S, turn;                       // turn of `parts`: two uses in a row do not meet, and a third comes behind a barrier
  float top, temperature, step, reach;
  double max, factor, floor_w;
  float edge;                        // kept: tokens above the border, and of those at it the ones up to a token
  int edge_token;

  __device__ __forceinline__ RowShared* other(int r) const { return cooperative_groups::this_cluster().map_shared_rank(sh, r); }
  __device__ __forceinline__ void sync() const {
    if (ranks > 1) cooperative_groups::this_cluster().sync();
    else __syncthreads();
  }
  __device__ __forceinline__ bool kept(float x, int i) const { return x > edge || (x == edge && i <= edge_token); }
  __device__ __forceinline__ double weight(float x) const { return weight_of(x, top, max, factor, reach, S, sh->table); }
  // Bin 0: the maximum; bin b: distances above (b - 1) / 128 and up to b / 128 times T; the last one: all beyond, whose weights round to 0.
  __device__ __forceinline__ int bin_of(float x) const {               // never falls as x falls
    return min_of(__float2int_ru((top - x) * step), kBins - 1);      // saturates
  }
  __device__ __forceinline__ void set_edge(unsigned long long c) {
    edge = key_value(static_cast<uint32_t>(c >> 32));
    edge_token = static_cast<int>(~static_cast<uint32_t>(c));
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {      // f(four logits, the first one's token) over the thread's run
#pragma unroll 1
    for (int i = 0; i < shape.run; i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(own + i);
      const float v[4] = {t.x, t.y, t.z, t.w};
      f(v, mine + i);
    }
  }
};

// A row's kernel runs through most of its code once, so a row that is alone waits for instructions above all (see the top).  Calls out of line do not help, as they put the row's values into memory (256 rows of 131,072: 435 us
// against 341).

// Running sum over the CTA's threads, inclusive, and the CTA's sum.
struct RunUp {
  unsigned long long upto, all;
};
__device__ __noinline__ RunUp run_up(RowShared& sh, unsigned long long v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_upto(v);
  __syncthreads();
  if (lane == 31) sh.scan[warp][0] = v;
  __syncthreads();
  const unsigned long long upto = warp_upto(lane < kRowWarps ? sh.scan[lane][0] : 0ull);
  const unsigned long long before = __shfl_sync(0xffffffffu, upto, warp > 0 ? warp - 1 : 0);
  return {warp > 0 ? v + before : v, __shfl_sync(0xffffffffu, upto, kRowWarps - 1)};
}

// What the tokens of a group of four add to a running mass: ones for kept tokens equal to `x0`; or kept weights above the floor; or ones for kept
// tokens of any weight above the floor.
enum Mass { kTies, kWeights, kAny };
__device__ __forceinline__ void mass_of_four(const Row& w, Mass kind, float x0, const float (&v)[4], int i, unsigned long long (&m)[4]) {
  bool in[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) in[j] = w.kept(v[j], i + j), m[j] = 0;
  if (!(in[0] || in[1] || in[2] || in[3])) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double g = w.weight(v[j]);
    const bool counts = in[j] && g >= w.floor_w;
    if (kind == kTies) m[j] = in[j] && v[j] == x0;
    else if (kind == kAny) m[j] = counts && static_cast<double>(v[j]) - w.max > -745.13 * w.temperature;
    else m[j] = counts ? rounded(g) : 0ull;
  }
}

// The first token at which the running mass reaches its target, by token: with `known` the thread's own mass is `sum`.  The target is `ties` for
// kTies, 1 for kAny, else u times the whole.  -1 in all threads of the cluster but one.
__device__ __forceinline__ int locate(Row& w, Mass kind, float x0, unsigned long long ties, float u, bool known, unsigned long long sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  RowShared& sh = *w.sh;
  if (!known) {
    sum = 0;
    w.each([&](const float (&v)[4], int i) {
      unsigned long long m[4];
      mass_of_four(w, kind, x0, v, i, m);
      sum += m[0] + m[1] + (m[2] + m[3]);
    });
  }
  const RunUp run_sum = run_up(sh, sum);
  unsigned long long upto = run_sum.upto, total = run_sum.all;
  if (w.ranks > 1) {
    if (threadIdx.x < w.ranks) w.other(threadIdx.x)->parts[w.turn][w.rank][0] = total;
    w.sync();
    const unsigned long long part = lane < w.ranks ? sh.parts[w.turn][lane][0] : 0ull;
    upto += warp_total(lane < w.rank ? part : 0ull);
    total = warp_total(part);
    w.turn ^= 1;
  }
  unsigned long long target = kind == kTies ? ties : kind == kAny ? 1ull
      : static_cast<unsigned long long>(static_cast<double>(u) * static_cast<double>(total)) + 1;
  if (target > total) target = total;
  const unsigned owner = __ballot_sync(0xffffffffu, upto >= target && upto - sum < target);
  if (owner == 0) return -1;
  // the owner's run, a group of four per lane
  const int src = __ffs(owner) - 1;
  unsigned long long left = __shfl_sync(0xffffffffu, target - (upto - sum), src);
  const float* run = w.own + (src - lane) * w.shape.stride;
  const int first = w.mine + (src - lane) * w.shape.run;
#pragma unroll 1
  for (int base = 0; base < w.shape.run; base += 128) {
    const int i = base + lane * 4;
    unsigned long long m[4] = {0, 0, 0, 0};
    if (i < w.shape.run) {
      const float4 t = *reinterpret_cast<const float4*>(run + i);
      const float v[4] = {t.x, t.y, t.z, t.w};
      mass_of_four(w, kind, x0, v, first + i, m);
    }
    const unsigned long long four = m[0] + m[1] + (m[2] + m[3]), up = warp_upto(four);
    const bool here = up >= left && up - four < left;
    if (__any_sync(0xffffffffu, here)) {
      int j = 0;
      unsigned long long rest = left - (up - four);
#pragma unroll
      for (int c = 0; c < 3; ++c)
        if (j == c && rest > m[c]) rest -= m[c], ++j;
      return here ? first + i + j : -1;
    }
    left -= __shfl_sync(0xffffffffu, up, 31);
  }
  return -1;
}

// The border by value in any row: the edge becomes the first kept token of the bins from .. to, from the front of the order, at which the running
// mass (ones with `ones`, else the weights) reaches `target`.  Histograms of the masses over fine steps of these bins, then over ever finer
// ranges of the logits' bits, until the border's place fits the list.
__device__ __forceinline__ void cut(Row& w, const bool ones, unsigned long long target, const int from_bin, const int to_bin) {
  const int tid = threadIdx.x, lane = tid & 31;
  RowShared& sh = *w.sh;
  int level = 0, shift = 0;
  uint32_t lo_key = 0, hi_key = 0xffffffffu;
  const float origin = from_bin - 1.f, scale = static_cast<float>(kSteps - 1) / (to_bin - from_bin + 1);
  auto place = [&](float x, int i) -> int {              // at this level; -1: not a candidate
    int s;
    if (level == 0) {
      const int b = w.bin_of(x);
      s = b < from_bin || b > to_bin ? -1 : max_of(0, min_of(kSteps - 1, __float2int_ru(((w.top - x) * w.step - origin) * scale)));
    } else {
      const uint32_t key = order_key(x);
      s = key < lo_key || key > hi_key ? -1 : static_cast<int>((hi_key - key) >> shift);
    }
    return s >= 0 && w.kept(x, i) ? s : -1;
  };
  auto mass_of = [&](float x) -> unsigned long long { return ones ? 1ull : rounded(w.weight(x)); };
  for (;;) {
    w.sync();                                            // the list of an earlier use has been read
    for (int i = tid; i < kSteps; i += kRowThreads) sh.hist[i] = sh.upper[0][i] = sh.upper[1][i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < w.shape.run; ++i) {
      const float x = w.own[i];
      const int s = place(x, w.mine + i);
      if (s < 0) continue;
      const unsigned long long m = mass_of(x);
      const uint32_t m0 = m & 0xffff, m1 = (m >> 16) & 0xffff, m2 = static_cast<uint32_t>(m >> 32);
      if (m0) atomicAdd(&sh.hist[s], m0);
      if (m1) atomicAdd(&sh.upper[0][s], m1);
      if (m2) atomicAdd(&sh.upper[1][s], m2);
    }
    w.sync();
    unsigned long long h[kOwnSteps], sum = 0;
#pragma unroll
    for (int j = 0; j < kOwnSteps; ++j) {
      h[j] = 0;
#pragma unroll 1
      for (int r = 0; r < w.ranks; ++r) {
        const RowShared* from = w.other(r);
        const int at = tid * kOwnSteps + j;
        h[j] += from->hist[at] + (static_cast<unsigned long long>(from->upper[0][at]) << 16) + (static_cast<unsigned long long>(from->upper[1][at]) << 32);
      }
      sum += h[j];
    }
    const unsigned long long upto = run_up(sh, sum).upto;
    if (upto >= target && upto - sum < target) {         // one thread of every CTA
      unsigned long long left = target - (upto - sum);
      int s = tid * kOwnSteps;
#pragma unroll
      for (int j = 0; j < kOwnSteps - 1; ++j) {
        if (left <= h[j]) break;
        left -= h[j];
        ++s;
      }
      sh.step_at = s;
      sh.found_left = left;
      sh.list_size = 0;
      sh.lo_key = 0xffffffffu;
      sh.hi_key = 0;
    }
    w.sync();                                            // the histograms have been read, and the list is empty
    const int step_at = sh.step_at;
    target = sh.found_left;
    RowShared* lead = w.other(0);
    uint32_t least = 0xffffffffu, most = 0;
#pragma unroll 1
    for (int i = 0; i < w.shape.run; ++i) {
      const float x = w.own[i];
      if (place(x, w.mine + i) != step_at) continue;
      const unsigned long long m = mass_of(x);
      if (m == 0) continue;
      const uint32_t key = order_key(x), at = atomicAdd(&lead->list_size, 1u);
      least = min(least, key);
      most = key > most ? key : most;
      if (at < kList) lead->list.key[at] = composite(x, w.mine + i), lead->list.mass[at] = m;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0 && most != 0) atomicMin(&lead->lo_key, least), atomicMax(&lead->hi_key, most);
    w.sync();
    const int size = static_cast<int>(lead->list_size);
    const uint32_t least_all = lead->lo_key, most_all = lead->hi_key;
    if (size <= kList) {
      if (w.rank == 0) {
        for (int i = tid; i < size; i += kRowThreads) sh.sorted_key[i] = sh.list.key[i], sh.sorted_mass[i] = sh.list.mass[i];
        sort_by_key<kRowThreads>(sh.sorted_key, sh.sorted_mass, size);
        unsigned long long m[kOwnList], own_sum = 0;
#pragma unroll
        for (int j = 0; j < kOwnList; ++j) {
          const int i = tid * kOwnList + j;
          m[j] = i < size ? sh.sorted_mass[i] : 0;
          own_sum += m[j];
        }
        unsigned long long up = run_up(sh, own_sum).upto - own_sum;
#pragma unroll
        for (int j = 0; j < kOwnList; ++j) {
          if (up < target && up + m[j] >= target)
            for (int r = 0; r < w.ranks; ++r) w.other(r)->found_key = sh.sorted_key[tid * kOwnList + j];
          up += m[j];
        }
      }
      w.sync();
      w.set_edge(sh.found_key);
      return;
    }
    if (least_all == most_all) {                         // equal logits: so many of them, by token
      const float x0 = key_value(least_all);
      const unsigned long long one = mass_of(x0);
      const int token = locate(w, kTies, x0, (target + one - 1) / one, 0.f, false, 0);
      if (token >= 0)
        for (int r = 0; r < w.ranks; ++r) w.other(r)->found_key = static_cast<uint32_t>(~token);
      w.sync();
      w.edge = x0;
      w.edge_token = static_cast<int>(~static_cast<uint32_t>(sh.found_key));
      return;
    }
    lo_key = least_all, hi_key = most_all;               // logits of one place: a range of bits
    const int width = 32 - __clz(hi_key - lo_key);
    shift = width > 11 ? width - 11 : 0;
    ++level;
  }
}

// Three sums over the cluster, the same in all threads.
struct Sums {
  unsigned long long v[3];
};
__device__ __forceinline__ Sums combine(Row& w, Sums s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  RowShared& sh = *w.sh;
#pragma unroll 1
  for (int stage = 0; stage < 3; ++stage) {
#pragma unroll
    for (int c = 0; c < 3; ++c) s.v[c] = warp_total(s.v[c]);
    if (stage == 0) {
      __syncthreads();
      if (lane == 0)
#pragma unroll
        for (int c = 0; c < 3; ++c) sh.scan[warp][c] = s.v[c];
      __syncthreads();
#pragma unroll
      for (int c = 0; c < 3; ++c) s.v[c] = lane < kRowWarps ? sh.scan[lane][c] : 0ull;
    } else if (stage == 1) {
      if (w.ranks == 1) break;
      if (threadIdx.x < w.ranks)
#pragma unroll
        for (int c = 0; c < 3; ++c) w.other(threadIdx.x)->parts[w.turn][w.rank][c] = s.v[c];
      w.sync();
#pragma unroll
      for (int c = 0; c < 3; ++c) s.v[c] = lane < w.ranks ? sh.parts[w.turn][lane][c] : 0ull;
      w.turn ^= 1;
    }
  }
  return s;
}
__device__ __forceinline__ uint32_t combine_max(Row& w, uint32_t v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  RowShared& sh = *w.sh;
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if (lane == 0) sh.scan[warp][0] = v;
  __syncthreads();
  v = __reduce_max_sync(0xffffffffu, lane < kRowWarps ? static_cast<uint32_t>(sh.scan[lane][0]) : 0u);
  if (w.ranks > 1) {
    if (threadIdx.x < w.ranks) w.other(threadIdx.x)->parts[w.turn][w.rank][0] = v;
    w.sync();
    v = __reduce_max_sync(0xffffffffu, lane < w.ranks ? static_cast<uint32_t>(sh.parts[w.turn][lane][0]) : 0u);
    w.turn ^= 1;
  }
  return v;
}

// Sums without a list: kept weights in front of the bins lo .. hi, behind them and in them.
__device__ __forceinline__ Sums sum_weights(Row& w, const float y_lo, const float y_hi) {
  Sums s = {{0, 0, 0}};
  w.each([&](const float (&v)[4], int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float y = (w.top - v[j]) * w.step;
      if (w.kept(v[j], i + j)) s.v[y <= y_lo ? 0 : y <= y_hi ? 2 : 1] += rounded(w.weight(v[j]));
    }
  });
  return combine(w, s);
}

// The first of the highest logits, in all threads.
__device__ __forceinline__ int first_highest(Row& w, int vocab) {
  uint32_t first = 0;
  w.each([&](const float (&v)[4], int i) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v[j] == w.top && i + j < vocab) first = first > ~static_cast<uint32_t>(i + j) ? first : ~static_cast<uint32_t>(i + j);
  });
  return static_cast<int>(~combine_max(w, first));
}

template <typename T>
__device__ __forceinline__ void sample_row(const SampleArgs& a, const int row, uint8_t* smem) {
  RowShared& sh = *reinterpret_cast<RowShared*>(smem);
  float* data = reinterpret_cast<float*>(smem + sizeof(RowShared));
  // The other CTAs' shared memory may be written once they have all started: they say so here, the wait is in front of the first write.  No data
  // passes with it, so it orders nothing (relaxed).
  asm volatile("barrier.cluster.arrive.relaxed;");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.vocab;
  Row w;
  w.sh = &sh;
  w.rank = cooperative_groups::this_cluster().block_rank(), w.ranks = cooperative_groups::this_cluster().num_blocks();
  const int rank = w.rank, ranks = w.ranks;
  w.shape = row_shape(V, ranks);
  const RowShape shape = w.shape;
  const int begin = rank * shape.slice;
  w.mine = begin + tid * shape.run, w.own = data + tid * shape.stride;
  w.S = a.bits, w.turn = 0;
  w.edge = -INFINITY, w.edge_token = 0x7fffffff;
  w.temperature = fminf(a.temperatures[row], 1e30f);     // beyond that all finite logits weigh the same
  const float p = a.top_p ? a.top_p[row] : 1.f, u = fminf(a.uniforms[row], 1.f);
  int k = a.top_k ? a.top_k[row] : 0;
  const float floor_w = a.min_p ? a.min_p[row] : 0.f;
  w.floor_w = (floor_w > 1.f ? 1.0 : floor_w > 0.f ? static_cast<double>(floor_w) : 0.0) * static_cast<double>(1ull << a.bits);

  // ---- the CTA's logits; NaN and what lies behind the row as -inf
  float top = -INFINITY;
  {
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride + begin;
    const int n = min(shape.slice, V - begin);           // may be negative
    auto clean = [](float v) { return v != v ? -INFINITY : v; };
    const int all = kRowThreads * shape.run;
    constexpr int W = 16 / sizeof(T), STEP = kRowThreads * W;
    const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0;
    // owner and place of a group of four, kept up from trip to trip instead of divided out
    int owner = (tid * W) / shape.run, at = (tid * W) % shape.run;
    const int more = STEP / shape.run, rest = STEP % shape.run;
    auto put = [&](const float (&v)[W]) {
#pragma unroll
      for (int j = 0; j < W; ++j) top = fmaxf(top, v[j]);
      int o = owner, c = at;
#pragma unroll
      for (int j = 0; j < W; j += 4) {
        if (o < kRowThreads) *reinterpret_cast<float4*>(data + o * shape.stride + c) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        c += 4;
        if (c == shape.run) c = 0, ++o;
      }
      owner += more, at += rest;
      if (at >= shape.run) at -= shape.run, ++owner;
    };
    int i = tid * W;
    if (wide) {
      constexpr int AHEAD = 4;                           // loads in flight
#pragma unroll 1
      for (; i + (AHEAD - 1) * STEP + W <= n; i += AHEAD * STEP) {
        uint4 raw[AHEAD];
#pragma unroll
        for (int c = 0; c < AHEAD; ++c) raw[c] = __ldg(reinterpret_cast<const uint4*>(x + i + c * STEP));
#pragma unroll
        for (int c = 0; c < AHEAD; ++c) {
          const T* e = reinterpret_cast<const T*>(&raw[c]);
          float v[W];
#pragma unroll
          for (int j = 0; j < W; ++j) v[j] = clean(to_float<T>(e[j]));
          put(v);
        }
      }
    }
#pragma unroll 1
    for (; i < all; i += STEP) {
      float v[W];
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = i + j < n ? clean(to_float<T>(x[i + j])) : -INFINITY;
      put(v);
    }
    if (tid < 64) sh.table[tid] = kTable[tid];
    sh.drawn[tid] = 0;
    for (int j = tid; j < kSteps; j += kRowThreads) sh.hist[j] = 0;
    if (tid == 0) sh.list_size = 0;
  }
  asm volatile("barrier.cluster.wait;" ::: "memory");
  w.top = key_value(combine_max(w, order_key(top)));
  if (!(w.temperature > 0.f) || w.top == -INFINITY) {
    const int token = first_highest(w, V);
    if (rank == 0 && tid == 0) a.out[row] = token;
    return;
  }
  if (w.top == INFINITY) {                               // infinite logits share all the weight
    for (int i = 0; i < shape.run; ++i) w.own[i] = w.own[i] == INFINITY ? 0.f : -INFINITY;
    w.top = 0.f;
  }
  w.max = w.top, w.factor = 64.0 * 1.4426950408889634 / w.temperature;
  w.reach = 660.f * w.temperature;                       // distance beyond which a weight is 0
  w.step = fminf(kPerUnit / w.temperature, 3e38f);
  // in registers, unlike what calls see of the row
  const float* const own = data + tid * shape.stride;
  const float step = w.step, reach = w.reach;
  const double max = w.max, factor = w.factor, least_weight = w.floor_w;
  top = w.top;
  const int S = a.bits;

  if (k >= V || k < 0) k = 0;
  const bool nucleus = p < 1.f;
  bool summed = false;                                   // the thread's kept weights are known without another pass
  unsigned long long own_kept = 0;
  if (k > 0 || nucleus) {
    // ---- both borders at once.  A histogram of counts says in which bin the k-th token lies, and, as a bin's weights are alike to 0.8 %, between
    // which bins the nucleus ends; one pass over the weights then sums what lies outside these bins exactly and lists their tokens.
    const int last = k > 0 ? kBins : kBins - 1;          // what is in the last bin has no weight
#pragma unroll 2
    for (int i = 0; i < shape.run; i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(own + i);
      const float v[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b = min_of(__float2int_ru((top - v[j]) * step), kBins - 1);
        if (b < last) atomicAdd(&sh.hist[b >> 1], b & 1 ? 0x10000u : 1u);
      }
    }
    if (tid == 0) {
      sh.bin_k = kBins, sh.left_k = sh.count_k = 0;
      sh.bin_lo = sh.bin_hi = kBins;
      sh.before_lo = sh.upto_hi = 0xffffffffu;
    }
    w.sync();
    // a CTA adds up a share of the bins, a thread a run of up to four words of it, two bins each.  (Where every CTA adds up all bins and
    // finds the borders for itself, two barriers of the cluster less, a row of 32,000 takes 19.9 us against 16.5, 64 rows 25.7 against 25.3.)
    const int share = kBins / 2 / ranks, words = max_of(share / kRowThreads, 1), word0 = rank * share + tid * words;
    const bool busy = tid * words < share;
    uint32_t* own_count = &sh.upper[0][0] + tid * words * 2;       // of the share's bins
    int counted = 0;
    float mass = 0.f, spread = 0.f;                      // by where the bins' tokens lie on the average, and the variance of that
    const BinPlaces<sizeof(T) == 2> places(top, step);
    auto weight_of_bin = [&](int b, float& variance) {
      variance = 0.f;                                    // of the last bin, which weighs nothing
      const float g = b < kBins - 1 ? fast_exp2(-1.4426950408889634f / kPerUnit * places.of(b, variance)) : 0.f;
      variance *= g * g * (1.f / (kPerUnit * kPerUnit));
      return g;
    };
#pragma unroll 1
    for (int c = 0; c < words && busy; ++c) {
      uint32_t y[8], lo = 0, hi = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) y[r] = r < ranks ? (ranks > 1 ? w.other(r) : &sh)->hist[word0 + c] : 0u;
#pragma unroll
      for (int r = 0; r < 8; ++r) lo += y[r] & 0xffff, hi += y[r] >> 16;
      own_count[2 * c] = lo, own_count[2 * c + 1] = hi;
      counted += lo + hi;
      const int b = 2 * (word0 + c);
      float v0, v1;
      const float g0 = weight_of_bin(b, v0), g1 = weight_of_bin(b + 1, v1);
      mass += lo * g0 + hi * g1;
      spread += lo * v0 + hi * v1;
    }
    // running sums over the cluster's threads, inclusive, and the whole
    int upto = warp_upto(counted);
    float mass_up = warp_upto(mass), spread_up = warp_upto(spread), mass_all = 0.f, spread_all = 0.f;
    __syncthreads();
    if (lane == 31) sh.scan[warp][0] = upto, sh.scan[warp][1] = __float_as_uint(mass_up), sh.scan[warp][2] = __float_as_uint(spread_up);
    __syncthreads();
    int count_all = 0;
#pragma unroll 4
    for (int c = 0; c < kRowWarps; ++c) {
      const int n = static_cast<int>(sh.scan[c][0]);
      const float m = __uint_as_float(static_cast<uint32_t>(sh.scan[c][1])), e = __uint_as_float(static_cast<uint32_t>(sh.scan[c][2]));
      if (c < warp) upto += n, mass_up += m, spread_up += e;
      count_all += n, mass_all += m, spread_all += e;
    }
    if (ranks > 1) {
      if (tid < ranks) {
        unsigned long long* to = w.other(tid)->parts[w.turn][rank];
        to[0] = count_all, to[1] = __float_as_uint(mass_all), to[2] = __float_as_uint(spread_all);
      }
      w.sync();
      mass_all = spread_all = 0.f;
#pragma unroll 1
      for (int r = 0; r < ranks; ++r) {
        const float m = __uint_as_float(static_cast<uint32_t>(sh.parts[w.turn][r][1])), e = __uint_as_float(static_cast<uint32_t>(sh.parts[w.turn][r][2]));
        if (r < rank) upto += static_cast<int>(sh.parts[w.turn][r][0]), mass_up += m, spread_up += e;
        mass_all += m, spread_all += e;
      }
      w.turn ^= 1;
    }
    int bin_k = kBins, left_k = 0, count_k = 0;          // bin of the k-th token, its place there, tokens there
    if (k > 0) {
      if (busy && upto >= k && upto - counted < k) {     // one thread of the cluster
        int n = upto - counted;
        float m = mass_up - mass, e = spread_up - spread;
#pragma unroll 1
        for (int c = 0; c < 2 * words; ++c) {
          const int b = 2 * word0 + c, here = own_count[c];
          float variance;
          const float g = weight_of_bin(b, variance);
          if (n + here >= k) {
#pragma unroll 1
            for (int r = 0; r < ranks; ++r) {
              RowShared* to = w.other(r);
              to->bin_k = b, to->left_k = k - n, to->count_k = here;
              to->mass_k = m + (k - n) * g, to->spread_k = e + (k - n) * variance;
            }
            break;
          }
          n += here;
          m += here * g, e += here * variance;
        }
      }
      w.sync();
      bin_k = sh.bin_k, left_k = sh.left_k, count_k = sh.count_k;
      mass_all = sh.mass_k, spread_all = sh.spread_k;
    }
    int bin_lo = kBins, bin_hi = kBins - 1;              // bins among which the nucleus ends
    int listed = count_k;                                // tokens of the list
    if (nucleus) {
      // One standard deviation of the sum in front, and one of p times the whole, which in part is the same sum: with the bins' own widths a border
      // is seldom outside.  Such a row, and one whose bracket has more tokens than the list takes, finds it by the histograms of weights.  Means of
      // 20 calls (us) at 3.5, 2, 1.2, 1 and 0.6 deviations: 64 rows of 32,000, all filters, 28.4, 26.4, 25.2, 24.9, 24.5; 256 with top-p 68, 63, 60, 60,
      // 58.  64 of bf16 with top-p: 25.3, 25.3, 25.2, 25.3, 24.8 (with the bins' middles and half a bin for each token as the bound: 48 .. 65)
      auto off = [&](float m, float e) {
        float root;
        asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root) : "f"(e));
        return root + 1e-5f * m;
      };
      const float goal = p * mass_all, wide = p * off(mass_all, spread_all);
      if (busy && mass_up + off(mass_up, spread_up) + wide >= goal && !(mass_up - mass - off(mass_up - mass, spread_up - spread) - wide >= goal)) {
        // two threads may both see the border between them: the lower bin counts, which has the fewer tokens too
        int n = upto - counted;
        float m = mass_up - mass, e = spread_up - spread;
        bool lo = m + off(m, e) + wide >= goal, hi = m - off(m, e) - wide >= goal;
#pragma unroll 1
        for (int c = 0; c < 2 * words; ++c) {
          const int b = 2 * word0 + c, here = own_count[c];
          float variance;
          const float g = weight_of_bin(b, variance);
          m += here * g, e += here * variance;
          const bool lo1 = m + off(m, e) + wide >= goal, hi1 = m - off(m, e) - wide >= goal;
          const bool new_lo = lo1 && !lo, new_hi = hi1 && !hi;
          if (new_lo || new_hi)
#pragma unroll 1
            for (int r = 0; r < ranks; ++r) {
              RowShared* to = w.other(r);
              if (new_lo) atomicMin(&to->bin_lo, static_cast<uint32_t>(b)), atomicMin(&to->before_lo, static_cast<uint32_t>(n));
              if (new_hi) atomicMin(&to->bin_hi, static_cast<uint32_t>(b)), atomicMin(&to->upto_hi, static_cast<uint32_t>(n + here));
            }
          n += here;
          lo = lo1, hi = hi1;
        }
      }
      w.sync();
      bin_lo = static_cast<int>(sh.bin_lo), bin_hi = static_cast<int>(sh.bin_hi);
      const int before_lo = static_cast<int>(sh.before_lo), upto_hi = static_cast<int>(sh.upto_hi);
      if (bin_lo == kBins || bin_hi == kBins || bin_hi < bin_lo) {
        listed = bin_lo <= bin_k && bin_k < kBins ? k - left_k + count_k - before_lo : kList + 1;     // up to the k-th token's bin, or too many
        bin_hi = min_of(bin_k, kBins - 2);
      } else if (bin_hi >= bin_k) {
        listed = k - left_k + count_k - before_lo;
        bin_hi = min_of(bin_k, kBins - 2);
      } else {
        listed += upto_hi - before_lo;
      }
    }
    bool done = listed <= kList && (bin_lo <= bin_hi || !nucleus);
    RowShared* lead = w.other(0);
    // a bin's tokens are told by ceil(y) <= b where y <= b
    const float y_lo = bin_lo - 1.f, y_hi = bin_hi, y_k = bin_k < kBins ? bin_k - 1.f : INFINITY, y_k1 = bin_k < kBins - 1 ? bin_k : INFINITY;
    Sums sums = {{0, 0, 0}};                             // weights in front of the list's bins, and behind them up to the k-th token's
    if (done) {
      // All weights are added up; the tokens up to the list's bins, which are few in most rows, are looked at more closely.  32 tokens at a time:
      // those for the list are noted in a mask and put there behind the 32.
      unsigned long long all = 0, front = 0, list = 0;
      const float y_near = nucleus ? fmaxf(y_hi, y_k1 < INFINITY ? y_k1 : 0.f) : y_k1;          // the last of them
#pragma unroll 1
      for (int base = 0; base < shape.run; base += 32) {
        uint32_t noted = 0;
        const int end = min_of(base + 32, shape.run);
#pragma unroll 1
        for (int i = base; i < end; i += 4) {
          const float4 t = *reinterpret_cast<const float4*>(own + i);
          const float v[4] = {t.x, t.y, t.z, t.w};
          float y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = (top - v[j]) * step;
          const bool near = fminf(fminf(y[0], y[1]), fminf(y[2], y[3])) <= y_near;
          if (!near && !nucleus) continue;
          double g[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) g[j] = weight_of(v[j], top, max, factor, reach, S, sh.table);
          unsigned long long m[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) m[j] = rounded(y[j] <= y_k1 ? g[j] : 0.0);
          all += (m[0] + m[1]) + (m[2] + m[3]);
          if (near) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bool before = nucleus ? y[j] <= y_lo : y[j] <= y_k;
              const bool in = !before && ((nucleus && y[j] <= y_hi) || (y[j] > y_k && y[j] <= y_k1));
              if (before) front += m[j];
              if (before && g[j] >= least_weight) own_kept += m[j];
              if (in) list += m[j];
              noted |= static_cast<uint32_t>(in) << (i - base + j);
            }
          }
        }
        if (__any_sync(0xffffffffu, noted)) {            // one addition to the list's size per warp
          const int n = __popc(noted), upto_lane = warp_upto(n);
          uint32_t at = 0;
          if (lane == 31) at = atomicAdd(&lead->list_size, static_cast<uint32_t>(upto_lane));
          at = __shfl_sync(0xffffffffu, at, 31) + upto_lane - n;
#pragma unroll 1
          for (; noted; noted &= noted - 1, ++at) {
            const int i = base + __ffs(noted) - 1;
            if (at < kList)
              lead->list.key[at] = composite(own[i], begin + tid * shape.run + i),
              lead->list.mass[at] = rounded(weight_of(own[i], top, max, factor, reach, S, sh.table));
          }
        }
      }
      sums.v[0] = front, sums.v[1] = all - front - list;
      sums = combine(w, sums);
      done = static_cast<int>(lead->list_size) <= kList;
    }
    auto goal_of = [&](unsigned long long sum) -> unsigned long long {
      const double want = ceil(static_cast<double>(p) * static_cast<double>(sum));
      return want > 1.0 ? static_cast<unsigned long long>(want) : 1ull;
    };
    if (done) {
      const int size = static_cast<int>(lead->list_size);
      // every CTA sorts a copy of the list
#pragma unroll 1
      for (int i = tid; i < size; i += kRowThreads) sh.sorted_key[i] = lead->list.key[i], sh.sorted_mass[i] = lead->list.mass[i];
      sort_by_key<kRowThreads>(sh.sorted_key, sh.sorted_mass, size);
      // of the list in order: the k-th token's bin keeps its first left_k
      unsigned long long g[kOwnList], key[kOwnList];
      bool at_k[kOwnList];
      int before_k = 0;
#pragma unroll
      for (int j = 0; j < kOwnList; ++j) {
        const int i = tid * kOwnList + j;
        key[j] = i < size ? sh.sorted_key[i] : 0;
        g[j] = i < size ? sh.sorted_mass[i] : 0;
        at_k[j] = i < size && w.bin_of(key_value(static_cast<uint32_t>(key[j] >> 32))) == bin_k;
        before_k += at_k[j];
      }
      int place = 0;
      if (k > 0) {
        int upk = static_cast<int>(run_up(sh, before_k).upto) - before_k;
#pragma unroll
        for (int j = 0; j < kOwnList; ++j) {
          upk += at_k[j];
          if (at_k[j] && upk == left_k) sh.found_left = tid * kOwnList + j;   // place of the k-th token in the list
          if (at_k[j] && upk > left_k) g[j] = 0;
        }
        __syncthreads();
        place = static_cast<int>(sh.found_left);
      }
      if (nucleus) {
        unsigned long long sum = 0;
#pragma unroll
        for (int j = 0; j < kOwnList; ++j) sum += g[j];
        const RunUp run_sum = run_up(sh, sum);
        const unsigned long long front = sums.v[0], target = goal_of(front + sums.v[1] + run_sum.all);
        const bool gap = sums.v[1] != 0;                 // weights between the bins and the k-th token's
        // the border lies behind the front and among the list's first bins, or the bins were wrong
        if (tid == 0) sh.found_key = kList;
        __syncthreads();
        unsigned long long up = front + run_sum.upto - sum;
#pragma unroll
        for (int j = 0; j < kOwnList; ++j) {
          if (up < target && up + g[j] >= target && (!gap || w.bin_of(key_value(static_cast<uint32_t>(key[j] >> 32))) <= bin_hi))
            sh.found_key = tid * kOwnList + j;
          up += g[j];
        }
        __syncthreads();
        place = static_cast<int>(sh.found_key);
        done = place < kList && front < target;
      }
      if (done) {
        w.set_edge(sh.sorted_key[place]);
        // what is kept of the list, to its owners
#pragma unroll 1
        for (int i = tid; i <= place; i += kRowThreads) {
          const int token = static_cast<int>(~static_cast<uint32_t>(sh.sorted_key[i])) - begin;
          const unsigned long long m = sh.sorted_mass[i];
          if (token >= 0 && token < shape.slice && m > 0 && w.weight(key_value(static_cast<uint32_t>(sh.sorted_key[i] >> 32))) >= w.floor_w)
            atomicAdd(&sh.drawn[token / shape.run], m);
        }
        __syncthreads();
        own_kept += sh.drawn[tid];
        summed = true;
      }
    }
    if (!done) {
      // too many tokens in the list's bins, or the wrong bins: top-k first, then the nucleus of what it keeps
#pragma unroll 1
      for (int stage = k > 0 ? 0 : 1; stage < (nucleus ? 2 : 1); ++stage) {
        unsigned long long target = left_k;
        int from = bin_k, to = bin_k;
        if (stage == 1) {
          sums = sum_weights(w, y_lo, y_hi);
          target = goal_of(sums.v[0] + sums.v[1] + sums.v[2]);
          const bool inside = sums.v[0] < target && target <= sums.v[0] + sums.v[2];
          if (inside) target -= sums.v[0];
          from = inside ? bin_lo : 0, to = inside ? bin_hi : kBins - 1;
        }
        cut(w, stage == 0, target, from, to);
      }
    }
  }
  const bool any = !(u > 0.f);                           // the first kept token of any weight, however small
  const int token = locate(w, any ? kAny : kWeights, 0.f, 0, u, summed && !any, own_kept);
  if (token >= 0) a.out[row] = token;
}

// A cluster per row; or, with a list of rows (their number first), a few clusters that walk it.
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2) sample_row_kernel(const SampleArgs a, const int32_t* list) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int ranks = cooperative_groups::this_cluster().num_blocks(), first = blockIdx.x / ranks;
  if (list == nullptr) return sample_row<T>(a, first, smem);
  for (int i = first; i < list[0]; i += gridDim.x / ranks) {
    sample_row<T>(a, list[1 + i], smem);
    cooperative_groups::this_cluster().sync();           // the row's shared memory is used again
  }
}

template <typename T>
int launch_rows(const SampleArgs& a, int64_t rows, int ranks, const int32_t* list, cudaStream_t s) {
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
  return launch_result(cudaLaunchKernelEx(&cfg, sample_row_kernel<T>, a, list));
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

bool fits_cluster(int vocab) { return row_smem(vocab, 8) <= 226 * 1024 && row_shape(vocab, 8).slice < 65536; }

// Whether passes of separate launches are faster than clusters.  Measured (us, clusters / passes, top-p and fp32 unless told otherwise, means over
// eight draws): 16 rows of 131,072 33 / 34, 32 40 / 38, 64 67 / 51, 256 251 / 142, 256 of bf16 247 / 144; 16 rows of 262,144 60 / 39; 64 rows of
// 65,536 37 / 38, 128 of bf16 63 / 62; with all filters 64 rows of 32,000 25 / 35, 256 55 / 56, top-p alone 512 104 / 94, 256 of bf16 63 / 65;
// 512 rows of 16,384 55 / 68, of 8,192 40 / 56; without filters 512 rows of 32,000 47 / 60, 256 of 131,072 107 / 99; with a small k 32 rows of
// 131,072 in bf16 33 / 52, 64 63 / 65.  Below 65,536 tokens the passes are not much ahead anywhere, take the host 14 us longer to launch and need a
// workspace.
bool wide_is_faster(int64_t rows, int vocab) {
  return fits_cluster(vocab) && sample_wide_takes(rows, vocab) && vocab >= 65536 && rows * vocab >= (int64_t(1) << 22);
}

}  // namespace
}  // namespace b200

extern "C" size_t b200_sample_filtered_workspace_bytes(int64_t num_rows, int32_t vocab_size) {
  using namespace b200;
  if (num_rows <= 0 || vocab_size <= 0) return 0;
  return wide_is_faster(num_rows, vocab_size) ? sample_wide_workspace_bytes(num_rows, vocab_size) : 0;
}

extern "C" int b200_sample_filtered(const void* logits, int64_t row_stride, int64_t num_rows, int32_t vocab_size,
                                    const float* uniforms, const float* temperatures, const int32_t* top_k, const float* top_p,
                                    const float* min_p, int64_t* out_tokens, void* workspace, size_t workspace_bytes, int32_t dtype,
                                    void* stream) {
  using namespace b200;
  if (num_rows < 0 || vocab_size <= 0 || row_stride < vocab_size) return B200_ERR_ARG;
  if (dtype != B200_DTYPE_F32 && dtype != B200_DTYPE_BF16) return B200_ERR_UNSUPPORTED;
  if (num_rows == 0) return B200_OK;
  if (!logits || !uniforms || !temperatures || !out_tokens) return B200_ERR_ARG;
  if (num_rows > 2147483647 || vocab_size > (1 << 24)) return B200_ERR_TOO_LARGE;
  const size_t needed = b200_sample_filtered_workspace_bytes(num_rows, vocab_size);
  if (needed > 0 && (!workspace || workspace_bytes < needed)) return B200_ERR_WORKSPACE;
  SampleArgs a{logits, row_stride, vocab_size, uniforms, temperatures, top_k, top_p, min_p, out_tokens, 62};
  while ((1ll << (62 - a.bits)) < vocab_size) --a.bits;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int sms = sm_count_cached();
  if (sms <= 0) sms = 148;
  if (fits_cluster(vocab_size)) {
    if (a.bits > 45) a.bits = 45;                        // weights below e^-32 round to 0
    const int32_t* list = nullptr;
    int64_t rows = num_rows;
    // CTAs of a row: as many as let two of them fit an SM; more, down to 4,096 logits each, while one wave of CTAs takes all rows.  Times in us of
    // 1, 2, 4 and 8 CTAs: 1 row of 32,000 29, 25, 21, 19; 16 of 32,000 33, 27, 23, 22; 64 of 32,000 38, 29, 29, 46; 256 of 32,000 84, 78, 99,
    // 152; 512 of 8,000 45, 69, 117, 243; 8 of 4,000 17, 19, 19, 19; 32 of 131,072 with 4 and 8 78, 79.
    int ranks = 1;
    while (ranks < 8 && row_smem(vocab_size, ranks) > 110 * 1024) ranks *= 2;
    while (ranks < 8 && num_rows * ranks * 2 <= 2 * sms && vocab_size / ranks > 4096) ranks *= 2;
    if (needed > 0) {
      const int rc = sample_wide_launch(a, num_rows, dtype, workspace, &list, s);
      if (rc != B200_OK) return rc;
      rows = 2 * sms / ranks;                            // clusters that walk the list, most often empty
    }
    if (rows * ranks <= 2147483647)
      return dtype == B200_DTYPE_F32 ? launch_rows<float>(a, rows, ranks, list, s) : launch_rows<__nv_bfloat16>(a, rows, ranks, list, s);
  }
  const int grid = static_cast<int>(num_rows);
  if (dtype == B200_DTYPE_F32) sample_filtered_kernel<float><<<grid, kThreads, 0, s>>>(a);
  else sample_filtered_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
  return launch_result();
}
