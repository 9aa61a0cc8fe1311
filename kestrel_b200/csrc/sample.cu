// One token per row of logits: temperature, top-k, top-p, min-p, from given
// uniform numbers.
//
// With m the row's largest logit, w_j = exp((l_j - m) / T). Tokens are ranked by
// logit, equal ones by index. Kept are the k first; of these the shortest run from
// the first whose sum reaches p times all of theirs; of these those with w_j >=
// min_p. The token is the first in index order at which the running sum of what is
// kept exceeds u times their sum. No order of 150 thousand tokens is needed for
// that: a rank is a place in the order of the pair (logit, -index), so each cut is
// one such pair, and everything else is sums.
//
// Sums decide between neighbours that differ by a millionth of the row, so weights
// are computed in 64 bits (good to 2e-13) and every sum is either of whole numbers
// or in an order that does not depend on timing.
//
// A cluster of up to eight blocks holds a row in its shared memory: the logits are
// read once. On the way into it the maximum; then a histogram over (m - l) finds
// the bins in which the cuts for k and p lie (for p from the bins' counts, so the
// next pass checks it); then one pass over the weights sums what lies above the
// bin, warp by warp, and collects the bin's tokens in one block, which finds the
// cut among them, pair by pair. Each warp has a stretch of indices, so that the
// stretches' sums lead to the one that holds the token, and only it is read again.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "attn_dev.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv.h"
#include "sample.h"

namespace cg = cooperative_groups;

namespace kc {

constexpr int SMP_THREADS = 512, SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_CLUSTER = 8;    // blocks of a row, at most
constexpr int SMP_ALL = SMP_CLUSTER * SMP_WARPS;
constexpr int SMP_COARSE = 128;   // bins of the histogram: four a lane
constexpr int SMP_FINE = 128;     // and of one of them
constexpr int SMP_BINS = SMP_COARSE * SMP_FINE;
constexpr int SMP_LIST = 1024;    // tokens of a bin that one block looks through
constexpr int SMP_SHORT = 512;    // tokens that top-k leaves to one block
constexpr int SMP_TRIES = 40;     // bins looked at for top-p, at most
constexpr float SMP_SPAN = 24.f;  // the histogram reaches so far below the maximum
constexpr double SMP_UNIT = 17592186044416.0;  // 2^44: sums of a list in whole numbers

// What the blocks of a row share: in every block, written by its peers. What they
// tell each other again goes to one of two places by turns: there is a barrier of
// the cluster between two writes to the same, behind which all have read the first.
struct alignas(16) SampleShared {
  union {
    uint32_t coarse[SMP_COARSE][32];  // a column a lane: no two of a warp meet in a bank
    struct {
      uint64_t comp[SMP_LIST];  // listed tokens (rank 0), once the histograms are through
      uint64_t weight[SMP_LIST];
    };
  };
  uint32_t fine[SMP_FINE];
  uint16_t bins[2][SMP_CLUSTER][SMP_COARSE];  // the blocks' histograms (a block holds fewer than 2^16)
  double part[2][4][SMP_ALL];                 // the warps' sums
  uint64_t span[SMP_CLUSTER][2];
  float top[SMP_CLUSTER], low[SMP_CLUSTER];
  int first[SMP_CLUSTER];
  int listed[SMP_TRIES + 1];  // (rank 0)
  // From rank 0: the cut for k; then the stretch that holds the token.
  uint64_t cut;
  double left, total;
  int owner;
  // The block's own.
  double table[16];
  uint64_t add[SMP_ALL];
  uint64_t best, least;
  float red[2 * SMP_WARPS];
};
static_assert(SMP_COARSE == 128 && SMP_FINE == 128 && SMP_ALL == 128, "four a lane");

// A token's place in the order: logit, then the lower index.
__device__ __forceinline__ uint32_t order_key(float l) {
  const uint32_t b = __float_as_uint(l);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
// The logit of a key.
__device__ __forceinline__ float order_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ uint64_t order_of(float l, int index) {
  return (uint64_t)order_key(l) << 32 | (uint32_t)~index;
}

// 2^x for x = d c in -100 .. 0, d <= 0; exactly 1 at 0. x lands on multiples of
// 2^-44 in the mantissa of 384 + x; the nearest multiple of 1/16 is taken from the
// table (one entry a bank: no conflicts), the rest, 1/32 at most, from five terms
// of the series (the sixth is below 2e-13).
__device__ __forceinline__ double weight_of(double d, double c, const double* table) {
  const double y = fma(d, c, 384.0);
  const int h = (__double2hiint(y) + 0x80) & ~0xff;
  const double r = y - __hiloint2double(h, 0);
  double p = 1.3333558146428443e-3;       // ln 2 ^ 5 / 5!
  p = fma(p, r, 9.6181291076284772e-3);   // ^ 4 / 4!
  p = fma(p, r, 5.5504108664821580e-2);   // ^ 3 / 3!
  p = fma(p, r, 2.4022650695910072e-1);   // ^ 2 / 2!
  p = fma(p, r, 6.9314718055994531e-1);   // ln 2
  p = fma(p, r, 1.0);
  const double w = table[(h >> 8) & 15] * p;
  return __hiloint2double(__double2hiint(w) + ((h << 8) & 0x0ff00000) - (128 << 20), __double2loint(w));
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_scan(double v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else {
    alignas(8) T x[4];
    *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)x[i];
  }
}

// 128 values, four a lane; every warp holds the same ones and finds the same.
struct Quad {
  double v[4], before;  // before: the sum of the lanes before
  __device__ __forceinline__ void scan(int lane) {
    const double own = (v[0] + v[1]) + (v[2] + v[3]);
    before = warp_scan(own, lane) - own;
  }
  __device__ __forceinline__ double upto(int e) const {  // up to and with the e-th
    double s = before;
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (y <= e) s += v[y];
    return s;
  }
  // The value that fn(e) has in the lane and place of `at`.
  template <class Fn>
  static __device__ __forceinline__ double of(int at, Fn fn) {
    double x = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e == (at & 3)) x = fn(e);
    return __shfl_sync(0xffffffffu, x, at >> 2);
  }
  // The first (last) place for which fn(e) holds, of all 128; INT_MAX (-1): none.
  template <class Fn>
  static __device__ __forceinline__ int first(int lane, Fn fn) {
    int at = INT_MAX;
#pragma unroll
    for (int e = 3; e >= 0; --e)
      if (fn(e)) at = 4 * lane + e;
    return __reduce_min_sync(0xffffffffu, at);
  }
  template <class Fn>
  static __device__ __forceinline__ int last(int lane, Fn fn) {
    int at = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (fn(e)) at = 4 * lane + e;
    return __reduce_max_sync(0xffffffffu, at);
  }
};

template <typename T>
struct SampleRow {
  SampleShared& s;
  T* logits;              // the block's stretch in shared memory, `chunk` of them
  int chunk, at;          // index of its first
  cg::cluster_group cluster;
  int rank, blocks, tid, warp, lane;
  int turn;               // of what the blocks tell each other
  float m, scale;         // the maximum; bins per unit of m - l
  double c;               // log2(e) / T
  float c32;

  // fn(l, index) of four values a lane at a time, over the warp's stretch (whole warps).
  template <class Fn>
  __device__ __forceinline__ void each4(Fn fn) {
    const int seg = chunk / SMP_WARPS;
    for (int i = warp * seg + 4 * lane; i < (warp + 1) * seg; i += 128) {
      float v[4];
      load4(logits + i, v);
      fn(v, at + i);
    }
  }
  // How far below the maximum, in bins; the bin.
  __device__ __forceinline__ float depth(float l) const { return fminf((m - l) * scale, SMP_BINS - 1); }
  static __device__ __forceinline__ int whole(float depth) {
    return __float_as_int(__fadd_rd(depth, 8388608.f)) & (SMP_BINS - 1);  // (a conversion takes eight times as long)
  }
  // Below 2^-100: zero. (Not a number: minus infinity at T = inf.) Without a branch,
  // so that several are under way.
  __device__ __forceinline__ double weight(float l) const {
    const double w = weight_of((double)l - (double)m, c, s.table);
    const bool some = (m - l) * c32 < 100.f;
    return __hiloint2double(some ? __double2hiint(w) : 0, some ? __double2loint(w) : 0);
  }
  // What a bin's tokens weigh, by its middle (f32 is enough: it is checked).
  __device__ __forceinline__ double guess(uint32_t n, float middle) const {
    return n ? (double)n * exp2f(-middle / scale * c32) : 0.0;
  }
  // Sums of the lanes' v[y] over all blocks, in every lane, after a barrier.
  template <int N>
  __device__ __forceinline__ void totals(double (&v)[N]) {
    double(*part)[SMP_ALL] = s.part[turn & 1];
#pragma unroll
    for (int y = 0; y < N; ++y) {
      v[y] = warp_sum(v[y]);
      if (lane < blocks) *cluster.map_shared_rank(&part[y][rank * SMP_WARPS + warp], lane) = v[y];
    }
    cluster.sync();
    ++turn;
#pragma unroll
    for (int y = 0; y < N; ++y) {
      double sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * lane + e < blocks * SMP_WARPS) sum += part[y][4 * lane + e];
      v[y] = warp_sum(sum);
    }
  }
  // The blocks' histograms (told at turn `of`), in every warp.
  __device__ __forceinline__ void gather_bins(int of, uint32_t (&n)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) n[e] = 0;
    for (int b = 0; b < blocks; ++b) {
      const uint2 y = *reinterpret_cast<const uint2*>(&s.bins[of & 1][b][4 * lane]);
      n[0] += y.x & 0xffff;
      n[1] += y.x >> 16;
      n[2] += y.y & 0xffff;
      n[3] += y.y >> 16;
    }
  }
  // Tokens by bins of one coarse bin, of all blocks; the f32 sums of all weights and
  // of those above the coarse bin. Only logits from `floor` on.
  __device__ __forceinline__ void fine_bins(int coarse, float floor, uint32_t (&n)[4], double& all, double& above) {
    const float begins = coarse * SMP_FINE, ends = begins + SMP_FINE;
    if (tid < SMP_FINE) s.fine[tid] = 0;
    __syncthreads();
    float sum = 0.f, over = 0.f;
    each4([&](const float (&v)[4], int) {
      float r[4], w[4];
      bool here = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r[e] = v[e] >= floor ? depth(v[e]) : -1.f;
        here |= r[e] >= begins && r[e] < ends;
        w[e] = exp2_fast((v[e] - m) * c32);
        w[e] = r[e] >= 0.f && v[e] > -INFINITY ? w[e] : 0.f;
      }
      sum += (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = r[e] < begins ? w[e] : 0.f;
      over += (w[0] + w[1]) + (w[2] + w[3]);
      if (__any_sync(0xffffffffu, here)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r[e] >= begins && r[e] < ends) atomicAdd(&s.fine[whole(r[e]) & (SMP_FINE - 1)], 1u);
      }
    });
    __syncthreads();
    for (int y = tid; y < SMP_FINE * blocks; y += SMP_THREADS)
      cluster.map_shared_rank(&s.bins[turn & 1][rank][0], y / SMP_FINE)[y % SMP_FINE] = (uint16_t)s.fine[y % SMP_FINE];
    double v[2] = {sum, over};
    totals(v);
    all = v[0];
    above = v[1];
    gather_bins(turn - 1, n);
  }
  // Adds a token to rank 0's list (whole warps; nothing past its end).
  __device__ __forceinline__ void list(bool mine, int which, uint64_t comp, double w) {
    const unsigned who = __ballot_sync(0xffffffffu, mine);
    if (!who) return;
    const int lead = __ffs(who) - 1;
    int base = 0;
    if (lane == lead) base = atomicAdd(cluster.map_shared_rank(&s.listed[which], 0), __popc(who));
    base = __shfl_sync(0xffffffffu, base, lead) + __popc(who & ((1u << lane) - 1));
    if (mine && base < SMP_LIST) {
      *cluster.map_shared_rank(&s.comp[base], 0) = comp;
      *cluster.map_shared_rank(&s.weight[base], 0) = (uint64_t)llrint(w * SMP_UNIT);
    }
  }
  // For each listed token i (in rank 0), by threads that share them where the list
  // is short: sum over the list's j of get(i, j), then done(i, sum).
  template <class Get, class Done>
  __device__ __forceinline__ void pairs(int members, Get get, Done done) {
    const int share = members <= SMP_THREADS / 8 ? 8 : members <= SMP_THREADS / 4 ? 4 : members <= SMP_THREADS / 2 ? 2 : 1;
    for (int i0 = 0; i0 < members; i0 += SMP_THREADS / share) {
      const int i = i0 + tid / share, mine = min(i, members - 1);
      uint64_t sum = 0;
      for (int j = tid % share; j < members; j += share) sum += get(mine, j);
      for (int w = 1; w < share; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, (unsigned long long)sum, w);
      if (i < members && tid % share == 0) done(i, sum);
    }
  }
  // The highest place among those of `bin` (and at or past `from`) from which on
  // `measure` of them reaches `want`, by halving the range of places: for bins of
  // more tokens than a list holds. (The lowest, if rounding says that all of them
  // do not.) The blocks take the same steps.
  template <class Measure>
  __device__ uint64_t halve(int bin, uint64_t from, double want, Measure measure) {
    uint64_t lo = ~0ull, hi = 0;
    const auto each = [&](auto fn) {
      each4([&](const float (&v)[4], int i) {
        for (int e = 0; e < 4; ++e) {
          const uint64_t o = order_of(v[e], i + e);
          if (whole(depth(v[e])) == bin && o >= from) fn(v[e], o);
        }
      });
    };
    each([&](float, uint64_t o) {
      lo = min(lo, o);
      hi = max(hi, o);
    });
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      lo = min(lo, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)lo, o));
      hi = max(hi, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)hi, o));
    }
    if (tid == 0) {
      s.least = ~0ull;
      s.best = 0;
    }
    __syncthreads();
    if (lane == 0) {
      atomicMin((unsigned long long*)&s.least, (unsigned long long)lo);
      atomicMax((unsigned long long*)&s.best, (unsigned long long)hi);
    }
    __syncthreads();
    if (tid < blocks) {
      uint64_t* to = cluster.map_shared_rank(&s.span[rank][0], tid);
      to[0] = s.least;
      to[1] = s.best;
    }
    cluster.sync();
    for (int b = 0; b < blocks; ++b) {
      lo = min(lo, s.span[b][0]);
      hi = max(hi, s.span[b][1]);
    }
    while (lo < hi) {
      const uint64_t mid = lo + (hi - lo + 1) / 2;
      double sum[1] = {0};
      each([&](float l, uint64_t o) {
        if (o >= mid) sum[0] += measure(l);
      });
      totals(sum);
      if (sum[0] >= want) lo = mid;
      else hi = mid - 1;
    }
    cluster.sync();
    return lo;
  }
};

template <typename T>
__global__ void __launch_bounds__(SMP_THREADS, 2) sample_kernel(const SampleArgs a, int chunk, bool wide) {
  extern __shared__ __align__(16) uint8_t smp_raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(smp_raw);
  pdl_enter();
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / blocks, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  SampleRow<T> x{s, reinterpret_cast<T*>(smp_raw + sizeof(SampleShared)), chunk, rank * chunk, cluster, rank, blocks,
                 tid, warp, lane, 0};

  // ---- the row into shared memory, its maximum and least value -------------------------
  const float temperature = a.temperature ? a.temperature[row] : 1.f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.f;
  const double p = top_p;
  const double least = a.min_p && a.min_p[row] > 0.f ? fmin(1.0, (double)a.min_p[row]) : 0.0;
  const bool by_k = k > 0 && k < a.n_vocab, by_p = top_p < 1.f, greedy = !(temperature > 0.f);
  if (by_k || by_p)
    for (int i = tid; i < SMP_COARSE * 32; i += SMP_THREADS) s.coarse[i / 32][i % 32] = 0;
  if (tid < 16) s.table[tid] = exp2(tid / 16.0);
  if (tid <= SMP_TRIES) s.listed[tid] = 0;
  float top = -INFINITY, low = INFINITY;
  {
    const T* from = static_cast<const T*>(a.logits) + row * a.stride + x.at;
    const int have = min(chunk, a.n_vocab - x.at);  // (below zero: none)
    constexpr int V = 16 / sizeof(T);
    // Not a number: minus infinity. Minus zero: zero, as which it ranks.
    const auto take = [&](float l) {
      l = l != l ? -INFINITY : l + 0.f;
      top = fmaxf(top, l);
      if (l > -INFINITY) low = fminf(low, l);
      return l;
    };
    int done = 0;
    if (wide) {
      done = max(have, 0) / V * V;
      for (int i0 = V * tid; i0 < done; i0 += 4 * V * SMP_THREADS) {
        uint4 in[4];
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (i0 + y * V * SMP_THREADS < done)
            in[y] = __ldcs(reinterpret_cast<const uint4*>(from + i0 + y * V * SMP_THREADS));
#pragma unroll
        for (int y = 0; y < 4; ++y)
          if (i0 + y * V * SMP_THREADS < done) {
            alignas(16) T v[V];
            *reinterpret_cast<uint4*>(v) = in[y];
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = (T)take((float)v[e]);
            *reinterpret_cast<uint4*>(x.logits + i0 + y * V * SMP_THREADS) = *reinterpret_cast<uint4*>(v);
          }
      }
    }
    for (int i = done + tid; i < chunk; i += SMP_THREADS) x.logits[i] = i < have ? (T)take((float)from[i]) : (T)-INFINITY;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  float* red_f = s.red;
  if (lane == 0) {
    red_f[2 * warp] = top;
    red_f[2 * warp + 1] = low;
  }
  __syncthreads();
  for (int w = 0; w < SMP_WARPS; ++w) {
    top = fmaxf(top, red_f[2 * w]);
    low = fminf(low, red_f[2 * w + 1]);
  }
  if (tid < blocks) {
    *cluster.map_shared_rank(&s.top[rank], tid) = top;
    *cluster.map_shared_rank(&s.low[rank], tid) = low;
  }
  cluster.sync();  // (every block's shared memory is ready for its peers)
  for (int b = 0; b < blocks; ++b) {
    top = fmaxf(top, s.top[b]);
    low = fminf(low, s.low[b]);
  }
  if (top == -INFINITY) {  // nothing to choose from
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.probs) a.probs[row] = 0.f;
    }
    return;
  }
  if (top == INFINITY && !greedy) {
    // Infinite ones share everything.
    for (int i = tid; i < chunk; i += SMP_THREADS) x.logits[i] = (float)x.logits[i] == INFINITY ? (T)0.f : (T)-INFINITY;
    top = low = 0.f;
    __syncthreads();
  }
  x.m = top;

  if (greedy) {
    int first = INT_MAX;
    x.each4([&](const float (&v)[4], int i) {
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (v[e] == top) first = min(first, i + e);
    });
    first = __reduce_min_sync(0xffffffffu, first);
    int* red = reinterpret_cast<int*>(s.red);
    __syncthreads();
    if (lane == 0) red[warp] = first;
    __syncthreads();
    for (int w = 0; w < SMP_WARPS; ++w) first = min(first, red[w]);
    if (tid == 0) *cluster.map_shared_rank(&s.first[rank], 0) = first;
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int b = 0; b < blocks; ++b) first = min(first, s.first[b]);
      a.tokens[row] = first;
      if (a.probs) a.probs[row] = 1.f;
    }
    return;
  }
  x.c = 1.4426950408889634 / temperature;
  x.c32 = (float)fmin(x.c, 3e38);
  x.scale = (SMP_BINS - 1) / fmaxf(fminf(SMP_SPAN, top - low), 1e-30f);
  const float u = a.u[row];
  const double draw = fminf(u > 0.f ? u : 0.f, 0x1.fffffep-1f);

  // ---- the histogram ------------------------------------------------------------------------
  uint64_t cut = 0;   // kept: the places from it on
  uint32_t count[4];  // tokens of coarse bins 4 lane ..
  const int seg = chunk / SMP_WARPS;
  if (by_k || by_p) {
    // What is below (1 - p) / n_vocab of the first adds up to less than 1 - p of
    // all: top-p alone never reaches it. (A little further for roundings.)
    const float reach =
        by_k ? INFINITY : temperature * (logf((float)a.n_vocab) - logf(fmaxf(1.f - top_p, 1e-7f)) + 0.01f);
    x.each4([&](const float (&v)[4], int) {
      int b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = x.whole(x.depth(v[e])) / SMP_FINE;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (top - v[e] <= reach) atomicAdd(&s.coarse[b[e]][lane], 1u);
    });
    __syncthreads();
    {
      // Four threads a bin, eight columns each.
      const int bin = tid / 4, col = 8 * (tid & 3);
      uint32_t n = 0;
#pragma unroll
      for (int y = 0; y < 8; ++y) n += s.coarse[bin][col + ((y + bin) & 7)];
      n += __shfl_xor_sync(0xffffffffu, n, 1);
      n += __shfl_xor_sync(0xffffffffu, n, 2);
      for (int b = tid & 3; b < blocks; b += 4) cluster.map_shared_rank(&s.bins[0][rank][0], b)[bin] = (uint16_t)n;
    }
    cluster.sync();
    ++x.turn;
    x.gather_bins(0, count);
  }

  // ---- top-k ------------------------------------------------------------------------------------
  float floor = -INFINITY;  // (no token below it is kept)
  if (by_k) {
    // (Whole numbers, exact in 64 bits.)
    Quad q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = count[e];
    q.scan(lane);
    const int coarse = Quad::first(lane, [&](int e) { return q.upto(e) >= k; });
    const double through = Quad::of(coarse, [&](int e) { return q.upto(e); });
    if (through <= SMP_SHORT) {
      // Few enough: one block does the rest with them, pair by pair.
      const float ends = (coarse + 1) * SMP_FINE;
      x.each4([&](const float (&v)[4], int i) {
        bool here[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) here[e] = x.depth(v[e]) < ends;
        if (__any_sync(0xffffffffu, here[0] || here[1] || here[2] || here[3])) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x.list(here[e], 0, order_of(v[e], i + e), x.weight(v[e]));
        }
      });
      cluster.sync();
      if (rank != 0) return;
      const int members = s.listed[0];
      uint64_t *placed = s.comp + SMP_SHORT, *kept = s.weight + SMP_SHORT;
      if (tid == 0) s.add[0] = 0;
      // The weights of those at a token's place and above, and in the low bits its
      // rank (512 weights of 2^44 leave room). The k-th's are all of theirs.
      x.pairs(
          members, [&](int i, int j) { return s.comp[j] >= s.comp[i] ? (s.weight[j] << 10) + 1 : 0ull; },
          [&](int i, uint64_t sum) {
            placed[i] = sum;
            if ((sum & 1023) == (uint64_t)k) s.best = sum >> 10;
          });
      __syncthreads();
      const double target = by_p ? p * (double)s.best : INFINITY;
      if (tid < members) {
        const uint64_t w = s.weight[tid], rest = (placed[tid] >> 10) - w, rank_of = placed[tid] & 1023;
        const bool keep = rank_of <= (uint64_t)k && (rank_of == 1 || (double)rest < target) && (double)w >= least * SMP_UNIT;
        kept[tid] = keep ? w : 0;
        if (keep) atomicAdd((unsigned long long*)&s.add[0], (unsigned long long)w);
      }
      __syncthreads();
      const double total = (double)s.add[0], want = draw * total;
      x.pairs(
          members, [&](int i, int j) { return ~(uint32_t)s.comp[j] <= ~(uint32_t)s.comp[i] ? kept[j] : 0ull; },
          [&](int i, uint64_t sum) {
            if ((double)sum > want && (double)(sum - kept[i]) <= want && kept[i]) {
              a.tokens[row] = (int)~(uint32_t)s.comp[i];
              if (a.probs) a.probs[row] = (float)((double)kept[i] / total);
            }
          });
      return;
    }
    // The bin that holds the k-th, then its place among the bin's.
    int rest = k - (int)Quad::of(coarse, [&](int e) { return q.upto(e) - q.v[e]; });
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int b = 4 * lane + e;
      count[e] = b < coarse ? count[e] : b == coarse ? rest : 0;
    }
    uint32_t n[4];
    double none;
    x.fine_bins(coarse, floor, n, none, none);
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = n[e];
    q.scan(lane);
    const int fine = Quad::first(lane, [&](int e) { return q.upto(e) >= rest; }), bin = coarse * SMP_FINE + fine;
    rest -= (int)Quad::of(fine, [&](int e) { return q.upto(e) - q.v[e]; });
    const float begins = bin, ends = bin + 1;
    x.each4([&](const float (&v)[4], int i) {
      bool here[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float r = x.depth(v[e]);
        here[e] = r >= begins && r < ends;
      }
      if (__any_sync(0xffffffffu, here[0] || here[1] || here[2] || here[3])) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x.list(here[e], 0, order_of(v[e], i + e), 0.0);
      }
    });
    cluster.sync();
    const int members = *cluster.map_shared_rank(&s.listed[0], 0);
    if (members <= SMP_LIST) {
      if (rank == 0)
        x.pairs(
            members, [&](int i, int j) { return (uint64_t)(s.comp[j] >= s.comp[i]); },
            [&](int i, uint64_t sum) {
              if (sum == (uint64_t)rest)
                for (int b = 0; b < blocks; ++b) *cluster.map_shared_rank(&s.cut, b) = s.comp[i];
            });
      cluster.sync();
      cut = s.cut;
    } else {
      cut = x.halve(bin, 0, rest, [](float) { return 1.0; });
    }
    floor = order_value((uint32_t)(cut >> 32));
  }

  // ---- weights: sums of what is kept, and the place at which top-p ends -----------------------------
  // The warps' sums of what is kept: s.part[stretch & 1][3].
  int stretch;
  double sums[4] = {0, 0, 0, 0};  // of all, above the bin, in it, kept above it
  if (by_p) {
    // Bins gfrom .. gto are left in question. A coarse one is chosen by the counts'
    // weights, then a bin by those of its own and f32 sums, which a pass checks in
    // 64 bits: if the target is not reached there, the bins on that side are out.
    int gfrom = 0, gto = SMP_BINS - 1, bin = 0, coarse = -1, tries = 0, last = 0, moves = 0;
    uint32_t n[4] = {0, 0, 0, 0};  // tokens of the coarse bin's
    Quad q, fq;                    // weights by the counts
    double fix = 0;                // the sum above the coarse bin
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = x.guess(count[e], (4 * lane + e + 0.5f) * SMP_FINE);
    q.scan(lane);
    double target = p * Quad::of(SMP_COARSE - 1, [&](int e) { return q.upto(e); });
    const auto coarse_open = [&](int e) {
      const int b = 4 * lane + e;
      return count[e] > 0 && b * SMP_FINE <= gto && (b + 1) * SMP_FINE > gfrom;
    };
    const auto fine_open = [&](int e) {
      const int g = coarse * SMP_FINE + 4 * lane + e;
      return n[e] > 0 && g >= gfrom && g <= gto;
    };
    while (true) {
      int next = coarse;
      if (coarse < 0) {
        next = Quad::first(lane, [&](int e) { return coarse_open(e) && q.upto(e) >= target; });
        if (next == INT_MAX) next = Quad::last(lane, coarse_open);
      } else if (Quad::first(lane, fine_open) == INT_MAX) {
        // None left in this one: the next one in the direction of the target.
        next = Quad::first(lane, [&](int e) { return coarse_open(e) && 4 * lane + e > coarse; });
        if (next == INT_MAX) next = Quad::last(lane, [&](int e) { return coarse_open(e) && 4 * lane + e < coarse; });
      }
      if (next < 0) break;  // (rounding: the last bin stands)
      while (next != coarse) {
        const int was = coarse;
        coarse = next;
        double all;
        x.fine_bins(coarse, floor, n, all, fix);
#pragma unroll
        for (int e = 0; e < 4; ++e) fq.v[e] = x.guess(n[e], coarse * SMP_FINE + 4 * lane + e + 0.5f);
        fq.scan(lane);
        if (tries == 0) {
          target = p * all;
          // The f32 sums may already say that it is another coarse bin.
          const double here = Quad::of(SMP_FINE - 1, [&](int e) { return fq.upto(e); });
          const bool high = fix >= target, low_of = fix + here < target;
          if ((high || low_of) && moves++ < 4) {
            const int to = high ? Quad::last(lane, [&](int e) { return coarse_open(e) && 4 * lane + e < coarse; })
                                : Quad::first(lane, [&](int e) { return coarse_open(e) && 4 * lane + e > coarse; });
            if (to >= 0 && to < SMP_COARSE && to != was) next = to;
          }
        }
      }
      int fine = Quad::first(lane, [&](int e) { return fine_open(e) && fix + fq.upto(e) >= target; });
      if (fine == INT_MAX) fine = Quad::last(lane, fine_open);
      if (fine < 0) {  // the coarse bin holds nothing in question
        if (gfrom >= coarse * SMP_FINE) gfrom = max(gfrom, (coarse + 1) * SMP_FINE);
        else gto = min(gto, coarse * SMP_FINE - 1);
        continue;
      }
      bin = coarse * SMP_FINE + fine;
      last = tries;
#pragma unroll
      for (int y = 0; y < 4; ++y) sums[y] = 0;
      const auto pass = [&](auto bounded, auto limited) {
        const float begins = bin, ends = bin + 1;
        x.each4([&](const float (&v)[4], int i) {
          double w[4];
          bool here[4], over[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = x.weight(v[e]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float r = x.depth(v[e]);
            const bool keep = !decltype(bounded)::value || order_of(v[e], i + e) >= cut;
            here[e] = r >= begins && r < ends && keep;
            over[e] = r < begins && keep;
            if (keep) sums[0] += w[e];
            if (over[e]) sums[1] += w[e];
            if (decltype(limited)::value && over[e] && w[e] >= least) sums[3] += w[e];
          }
          if (__any_sync(0xffffffffu, here[0] || here[1] || here[2] || here[3])) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (here[e]) sums[2] += w[e];
              x.list(here[e], 1 + tries, order_of(v[e], i + e), w[e]);
            }
          }
        });
        if (!decltype(limited)::value) sums[3] = sums[1];
      };
      using std::false_type;
      using std::true_type;
      if (by_k) pass(true_type{}, true_type{});
      else if (least > 0) pass(false_type{}, true_type{});
      else pass(false_type{}, false_type{});
      stretch = x.turn;
      x.totals(sums);
      target = p * sums[0];
      const bool high = !(sums[1] < target), low_of = sums[1] + sums[2] < target;
      if (!(high || low_of) || tries + 1 >= SMP_TRIES) break;
      const int was_from = gfrom, was_to = gto;
      if (high) gto = bin - 1;
      else gfrom = bin + 1;
      const int others = Quad::last(lane, [&](int e) { return fine_open(e) || (coarse_open(e) && 4 * lane + e != coarse); });
      if (others < 0) {
        gfrom = was_from;
        gto = was_to;
        break;  // (rounding: the bin stands)
      }
      // The sum up to the bin's beginning is known: the estimates count from there.
      fix = sums[1] - Quad::of(fine, [&](int e) { return fq.upto(e) - fq.v[e]; });
      ++tries;
    }
    const int members = *cluster.map_shared_rank(&s.listed[1 + last], 0);
    if (members <= SMP_LIST) {
      if (rank == 0) {
        // In whole units: the order of the list does not matter.
        if (tid == 0) {
          s.best = 0;
          s.least = ~0ull;
        }
        if (tid < SMP_ALL) s.add[tid] = 0;
        __syncthreads();
        const double need = (target - sums[1]) * SMP_UNIT;
        x.pairs(
            members, [&](int i, int j) { return s.comp[j] >= s.comp[i] ? s.weight[j] : 0ull; },
            [&](int i, uint64_t sum) {
              atomicMin((unsigned long long*)&s.least, (unsigned long long)s.comp[i]);
              if ((double)sum >= need) atomicMax((unsigned long long*)&s.best, (unsigned long long)s.comp[i]);
            });
        __syncthreads();
        // (Rounding may leave the sum short of the target: all of the list.)
        const uint64_t end = s.best ? s.best : s.least;
        if (members) cut = max(cut, end);
        // What is kept of the list, to the stretches.
        for (int i = tid; i < members; i += SMP_THREADS)
          if (s.comp[i] >= cut && (double)s.weight[i] >= least * SMP_UNIT)
            atomicAdd((unsigned long long*)&s.add[(int)~(uint32_t)s.comp[i] / seg], (unsigned long long)s.weight[i]);
        __syncthreads();
        if (tid < blocks * SMP_WARPS) s.part[stretch & 1][3][tid] += (double)s.add[tid] / SMP_UNIT;
        __syncthreads();
      }
    } else {
      cut = max(cut, x.halve(bin, cut, target - sums[1], [&](float l) { return x.weight(l); }));
      double all_kept[4] = {0, 0, 0, 0};
      x.each4([&](const float (&v)[4], int i) {
        for (int e = 0; e < 4; ++e)
          if (order_of(v[e], i + e) >= cut) {
            const double w = x.weight(v[e]);
            if (w >= least) all_kept[3] += w;
          }
      });
      stretch = x.turn;
      x.totals(all_kept);
    }
  } else {
    x.each4([&](const float (&v)[4], int i) {
      if (by_k && !__any_sync(0xffffffffu, v[0] >= floor || v[1] >= floor || v[2] >= floor || v[3] >= floor)) return;
      double w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = x.weight(v[e]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (order_of(v[e], i + e) >= cut && w[e] >= least) sums[3] += w[e];
    });
    stretch = x.turn;
    x.totals(sums);
  }

  // ---- the stretch that holds the token, then the token ------------------------------------------------
  if (rank == 0 && warp == 0) {
    Quad q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = 4 * lane + e < blocks * SMP_WARPS ? s.part[stretch & 1][3][4 * lane + e] : 0.0;
    q.scan(lane);
    const double total = Quad::of(SMP_ALL - 1, [&](int e) { return q.upto(e); }), want = draw * total;
    // The first stretch past whose end the sum exceeds it; if rounding leaves none,
    // the last that holds anything.
    const int first = Quad::first(lane, [&](int e) { return q.v[e] > 0 && q.upto(e) > want; });
    const int last = Quad::last(lane, [&](int e) { return q.v[e] > 0; });
    const double left = first == INT_MAX ? INFINITY : want - Quad::of(first, [&](int e) { return q.upto(e) - q.v[e]; });
    if (lane < blocks) {
      SampleShared& to = *cluster.map_shared_rank(&s, lane);
      to.owner = first == INT_MAX ? last : first;
      to.left = left;
      to.total = total;
      to.cut = cut;
    }
  }
  cluster.sync();
  const int owner = s.owner;
  if (owner / SMP_WARPS != rank || owner % SMP_WARPS != warp) return;
  cut = s.cut;
  double run = 0, w_last = 0;
  int token = -1;  // the last kept one so far
  for (int i0 = warp * seg; i0 < (warp + 1) * seg; i0 += 32) {
    const float l = (float)x.logits[i0 + lane];
    double w = order_of(l, x.at + i0 + lane) >= cut ? x.weight(l) : 0.0;
    if (!(w >= least)) w = 0.0;
    const unsigned some = __ballot_sync(0xffffffffu, w > 0);
    if (!some) continue;
    const double upto = warp_scan(w, lane);
    const unsigned past = __ballot_sync(0xffffffffu, w > 0 && run + upto > s.left);
    const int pick = past ? __ffs(past) - 1 : 31 - __clz(some);
    token = x.at + i0 + pick;
    w_last = __shfl_sync(0xffffffffu, w, pick);
    if (past) break;
    run += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) {
    a.tokens[row] = token;
    if (a.probs) a.probs[row] = (float)(w_last / s.total);
  }
}

template <typename T>
static int run_sample(const SampleArgs& a, cudaStream_t st) {
  constexpr int FIXED = (sizeof(SampleShared) + 15) / 16 * 16;
  static_assert(FIXED == sizeof(SampleShared), "the logits behind it are aligned");
  const auto chunk_of = [&](int blocks) { return ((a.n_vocab + blocks - 1) / blocks + SMP_THREADS * 4 - 1) / (SMP_THREADS * 4) * (SMP_THREADS * 4); };
  // As few blocks as let two share an SM; more where rows leave SMs idle.
  int blocks = 1;
  while (blocks < SMP_CLUSTER && (FIXED + chunk_of(blocks) * (int)sizeof(T) > 112 * 1024 ||
                                  (a.n * blocks * 2 <= num_sms() && chunk_of(blocks) > SMP_THREADS * 8)))
    blocks *= 2;
  const int chunk = chunk_of(blocks), bytes = FIXED + chunk * (int)sizeof(T);
  static PerDeviceOnce attr;
  if (smem_attr_once(attr, sample_kernel<T>, 226 * 1024) != cudaSuccess || bytes > 226 * 1024) return KC_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)(a.n * blocks);
  cfg.blockDim = SMP_THREADS;
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = blocks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const bool wide = !((uintptr_t)a.logits & 15) && a.stride * sizeof(T) % 16 == 0;
  cudaLaunchKernelEx(&cfg, sample_kernel<T>, a, chunk, wide);
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  return KC_OK;
}

int launch_sample(const SampleArgs& a, int t, cudaStream_t st) {
  if (t == T_F32) return run_sample<float>(a, st);
  return t == T_F16 ? run_sample<__half>(a, st) : run_sample<__nv_bfloat16>(a, st);
}

}  // namespace kc
