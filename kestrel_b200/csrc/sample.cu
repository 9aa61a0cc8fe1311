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
// or in an order that does not depend on timing. The whole numbers are units of 2^-60
// of the largest weight, in two words, where any number of tokens may meet, and of
// 2^-54 in lists of 512: off by 2e-13 of it at most, however many there are. (By units
// of 2^-44, in one word, 400 thousand equal light tokens are off by 1e-8, and top-p ends
// elsewhere.)
//
// A cluster of up to eight blocks holds a row in its shared memory: the logits are
// read once. On the way into it the maximum; then a histogram over (m - l) finds
// the bins in which the cuts for k and p lie (for p from the bins' counts, so the
// next pass checks it); then one pass over the weights sums what lies above the
// bin, warp by warp, and collects the bin's tokens in one block, which finds the
// cut among them, pair by pair. Each warp has a stretch of indices, so that the
// stretches' sums lead to the one that holds the token, and only it is read again.
//
// Measured (B200): 256 rows of 151936 f32 logits 310 us under top-p (156 MB: 23.7 us
// at 6559 GB/s), 116 under top-k of 40, 144 without a cut; 32 rows of mixed settings 45;
// one row of 4096 8.1. Bound by the steps of a row, not by memory (DRAM 6% busy, the
// 64-bit pipe 16%): 33 rows of this size are under way, each a chain of a dozen steps
// with a barrier of the cluster behind it.
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
constexpr int SMP_LIST = 512;     // tokens of a bin that one block looks through
constexpr int SMP_SHORT = 256;    // tokens that top-k leaves to one block
constexpr int SMP_FEW = 128;      // the largest k for which the threads' maxima are looked at first
constexpr int SMP_NEAR = 1024;    // tokens of a coarse bin that a block keeps in mind
constexpr float SMP_SPAN = 24.f;  // the histogram reaches so far below the maximum
constexpr double SMP_UNIT = 0x1p54;  // a list's weights in whole numbers, whose sum fits 64 bits
constexpr int SMP_LOW = 16;          // sums over more: units of 2^-60, these bits apart

// What the blocks of a row share: in every block, written by its peers. What they
// tell each other again goes to one of two places by turns: there is a barrier of
// the cluster between two writes to the same, behind which all have read the first.
struct alignas(16) SampleShared {
  union {
    uint32_t coarse[SMP_COARSE][32];  // a column a lane: no two of a warp meet in a bank
    struct {                          // once that histogram is through:
      double weights[SMP_CLUSTER][SMP_FINE];  // the blocks' weights by bins of a coarse bin
      uint64_t comp[SMP_LIST];                // listed tokens (rank 0)
      uint64_t weight[SMP_LIST];
    };
  };
  // Sums of a block's weights, by bins of a coarse bin, then by stretches (add_weight):
  // fewer than 2^16 tokens, so either word holds.
  uint64_t fine[SMP_FINE];
  uint32_t fine_low[SMP_FINE];
  union {
    uint16_t bins[2][SMP_CLUSTER][SMP_COARSE];  // the blocks' counts (a block holds fewer than 2^16)
    uint32_t mass[SMP_CLUSTER][SMP_COARSE];     // or weights
  };
  double part[2][3][SMP_ALL];  // the warps' sums
  uint16_t near[SMP_NEAR];     // places of tokens of a coarse bin in the block's stretch
  int n_near;
  uint64_t span[SMP_CLUSTER][2];
  float top[SMP_CLUSTER], low[SMP_CLUSTER];
  int first[SMP_CLUSTER];  // greedy: the blocks' first maxima
  int listed[3];  // (rank 0)
  int listed_by[SMP_ALL];  // (by warps)
  // From rank 0: the cut for k; then the stretch that holds the token.
  uint64_t cut;
  double left, total;
  int owner;
  // The block's own.
  double table[16];
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
  // (By halves: the steps wait for each other less.)
  const double r2 = r * r;
  const double lo = fma(6.9314718055994531e-1, r, 1.0);                      // ln 2
  const double mid = fma(5.5504108664821580e-2, r, 2.4022650695910072e-1);   // its powers by n!
  const double hi = fma(1.3333558146428443e-3, r, 9.6181291076284772e-3);
  const double p = fma(r2, fma(r2, hi, mid), lo);
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

// ONE: a row is one block's, and no cluster is launched.
template <typename T, bool ONE>
struct SampleRow {
  SampleShared& s;
  T* logits;              // the block's stretch in shared memory, `chunk` of them
  int chunk, at;          // index of its first
  cg::cluster_group cluster;
  int rank, blocks, tid, warp, lane;
  int turn;               // of what the blocks tell each other
  float m, scale;         // the maximum; bins per unit of m - l
  double c;               // log2(e) / T
  float c32, least_l;     // in f32; the least logit that has a weight

  // A barrier of all blocks of the row; a place in block r's shared memory.
  __device__ __forceinline__ void sync() {
    if constexpr (ONE) __syncthreads();
    else cluster.sync();
  }
  template <class P>
  __device__ __forceinline__ P* in_block(P* p, int r) {
    if constexpr (ONE) return p;
    else return cluster.map_shared_rank(p, r);
  }
  // fn(l, index) of four values a lane at a time, over the warp's stretch (whole
  // warps). The next ones are asked for before the last are at work.
  template <class Fn>
  __device__ __forceinline__ void each4(Fn fn) {
    const int seg = chunk / SMP_WARPS, end = (warp + 1) * seg;
    float v[4];
    load4(logits + warp * seg + 4 * lane, v);
    for (int i = warp * seg + 4 * lane; i < end;) {
      float now[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) now[e] = v[e];
      const int here = i;
      i += 128;
      if (i < end) load4(logits + i, v);
      fn(now, at + here);
    }
  }
  // fn(l) of eight values a lane at a time, in no order; not a number where there is
  // none. (For short work, so that more of it is under way.)
  template <class Fn>
  __device__ __forceinline__ void each8(Fn fn) {
    const int seg = chunk / SMP_WARPS, end = (warp + 1) * seg;
    for (int i = warp * seg + 4 * lane; i < end; i += 256) {
      float v[8], w[4];
      load4(logits + i, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = w[e];
      const bool more = i + 128 < end;
      if (more) load4(logits + i + 128, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 + e] = more ? w[e] : NAN;
      fn(v);
    }
  }
  // How far below the maximum, in bins; the bin.
  __device__ __forceinline__ float depth(float l) const { return fminf((m - l) * scale, SMP_BINS - 1); }
  static __device__ __forceinline__ int whole(float depth) {
    return __float_as_int(__fadd_rd(depth, 8388608.f)) & (SMP_BINS - 1);  // (a conversion takes eight times as long)
  }
  // Below 2^-100: zero, as minus infinity has at every T. (By the least logit that has
  // a weight: (m - l) / T in f32 is not finite where m - l or 1 / T is not, though the
  // quotient may be small.) Without a branch, so that several are under way.
  __device__ __forceinline__ double weight(float l) const {
    const double w = weight_of((double)l - (double)m, c, s.table);
    const bool some = l >= least_l;
    return __hiloint2double(some ? __double2hiint(w) : 0, some ? __double2loint(w) : 0);
  }
  // Sums of the lanes' v[y] over all blocks: told before a barrier, in every lane
  // behind it.
  template <int N>
  __device__ __forceinline__ void tell(double (&v)[N]) {
    double(*part)[SMP_ALL] = s.part[turn++ & 1];
#pragma unroll
    for (int y = 0; y < N; ++y) {
      v[y] = warp_sum(v[y]);
      if (lane < blocks) *in_block(&part[y][rank * SMP_WARPS + warp], lane) = v[y];
    }
  }
  template <int N>
  __device__ __forceinline__ void gather(double (&v)[N]) {
    double(*part)[SMP_ALL] = s.part[(turn - 1) & 1];
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
  // s.fine: cleared (a barrier is the caller's), one weight more, what it holds.
  __device__ __forceinline__ void clear_weights() {
    if (tid < SMP_FINE) {
      s.fine[tid] = 0;
      s.fine_low[tid] = 0;
    }
  }
  __device__ __forceinline__ void add_weight(int bin, double w) {
    const uint64_t units = (uint64_t)llrint(w * 0x1p60);
    const uint32_t low = (uint32_t)units & ((1u << SMP_LOW) - 1);
    atomicAdd((unsigned long long*)&s.fine[bin], (unsigned long long)(units >> SMP_LOW));
    if (low) atomicAdd(&s.fine_low[bin], low);
  }
  __device__ __forceinline__ double weights_of(int bin) const {
    return (double)s.fine[bin] * 0x1p-44 + (double)s.fine_low[bin] * 0x1p-60;
  }
  // Tokens by bins of one coarse bin, of all blocks.
  __device__ __forceinline__ void fine_bins(int coarse, uint32_t (&n)[4]) {
    const float begins = coarse * SMP_FINE, ends = begins + SMP_FINE;
    uint32_t* fine = reinterpret_cast<uint32_t*>(s.fine);
    if (tid < SMP_FINE) fine[tid] = 0;
    __syncthreads();
    each4([&](const float (&v)[4], int) {
      float r[4];
      bool here = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r[e] = depth(v[e]);
        here |= r[e] >= begins && r[e] < ends;
      }
      if (__any_sync(0xffffffffu, here)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r[e] >= begins && r[e] < ends) atomicAdd(&fine[whole(r[e]) & (SMP_FINE - 1)], 1u);
      }
    });
    __syncthreads();
    for (int y = tid; y < SMP_FINE * blocks; y += SMP_THREADS)
      in_block(&s.bins[turn & 1][rank][0], y / SMP_FINE)[y % SMP_FINE] = (uint16_t)fine[y % SMP_FINE];
    sync();
    gather_bins(turn++, n);
  }
  // The weight of a listed token, as it was before it became a whole number: min-p goes
  // by it everywhere.
  __device__ __forceinline__ double weight_at(uint64_t comp) const { return weight(order_value((uint32_t)(comp >> 32))); }
  // Adds a token to rank 0's list (whole warps; nothing past its end).
  __device__ __forceinline__ void list(bool mine, int which, uint64_t comp, double w) {
    const unsigned who = __ballot_sync(0xffffffffu, mine);
    if (!who) return;
    const int lead = __ffs(who) - 1;
    int base = 0;
    if (lane == lead) base = atomicAdd(in_block(&s.listed[which], 0), __popc(who));
    base = __shfl_sync(0xffffffffu, base, lead) + __popc(who & ((1u << lane) - 1));
    if (mine && base < SMP_LIST) {
      *in_block(&s.comp[base], 0) = comp;
      *in_block(&s.weight[base], 0) = (uint64_t)llrint(w * SMP_UNIT);
    }
  }
  // For each listed token i (in rank 0), by threads that share them where the list
  // is short: the sum of of[j] over the list's j with is(i, j), and how many there are,
  // then done(i, sum, count).
  template <class Is, class Done>
  __device__ __forceinline__ void pairs(int members, const uint64_t* of, Is is, Done done) {
    const int share = members <= SMP_THREADS / 8 ? 8 : members <= SMP_THREADS / 4 ? 4 : members <= SMP_THREADS / 2 ? 2 : 1;
    for (int i0 = 0; i0 < members; i0 += SMP_THREADS / share) {
      const int i = i0 + tid / share, mine = min(i, members - 1);
      uint64_t sum = 0;
      int count = 0;
      for (int j = tid % share; j < members; j += share) {
        const bool one = is(mine, j);
        sum += one ? of[j] : 0;
        count += one;
      }
      for (int w = 1; w < share; w <<= 1) {
        sum += __shfl_xor_sync(0xffffffffu, (unsigned long long)sum, w);
        count += __shfl_xor_sync(0xffffffffu, count, w);
      }
      if (i < members && tid % share == 0) done(i, sum, count);
    }
  }
  // The blocks' s.fine, summed, after a barrier: four a lane.
  __device__ __forceinline__ void gather_fine(double (&in)[4]) {
    for (int y = tid; y < SMP_FINE * blocks; y += SMP_THREADS)
      in_block(&s.weights[rank][0], y / SMP_FINE)[y % SMP_FINE] = weights_of(y % SMP_FINE);
    sync();
#pragma unroll
    for (int e = 0; e < 4; ++e) in[e] = 0;
    for (int b = 0; b < blocks; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) in[e] += s.weights[b][4 * lane + e];
  }
  // The highest place among those of `bin` (and at or past `from`) from which on
  // `measure` of them (up to 1 each) reaches `want`, for bins of more tokens than a
  // list holds, as where many are equal: the range of places is cut into 128, again
  // and again. (The lowest, if rounding says that all of them do not reach it.) The
  // blocks take the same steps.
  template <class Measure>
  __device__ uint64_t narrow(int bin, uint64_t from, double want, bool near, Measure measure) {
    uint64_t lo = ~0ull, hi = 0;
    // (`near`: the block keeps the bin's tokens in mind, if they are not too many.)
    const auto each = [&](auto fn) {
      if (near && s.n_near <= SMP_NEAR) {
        for (int j = tid; j < s.n_near; j += SMP_THREADS) {
          const int i = s.near[j];
          const float l = (float)logits[i];
          const uint64_t o = order_of(l, at + i);
          if (whole(depth(l)) == bin && o >= from) fn(l, o);
        }
        return;
      }
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
      uint64_t* to = in_block(&s.span[rank][0], tid);
      to[0] = s.least;
      to[1] = s.best;
    }
    sync();
    for (int b = 0; b < blocks; ++b) {
      lo = min(lo, s.span[b][0]);
      hi = max(hi, s.span[b][1]);
    }
    while (lo < hi) {
      const int shift = max(0, 57 - __clzll((long long)(hi - lo)));  // (hi - lo) >> shift < 128
      clear_weights();
      __syncthreads();
      each([&](float l, uint64_t o) {
        if (o >= lo && o <= hi) add_weight((int)((o - lo) >> shift), measure(l));
      });
      __syncthreads();
      Quad f;
      gather_fine(f.v);
      f.scan(lane);
      const double all = Quad::of(SMP_FINE - 1, [&](int e) { return f.upto(e); });
      int part = Quad::last(lane, [&](int e) { return f.v[e] > 0 && all - (f.upto(e) - f.v[e]) >= want; });
      if (part < 0) part = max(0, Quad::first(lane, [&](int e) { return f.v[e] > 0; }) & (SMP_FINE - 1));
      want -= all - Quad::of(part, [&](int e) { return f.upto(e); });
      lo += (uint64_t)part << shift;
      hi = lo + min(hi - lo, ((uint64_t)1 << shift) - 1);  // (the part's end may lie past 64 bits)
      sync();  // (all have read the sums)
    }
    return lo;
  }
};

template <typename T, bool ONE>
__global__ void __launch_bounds__(SMP_THREADS, 2) sample_kernel(const SampleArgs a, int chunk, bool wide) {
  extern __shared__ __align__(16) uint8_t smp_raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(smp_raw);
  pdl_enter();
  cg::cluster_group cluster = cg::this_cluster();
  // A block's shared memory may be written by its peers once it runs: all say so here,
  // and the first to write waits for it, behind its loads.
  if constexpr (!ONE) cluster.barrier_arrive();
  const int blocks = ONE ? 1 : (int)cluster.num_blocks(), rank = ONE ? 0 : (int)cluster.block_rank();
  const int row = blockIdx.x / blocks, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  SampleRow<T, ONE> x{s, reinterpret_cast<T*>(smp_raw + sizeof(SampleShared)), chunk, rank * chunk, cluster, rank, blocks,
                 tid, warp, lane, 0};

  // ---- the row into shared memory, its maximum and least value -------------------------
  const int64_t number = row + (a.at ? *a.at : 0);  // the row's of u and probs
  const float temperature = a.temperature ? a.temperature[row] : 1.f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.f;
  const double p = top_p;
  const double least = a.min_p && a.min_p[row] > 0.f ? fmin(1.0, (double)a.min_p[row]) : 0.0;
  const bool by_k = k > 0 && k < a.n_vocab, by_p = top_p < 1.f, greedy = !(temperature > 0.f);
  if (by_k || by_p)
    for (int i = tid; i < SMP_COARSE * 32; i += SMP_THREADS) s.coarse[i / 32][i % 32] = 0;
  if (tid < 16) s.table[tid] = exp2(tid / 16.0);
  if (tid < 3) s.listed[tid] = 0;
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
  float thread_top = top;  // of the thread's own tokens
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
  if constexpr (!ONE) cluster.barrier_wait();
  if (tid < blocks) {
    *x.in_block(&s.top[rank], tid) = top;
    *x.in_block(&s.low[rank], tid) = low;
  }
  x.sync();  // (and what the blocks have set up of their own is ready for their peers)
  for (int b = 0; b < blocks; ++b) {
    top = fmaxf(top, s.top[b]);
    low = fminf(low, s.low[b]);
  }
  if (top == -INFINITY) {  // nothing to choose from
    if (rank == 0 && tid == 0) {
      a.tokens[row] = -1;
      if (a.probs) a.probs[number] = 0.f;
    }
    return;
  }
  if (top == INFINITY && !greedy) {
    // Infinite ones share everything.
    for (int i = tid; i < chunk; i += SMP_THREADS) x.logits[i] = (float)x.logits[i] == INFINITY ? (T)0.f : (T)-INFINITY;
    thread_top = thread_top == INFINITY ? 0.f : -INFINITY;
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
    if (tid == 0) *x.in_block(&s.first[rank], 0) = first;
    x.sync();
    if (rank == 0 && tid == 0) {
      for (int b = 0; b < blocks; ++b) first = min(first, s.first[b]);
      a.tokens[row] = first;
      if (a.probs) a.probs[number] = 1.f;
    }
    return;
  }
  x.c = 1.4426950408889634 / temperature;
  x.c32 = (float)fmin(x.c, 3e38);
  x.least_l = fmaxf(__double2float_ru((double)top - 100.0 / x.c), -3.4028235e38f);
  x.scale = (SMP_BINS - 1) / fmaxf(fminf(SMP_SPAN, top - low), 1e-30f);
  const float u = a.u[number];
  const double draw = fminf(u > 0.f ? u : 0.f, 0x1.fffffep-1f);

  // ---- the histogram ------------------------------------------------------------------------
  uint64_t cut = 0;  // kept: the places from it on
  const int seg = chunk / SMP_WARPS;
  // Sums of a histogram's columns, told to all blocks: four threads a bin, eight
  // columns each.
  const auto tell_columns = [&](auto put) {
    __syncthreads();
    const int bin = tid / 4, col = 8 * (tid & 3);
    uint32_t n = 0;
#pragma unroll
    for (int y = 0; y < 8; ++y) n += s.coarse[bin][col + ((y + bin) & 7)];
    n += __shfl_xor_sync(0xffffffffu, n, 1);
    n += __shfl_xor_sync(0xffffffffu, n, 2);
    for (int b = tid & 3; b < blocks; b += 4) put(b, bin, n);
    x.sync();
  };

  // ---- top-k ------------------------------------------------------------------------------------
  float floor = -INFINITY;  // (no token below it is kept)
  if (by_k) {
    // The tokens down to a coarse bin to rank 0's list; how many there were. (Every
    // block counts its own: rank 0's list is gone with rank 0.)
    const auto list_down_to = [&](int coarse) {
      const float ends = (coarse + 1) * SMP_FINE;
      int mine = 0;
      x.each4([&](const float (&v)[4], int i) {
        bool here[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) here[e] = x.depth(v[e]) < ends;
        if (__any_sync(0xffffffffu, here[0] || here[1] || here[2] || here[3])) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            mine += here[e];
            x.list(here[e], 0, order_of(v[e], i + e), x.weight(v[e]));
          }
        }
      });
      mine = __reduce_add_sync(0xffffffffu, mine);
      if (lane < blocks) *x.in_block(&s.listed_by[rank * SMP_WARPS + warp], lane) = mine;
      x.sync();
      int all = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * lane + e < blocks * SMP_WARPS) all += s.listed_by[4 * lane + e];
      return (int)__reduce_add_sync(0xffffffffu, all);
    };
    // Few enough: rank 0 does the rest with them, pair by pair.
    const auto finish = [&](int members) {
      uint64_t *placed = s.comp + SMP_SHORT, *kept = s.weight + SMP_SHORT, *all = s.fine;
      uint16_t* ranks = s.near;
      if (tid == 0) *all = 0;
      // The weights of those at a token's place and above, and its rank. The k-th's
      // are all of theirs.
      x.pairs(
          members, s.weight, [&](int i, int j) { return s.comp[j] >= s.comp[i]; },
          [&](int i, uint64_t sum, int count) {
            placed[i] = sum;
            ranks[i] = (uint16_t)count;
            if (count == k) s.best = sum;
          });
      __syncthreads();
      const double target = by_p ? p * (double)s.best : INFINITY;
      if (tid < members) {
        const uint64_t w = s.weight[tid], rest = placed[tid] - w;
        const int rank_of = ranks[tid];
        const bool keep = rank_of <= k && (rank_of == 1 || (double)rest < target) && x.weight_at(s.comp[tid]) >= least;
        kept[tid] = keep ? w : 0;
        if (keep) atomicAdd((unsigned long long*)all, (unsigned long long)w);
      }
      __syncthreads();
      const double total = (double)*all, want = draw * total;
      x.pairs(
          members, kept, [&](int i, int j) { return ~(uint32_t)s.comp[j] <= ~(uint32_t)s.comp[i]; },
          [&](int i, uint64_t sum, int) {
            if ((double)sum > want && (double)(sum - kept[i]) <= want && kept[i]) {
              a.tokens[row] = (int)~(uint32_t)s.comp[i];
              if (a.probs) a.probs[number] = (float)((double)kept[i] / total);
            }
          });
    };
    uint32_t count[4];  // of coarse bins 4 lane ..
    Quad q;
    if (k <= SMP_FEW) {
      // The k-th largest of the threads' maxima is no more than the k-th largest
      // token: the tokens down to its coarse bin are enough, and seldom many more. (A
      // histogram of a value a thread instead of all: 256 rows of 151936 by top-k 40
      // took 123 us with that of all.)
      atomicAdd(&s.coarse[x.whole(x.depth(thread_top)) / SMP_FINE][lane], 1u);
      tell_columns([&](int b, int bin, uint32_t n) { x.in_block(&s.bins[0][rank][0], b)[bin] = (uint16_t)n; });
      x.gather_bins(x.turn++, count);
#pragma unroll
      for (int e = 0; e < 4; ++e) q.v[e] = count[e];
      q.scan(lane);
      const int coarse = Quad::first(lane, [&](int e) { return q.upto(e) >= k; });
      if (coarse < SMP_COARSE - 1) {
        const int members = list_down_to(coarse);
        if (members <= SMP_SHORT) {
          if (rank == 0) finish(members);
          return;
        }
      }
      for (int i = tid; i < SMP_COARSE * 32; i += SMP_THREADS) s.coarse[i / 32][i % 32] = 0;
      __syncthreads();
    }
    x.each4([&](const float (&v)[4], int) {
      int b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = x.whole(x.depth(v[e])) / SMP_FINE;
#pragma unroll
      for (int e = 0; e < 4; ++e) atomicAdd(&s.coarse[b[e]][lane], 1u);
    });
    const int counts = x.turn;
    tell_columns([&](int b, int bin, uint32_t n) {
      x.in_block(&s.bins[counts & 1][rank][0], b)[bin] = (uint16_t)n;
    });
    x.gather_bins(x.turn++, count);
    // (Whole numbers, exact in 64 bits.)
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = count[e];
    q.scan(lane);
    const int coarse = Quad::first(lane, [&](int e) { return q.upto(e) >= k; });
    const double through = Quad::of(coarse, [&](int e) { return q.upto(e); });
    if (k > SMP_FEW && through <= SMP_SHORT) {
      const int members = list_down_to(coarse);
      if (rank == 0) finish(members);
      return;
    }
    // The bin that holds the k-th, then its place among the bin's.
    int rest = k - (int)Quad::of(coarse, [&](int e) { return q.upto(e) - q.v[e]; });
    uint32_t n[4];
    x.fine_bins(coarse, n);
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
        for (int e = 0; e < 4; ++e) x.list(here[e], 2, order_of(v[e], i + e), 0.0);
      }
    });
    x.sync();
    const int members = *x.in_block(&s.listed[2], 0);
    if (members <= SMP_LIST) {
      if (rank == 0)
        x.pairs(
            members, s.weight, [&](int i, int j) { return s.comp[j] >= s.comp[i]; },
            [&](int i, uint64_t, int count) {
              if (count == rest)
                for (int b = 0; b < blocks; ++b) *x.in_block(&s.cut, b) = s.comp[i];
            });
      x.sync();
      cut = s.cut;
    } else {
      cut = x.narrow(bin, 0, rest, false, [](float) { return 1.0; });
    }
    floor = order_value((uint32_t)(cut >> 32));
  }

  // ---- weights: sums of what is kept, and the place at which top-p ends -----------------------------
  int stretch;                 // the warps' sums of what is kept: s.part[stretch & 1][2]
  double sums[3] = {0, 0, 0};  // of all, above a bin, kept
  if (by_p) {
    // The coarse bins' weights, in 2^-16 of a token at each bin's beginning.
    const float unit = x.c32 / x.scale;
    if (by_k) {
      for (int i = tid; i < SMP_COARSE * 32; i += SMP_THREADS) s.coarse[i / 32][i % 32] = 0;
      __syncthreads();
    }
    x.each8([&](const float (&v)[8]) {
      int b[8];
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // (However far apart two finite logits are, their step is finite.)
        const float t = fminf(x.m - v[e], 1e35f) * x.scale, begins = __fadd_rd(fminf(t, SMP_BINS - 1) * (1.f / SMP_FINE), 8388608.f);
        b[e] = __float_as_int(begins) & (SMP_COARSE - 1);
        const float part = exp2_fast(((begins - 8388608.f) * SMP_FINE - t) * unit);
        // (None is lost that has a weight; the last bin's many without any count nothing.)
        w[e] = t * unit < 100.f ? max(1, __float_as_int(__fadd_rn(part * 65536.f, 8388608.f)) & 0x1ffff) : 0;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v[e] >= floor) atomicAdd(&s.coarse[b[e]][lane], w[e]);  // (not of NAN)
    });
    tell_columns([&](int b, int bin, uint32_t n) { x.in_block(&s.mass[rank][0], b)[bin] = n; });
    Quad q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = 0;
    for (int b = 0; b < blocks; ++b) {
      const uint4 y = *reinterpret_cast<const uint4*>(&s.mass[b][4 * lane]);
      q.v[0] += y.x;
      q.v[1] += y.y;
      q.v[2] += y.z;
      q.v[3] += y.w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] *= exp2f(-((4 * lane + e) * SMP_FINE) * unit);
    q.scan(lane);
    // Coarse bins from .. to are left in question. The one in which the sum reaches the
    // target is taken by these weights; a pass checks it in 64 bits, and has its bins'.
    int from = 0, to = SMP_COARSE - 1, bin = 0;
    double target = p * Quad::of(SMP_COARSE - 1, [&](int e) { return q.upto(e); }), rest = 0;
    const auto open = [&](int e) { return q.v[e] > 0 && 4 * lane + e >= from && 4 * lane + e <= to; };
    int coarse = Quad::first(lane, [&](int e) { return open(e) && q.upto(e) >= target; });
    if (coarse == INT_MAX) coarse = Quad::last(lane, open);
    coarse = max(coarse, 0);  // (the first token's bin, if its weight is lost in 2^-16)
    Quad f;
    for (int tries = 0;; ++tries) {
      x.clear_weights();
      if (tid == 0) s.n_near = 0;
      __syncthreads();
#pragma unroll
      for (int y = 0; y < 3; ++y) sums[y] = 0;
      const auto pass = [&](auto bounded, auto limited) {
        const float begins = coarse * SMP_FINE, ends = begins + SMP_FINE;
        x.each4([&](const float (&v)[4], int i) {
          double w[4], over[4];
          bool here[4];
          // (Beyond the k first there is nothing: 32 rows of mixed settings take 47 us
          // so, 50 with the weights of all.)
          if (decltype(bounded)::value &&
              !__any_sync(0xffffffffu, v[0] >= floor || v[1] >= floor || v[2] >= floor || v[3] >= floor))
            return;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = x.weight(v[e]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float r = x.depth(v[e]);
            const bool keep = !decltype(bounded)::value || order_of(v[e], i + e) >= cut;
            here[e] = r >= begins && r < ends && keep;
            if (!keep) w[e] = 0.0;
            over[e] = r < begins ? w[e] : 0.0;
          }
          sums[0] += (w[0] + w[1]) + (w[2] + w[3]);
          sums[1] += (over[0] + over[1]) + (over[2] + over[3]);
          if (decltype(limited)::value) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (over[e] >= least) sums[2] += over[e];
          }
          if (__any_sync(0xffffffffu, here[0] || here[1] || here[2] || here[3])) {
            // To what the block keeps in mind, a place in the order of the lanes.
            unsigned who[4];
            int at = 0, all = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              who[e] = __ballot_sync(0xffffffffu, here[e]);
              at += __popc(who[e] & ((1u << lane) - 1));
              all += __popc(who[e]);
            }
            int base = 0;
            if (lane == 0) base = atomicAdd(&s.n_near, all);
            at += __shfl_sync(0xffffffffu, base, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (here[e]) {
                if (at < SMP_NEAR) s.near[at] = (uint16_t)(i + e - x.at);
                ++at;
              }
          }
        });
        if (!decltype(limited)::value) sums[2] = sums[1];
      };
      using std::false_type;
      using std::true_type;
      if (by_k) pass(true_type{}, true_type{});
      else if (least > 0) pass(false_type{}, true_type{});
      else pass(false_type{}, false_type{});
      __syncthreads();
      // The weights of the bins of the coarse one.
      const auto weigh = [&](float l, int i) {
        if (order_of(l, i) >= cut) x.add_weight(x.whole(x.depth(l)) & (SMP_FINE - 1), x.weight(l));
      };
      if (s.n_near <= SMP_NEAR) {
        for (int j = tid; j < s.n_near; j += SMP_THREADS) weigh((float)x.logits[s.near[j]], x.at + s.near[j]);
      } else {
        const float begins = coarse * SMP_FINE, ends = begins + SMP_FINE;
        x.each4([&](const float (&v)[4], int i) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (x.depth(v[e]) >= begins && x.depth(v[e]) < ends) weigh(v[e], i + e);
        });
      }
      __syncthreads();
      // (One barrier for both.)
      double total[2] = {sums[0], sums[1]};
      x.tell(total);
      x.gather_fine(f.v);
      x.gather(total);
      f.scan(lane);
      target = p * total[0];
      rest = target - total[1];  // of the coarse bin's
      const double inside = Quad::of(SMP_FINE - 1, [&](int e) { return f.upto(e); });
      // Not the bin: the next one in the target's direction that holds anything, and
      // from the third on those in question are halved.
      const bool high = !(rest > 0), low_of = inside < rest;
      if (!(high || low_of)) break;
      if (high) to = coarse - 1;
      else from = coarse + 1;
      int next = high ? Quad::last(lane, open) : Quad::first(lane, open);
      if (next < 0 || next >= SMP_COARSE) break;  // (rounding: the bin stands)
      if (tries > 1) {
        const int half = (from + to) / 2;
        next = Quad::last(lane, [&](int e) { return open(e) && 4 * lane + e <= half; });
        if (next < 0) next = Quad::first(lane, open);
      }
      coarse = next;
      x.sync();  // (all have read the weights)
    }
    // The bin in which the sum reaches the target, and what it lacks at its beginning.
    int fine = Quad::first(lane, [&](int e) { return f.v[e] > 0 && f.upto(e) >= rest; });
    if (fine == INT_MAX) fine = max(0, Quad::last(lane, [&](int e) { return f.v[e] > 0; }));
    rest -= Quad::of(fine, [&](int e) { return f.upto(e) - f.v[e]; });
    bin = coarse * SMP_FINE + fine;
    {
      // Its tokens to rank 0's list, those above it to what their stretches keep.
      const float begins = coarse * SMP_FINE, at_bin = bin, ends = bin + 1;
      x.clear_weights();
      __syncthreads();
      const auto place = [&](float l, int i, bool real) {
        const float r = x.depth(l);
        const bool keep = real && order_of(l, i) >= cut, here = keep && r >= at_bin && r < ends;
        const double w = x.weight(l);
        if (keep && r >= begins && r < at_bin && w >= least) x.add_weight((i - x.at) / seg, w);
        x.list(here, 1, order_of(l, i), w);
      };
      if (s.n_near <= SMP_NEAR) {
        for (int j0 = 0; j0 < s.n_near; j0 += SMP_THREADS) {
          const bool real = j0 + tid < s.n_near;
          const int i = real ? s.near[j0 + tid] : 0;
          place((float)x.logits[i], x.at + i, real);
        }
      } else {
        x.each4([&](const float (&v)[4], int i) {
          bool some = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) some |= x.depth(v[e]) >= begins && x.depth(v[e]) < ends;
          if (__any_sync(0xffffffffu, some)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) place(v[e], i + e, true);
          }
        });
      }
      __syncthreads();
      const double mine = warp_sum(sums[2]) + x.weights_of(warp);
      stretch = x.turn++;
      if (lane == 0) *x.in_block(&s.part[stretch & 1][2][rank * SMP_WARPS + warp], 0) = mine;
      x.sync();
    }
    const int members = *x.in_block(&s.listed[1], 0);
    if (members <= SMP_LIST) {
      if (rank == 0) {
        // In whole units: the order of the list does not matter.
        if (tid == 0) {
          s.best = 0;
          s.least = ~0ull;
        }
        x.clear_weights();
        __syncthreads();
        const double need = rest * SMP_UNIT;
        x.pairs(
            members, s.weight, [&](int i, int j) { return s.comp[j] >= s.comp[i]; },
            [&](int i, uint64_t sum, int) {
              atomicMin((unsigned long long*)&s.least, (unsigned long long)s.comp[i]);
              if ((double)sum >= need) atomicMax((unsigned long long*)&s.best, (unsigned long long)s.comp[i]);
            });
        __syncthreads();
        // (Rounding may leave the sum short of the target: all of the list.)
        const uint64_t end = s.best ? s.best : s.least;
        if (members) cut = max(cut, end);
        // What is kept of the list, to the stretches.
        for (int i = tid; i < members; i += SMP_THREADS) {
          const double w = x.weight_at(s.comp[i]);
          if (s.comp[i] >= cut && w >= least) x.add_weight((int)~(uint32_t)s.comp[i] / seg, w);
        }
        __syncthreads();
        if (tid < blocks * SMP_WARPS) s.part[stretch & 1][2][tid] += x.weights_of(tid);
        __syncthreads();
      }
    } else {
      cut = max(cut, x.narrow(bin, cut, rest, true, [&](float l) { return x.weight(l); }));
      double all_kept[3] = {0, 0, 0};
      x.each4([&](const float (&v)[4], int i) {
        for (int e = 0; e < 4; ++e)
          if (order_of(v[e], i + e) >= cut) {
            const double w = x.weight(v[e]);
            if (w >= least) all_kept[2] += w;
          }
      });
      stretch = x.turn;
      x.tell(all_kept);
      x.sync();
    }
  } else {
    x.each4([&](const float (&v)[4], int i) {
      if (by_k && !__any_sync(0xffffffffu, v[0] >= floor || v[1] >= floor || v[2] >= floor || v[3] >= floor)) return;
      double w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = x.weight(v[e]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (order_of(v[e], i + e) >= cut && w[e] >= least) sums[2] += w[e];
    });
    stretch = x.turn;
    x.tell(sums);
    x.sync();
  }

  // ---- the stretch that holds the token, then the token ------------------------------------------------
  if (rank == 0 && warp == 0) {
    Quad q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = 4 * lane + e < blocks * SMP_WARPS ? s.part[stretch & 1][2][4 * lane + e] : 0.0;
    q.scan(lane);
    const double total = Quad::of(SMP_ALL - 1, [&](int e) { return q.upto(e); }), want = draw * total;
    // The first stretch past whose end the sum exceeds it; if rounding leaves none,
    // the last that holds anything.
    const int first = Quad::first(lane, [&](int e) { return q.v[e] > 0 && q.upto(e) > want; });
    const int last = Quad::last(lane, [&](int e) { return q.v[e] > 0; });
    const double left = first == INT_MAX ? INFINITY : want - Quad::of(first, [&](int e) { return q.upto(e) - q.v[e]; });
    if (lane < blocks) {
      SampleShared& to = *x.in_block(&s, lane);
      to.owner = first == INT_MAX ? max(last, 0) : first;
      to.left = left;
      to.total = total;
      to.cut = cut;
    }
  }
  x.sync();
  const int owner = s.owner;
  if (owner / SMP_WARPS != rank) return;
  // The block's threads have a few tokens of the stretch each, in their order. (One
  // warp for all of them took 10 us.)
  cut = s.cut;
  const int per = (seg + SMP_THREADS - 1) / SMP_THREADS, first_at = (owner % SMP_WARPS) * seg + tid * per,
            end_at = min(first_at + per, (owner % SMP_WARPS + 1) * seg);
  const auto kept_weight = [&](int i) {
    const float l = (float)x.logits[i];
    const double w = order_of(l, x.at + i) >= cut ? x.weight(l) : 0.0;
    return w >= least ? w : 0.0;
  };
  double own = 0;
  for (int i = first_at; i < end_at; ++i) own += kept_weight(i);
  double upto = warp_scan(own, lane);
  double* sums_of = s.part[0][0];
  __syncthreads();
  if (lane == 31) sums_of[warp] = upto;
  if (tid == 0) {
    s.first[0] = INT_MAX;
    s.first[1] = -1;
  }
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto += sums_of[w];
  if (own > 0) {
    if (upto > s.left) atomicMin(&s.first[0], tid);
    atomicMax(&s.first[1], tid);
  }
  __syncthreads();
  // (If rounding leaves none past it, the last that holds anything.)
  if (tid != (s.first[0] != INT_MAX ? s.first[0] : s.first[1])) return;
  double run = upto - own, w_last = 0;
  int token = -1;
  for (int i = first_at; i < end_at; ++i) {
    const double w = kept_weight(i);
    if (w == 0) continue;
    token = x.at + i;
    w_last = w;
    run += w;
    if (run > s.left) break;
  }
  a.tokens[row] = token;
  if (a.probs) a.probs[number] = (float)(w_last / s.total);
}

constexpr int SMP_FIXED = (sizeof(SampleShared) + 15) / 16 * 16;
static_assert(SMP_FIXED == sizeof(SampleShared), "the logits behind it are aligned");

template <typename T, bool ONE>
static int run_blocks(const SampleArgs& a, int blocks, int chunk, cudaStream_t st) {
  const int bytes = SMP_FIXED + chunk * (int)sizeof(T);
  static PerDeviceOnce attr;
  if (smem_attr_once(attr, sample_kernel<T, ONE>, 226 * 1024) != cudaSuccess || bytes > 226 * 1024) return KC_ERR_CUDA;
  const bool wide = !((uintptr_t)a.logits & 15) && a.stride * sizeof(T) % 16 == 0;
  if constexpr (ONE) {
    launch_k(sample_kernel<T, ONE>, a.n, SMP_THREADS, bytes, st, a, chunk, wide);
  } else {
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
    cudaLaunchKernelEx(&cfg, sample_kernel<T, ONE>, a, chunk, wide);
    g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  }
  return KC_OK;
}

template <typename T>
static int run_sample(const SampleArgs& a, cudaStream_t st) {
  const auto chunk_of = [&](int blocks) { return ((a.n_vocab + blocks - 1) / blocks + SMP_THREADS * 4 - 1) / (SMP_THREADS * 4) * (SMP_THREADS * 4); };
  // As few blocks as let two share an SM; where rows leave SMs idle more, of 4096
  // tokens at least, but one for up to 8192 (us, one block and two: a row of 8192 bf16
  // under top-p 14.2 and 15.4, 32 of 8192 of mixed settings 21.4 and 22.6; of 16000
  // 25.6 and, in four, 25.2, one under top-p 18.6 and 16.4).
  int blocks = 1;
  while (blocks < SMP_CLUSTER && (SMP_FIXED + chunk_of(blocks) * (int)sizeof(T) > 112 * 1024 ||
                                  (a.n * blocks * 2 <= num_sms() && chunk_of(blocks) > SMP_THREADS * (blocks > 1 ? 8 : 16))))
    blocks *= 2;
  // (A block alone has barriers of its own and plain addresses: a row of 4096 takes 8.2
  // us so, 9.8 as a cluster of one, 16 of mixed settings 15.3 and 20.7.)
  return blocks == 1 ? run_blocks<T, true>(a, 1, chunk_of(1), st) : run_blocks<T, false>(a, blocks, chunk_of(blocks), st);
}

int launch_sample(const SampleArgs& a, int t, cudaStream_t st) {
  if (t == T_F32) return run_sample<float>(a, st);
  return t == T_F16 ? run_sample<__half>(a, st) : run_sample<__nv_bfloat16>(a, st);
}

}  // namespace kc
