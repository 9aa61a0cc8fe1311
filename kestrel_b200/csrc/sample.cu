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

#include "attn_dev.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv.h"
#include "sample.h"

namespace cg = cooperative_groups;

namespace kc {

constexpr int SMP_THREADS = 512, SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_CLUSTER = 8;    // blocks of a row, at most
constexpr int SMP_BINS = 2048;
constexpr int SMP_LIST = 1024;    // tokens of a bin that one block looks through
constexpr int SMP_TRIES = 40;     // bins looked at for top-p, at most
constexpr float SMP_SPAN = 24.f;  // the histogram reaches so far below the maximum
constexpr double SMP_UNIT = 17592186044416.0;  // 2^44: sums of a list in whole numbers

// What the blocks of a row share: in every block, written by its peers.
struct alignas(16) SampleShared {
  uint32_t bins[SMP_BINS];
  uint64_t comp[SMP_LIST];   // tokens of a bin (rank 0)
  uint64_t weight[SMP_LIST];
  double table[16];
  double warp_sum[SMP_CLUSTER * SMP_WARPS];  // kept weights of every warp's stretch (rank 0)
  double part[2][3][SMP_CLUSTER];  // by turns: the blocks' sums
  uint64_t span[SMP_CLUSTER][2];
  float top[SMP_CLUSTER], low[SMP_CLUSTER];
  int first[SMP_CLUSTER];
  int listed[SMP_TRIES + 1];  // (rank 0)
  // From rank 0: the cut for k; then the stretch that holds the token.
  uint64_t cut;
  double left, total;
  int owner;
  // The block's own.
  double red[SMP_WARPS];
  int red_i[SMP_WARPS];
  uint64_t best, least;
  uint64_t add[SMP_CLUSTER * SMP_WARPS];
  int found_bin, last_bin, found_above;
};

// A token's place in the order: logit, then the lower index.
__device__ __forceinline__ uint32_t order_key(float l) {
  const uint32_t b = __float_as_uint(l);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
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

template <typename T>
struct SampleRow {
  const SampleArgs& a;
  SampleShared& s;
  T* logits;              // the block's stretch in shared memory, `chunk` of them
  int chunk, at;          // index of its first
  cg::cluster_group cluster;
  int rank, blocks, tid, warp, lane;
  float m, scale;         // the maximum; bins per unit of m - l
  double c;               // log2(e) / T
  float c32;

  // fn(l, index) for the warp's stretch, four values a lane at a time.
  template <class Fn>
  __device__ __forceinline__ void each(Fn fn) {
    const int seg = chunk / SMP_WARPS;
    for (int i = warp * seg + 4 * lane; i < (warp + 1) * seg; i += 128) {
      float v[4];
      load4(logits + i, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) fn(v[e], at + i + e);
    }
  }
  __device__ __forceinline__ int bin_of(float l) const {
    return min(SMP_BINS - 1, __float2int_rz((m - l) * scale));
  }
  // Below 2^-100: zero. (Not a number: minus infinity at T = inf.)
  __device__ __forceinline__ double weight(float l) const {
    if (!((m - l) * c32 < 100.f)) return 0.0;
    return weight_of((double)l - (double)m, c, s.table);
  }
  // Puts v at slot[rank] of every block.
  template <typename V>
  __device__ __forceinline__ void tell(V* slot, V v) {
    if (tid < blocks) *cluster.map_shared_rank(slot + rank, tid) = v;
  }
  // Sum over the block, in every thread.
  __device__ __forceinline__ double block_sum(double v) {
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) s.red[warp] = v;
    __syncthreads();
    double sum = 0;
#pragma unroll
    for (int w = 0; w < SMP_WARPS; ++w) sum += s.red[w];
    return sum;
  }
  // Inclusive sum of v over the block's threads.
  __device__ __forceinline__ double block_scan(double v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    __syncthreads();
    if (lane == 31) s.red[warp] = v;
    __syncthreads();
    double base = 0;
    for (int w = 0; w < warp; ++w) base += s.red[w];
    return base + v;
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
  // fn(place, with, weight) for each of the listed tokens (in rank 0), `with` being
  // the weights of those at its place and above. Several threads share one where
  // the list is short.
  template <class Fn>
  __device__ __forceinline__ void pairs(int members, Fn fn) {
    const int share = members <= SMP_THREADS / 8 ? 8 : members <= SMP_THREADS / 4 ? 4 : members <= SMP_THREADS / 2 ? 2 : 1;
    for (int i0 = 0; i0 < members; i0 += SMP_THREADS / share) {
      const int i = i0 + tid / share, part = tid % share;
      const uint64_t o = i < members ? s.comp[i] : 0;
      uint64_t with = 0;
      for (int j = part; j < members; j += share)
        if (s.comp[j] >= o) with += s.weight[j];
      for (int w = 1; w < share; w <<= 1) with += __shfl_xor_sync(0xffffffffu, (unsigned long long)with, w);
      if (i < members && part == 0) fn(o, with, s.weight[i]);
    }
  }
  // The least place among those of `bin` (and at or past `from`) so that `measure`
  // of them and all above reaches `want`, by halving the range of places: for bins
  // of more tokens than a list holds. The blocks take the same steps.
  template <class Measure>
  __device__ uint64_t halve(int bin, uint64_t from, double want, Measure measure) {
    uint64_t lo = ~0ull, hi = 0;
    each([&](float l, int i) {
      const uint64_t o = order_of(l, i);
      if (bin_of(l) == bin && o >= from) {
        lo = min(lo, o);
        hi = max(hi, o);
      }
    });
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      lo = min(lo, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)lo, o));
      hi = max(hi, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)hi, o));
    }
    uint64_t* ends = s.comp + SMP_LIST - 2 * SMP_WARPS;
    __syncthreads();
    if (lane == 0) {
      ends[2 * warp] = lo;
      ends[2 * warp + 1] = hi;
    }
    __syncthreads();
    for (int w = 0; w < SMP_WARPS; ++w) {
      lo = min(lo, ends[2 * w]);
      hi = max(hi, ends[2 * w + 1]);
    }
    if (tid < blocks) {
      uint64_t* to = cluster.map_shared_rank(&s.span[rank][0], tid);
      to[0] = lo;
      to[1] = hi;
    }
    cluster.sync();
    for (int b = 0; b < blocks; ++b) {
      lo = min(lo, s.span[b][0]);
      hi = max(hi, s.span[b][1]);
    }
    // measure(>= lo) reaches `want` (or rounding says that nothing does: all).
    for (int turn = 0; lo < hi; ++turn) {
      const uint64_t mid = lo + (hi - lo + 1) / 2;
      double sum = 0;
      each([&](float l, int i) {
        const uint64_t o = order_of(l, i);
        if (bin_of(l) == bin && o >= from && o >= mid) sum += measure(l);
      });
      sum = block_sum(sum);
      tell(s.part[turn & 1][0], sum);
      cluster.sync();
      double all = 0;
      for (int b = 0; b < blocks; ++b) all += s.part[turn & 1][0][b];
      if (all >= want) lo = mid;
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
  SampleRow<T> x{a, s, reinterpret_cast<T*>(smp_raw + sizeof(SampleShared)), chunk, rank * chunk, cluster, rank, blocks,
                 tid, warp, lane};

  // ---- the row into shared memory, its maximum and least value -------------------------
  const float temperature = a.temperature ? a.temperature[row] : 1.f;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.f;
  const double p = top_p;
  const double least = a.min_p && a.min_p[row] > 0.f ? fmin(1.0, (double)a.min_p[row]) : 0.0;
  const bool by_k = k > 0 && k < a.n_vocab, by_p = top_p < 1.f, greedy = !(temperature > 0.f);
  for (int i = tid; i < SMP_BINS; i += SMP_THREADS) s.bins[i] = 0;
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
  float* red_f = reinterpret_cast<float*>(s.red);
  if (lane == 0) {
    red_f[2 * warp] = top;
    red_f[2 * warp + 1] = low;
  }
  __syncthreads();
  for (int w = 0; w < SMP_WARPS; ++w) {
    top = fmaxf(top, red_f[2 * w]);
    low = fminf(low, red_f[2 * w + 1]);
  }
  x.tell(s.top, top);
  x.tell(s.low, low);
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
    cluster.sync();
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
    x.each([&](float l, int i) {
      if (l == top) first = min(first, i);
    });
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s.red_i[warp] = first;
    __syncthreads();
    for (int w = 0; w < SMP_WARPS; ++w) first = min(first, s.red_i[w]);
    x.tell(s.first, first);
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

  // ---- the histogram ------------------------------------------------------------------------
  uint64_t cut = 0;  // kept: the places from it on
  double mine = 0;   // the warp's stretch of what is kept, this lane's share
  uint32_t count[4];  // of bins 4 tid ..
  if (by_k || by_p) {
    // What is below (1 - p) / n_vocab of the first adds up to less than 1 - p of
    // all: top-p alone never reaches it. (A little further for roundings.)
    const float reach =
        by_k ? INFINITY : temperature * (logf((float)a.n_vocab) - logf(fmaxf(1.f - top_p, 1e-7f)) + 0.01f);
    const int seg = chunk / SMP_WARPS;
    for (int i = warp * seg + 4 * lane; i < (warp + 1) * seg; i += 128) {
      float v[4];
      load4(x.logits + i, v);
      int b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = top - v[e] <= reach ? x.bin_of(v[e]) : -1;
      // (Equal logits over a whole warp are added at once.)
      const int b0 = __shfl_sync(0xffffffffu, b[0], 0);
      if (__all_sync(0xffffffffu, b[0] == b0 && b[1] == b0 && b[2] == b0 && b[3] == b0)) {
        if (lane == 0 && b0 >= 0) atomicAdd(&s.bins[b0], 128u);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (b[e] >= 0) atomicAdd(&s.bins[b[e]], 1u);
      }
    }
    cluster.sync();
#pragma unroll
    for (int e = 0; e < 4; ++e) count[e] = 0;
    for (int b = 0; b < blocks; ++b) {
      const uint4 y = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&s.bins[4 * tid], (rank + b) % blocks));
      count[0] += y.x;
      count[1] += y.y;
      count[2] += y.z;
      count[3] += y.w;
    }
  }

  // ---- top-k: the place of the k-th --------------------------------------------------------------
  if (by_k) {
    // (Whole numbers below 2^53.)
    const double own = (double)count[0] + count[1] + count[2] + count[3];
    double before = x.block_scan(own) - own;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (before < k && before + count[e] >= k) {
        s.found_bin = 4 * tid + e;
        s.found_above = (int)before;
      }
      before += count[e];
    }
    __syncthreads();
    const int bin = s.found_bin, rest = k - s.found_above;
    x.each([&](float l, int i) { x.list(x.bin_of(l) == bin, 0, order_of(l, i), 1.0 / SMP_UNIT); });
    cluster.sync();
    const int members = *cluster.map_shared_rank(&s.listed[0], 0);
    if (members <= SMP_LIST) {
      if (rank == 0) {
        x.pairs(members, [&](uint64_t o, uint64_t with, uint64_t) {
          if (with == (uint64_t)rest)
            for (int b = 0; b < blocks; ++b) *cluster.map_shared_rank(&s.cut, b) = o;
        });
      }
      cluster.sync();
      cut = s.cut;
    } else {
      cut = x.halve(bin, 0, rest, [](float) { return 1.0; });
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int b = 4 * tid + e;
      count[e] = b < bin ? count[e] : b == bin ? rest : 0;
    }
  }

  // ---- weights: sums of what is kept, and the place at which top-p ends -----------------------------
  const int seg = chunk / SMP_WARPS;
  if (by_p) {
    // Sums of the bins as their counts have them, from their middles.
    double est[4], own = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      est[e] = count[e] ? (double)count[e] * exp2f(-(4 * tid + e + 0.5f) / x.scale * x.c32) : 0.0;
      own += est[e];
    }
    const double upto = x.block_scan(own);  // inclusive
    const double whole = x.block_sum(own);
    double target = p * whole, fix = 0;
    int bin = 0, from = 0, to = SMP_BINS - 1;
    for (int turn = 0;; ++turn) {
      // The first bin at whose end the sum reaches the target, of those of from ..
      // to that hold anything; the last of them if none does.
      __syncthreads();
      if (tid == 0) {
        s.found_bin = INT_MAX;
        s.last_bin = -1;
      }
      __syncthreads();
      double run = upto - own + fix;
      int first_here = INT_MAX, last_here = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        run += est[e];
        const int b = 4 * tid + e;
        if (count[e] && b >= from && b <= to) {
          last_here = b;
          if (run >= target && first_here == INT_MAX) first_here = b;
        }
      }
      if (first_here != INT_MAX) atomicMin(&s.found_bin, first_here);
      if (last_here >= 0) atomicMax(&s.last_bin, last_here);
      __syncthreads();
      bin = s.found_bin != INT_MAX ? s.found_bin : s.last_bin >= 0 ? s.last_bin : bin;
      double all = 0, above = 0, in = 0;
      mine = 0;
      const auto pass = [&](auto bounded) {
        x.each([&](float l, int i) {
          const uint64_t o = order_of(l, i);
          const bool kept = !decltype(bounded)::value || o >= cut;
          const double w = kept ? x.weight(l) : 0.0;
          const int b = x.bin_of(l);
          all += w;
          if (b < bin) {
            above += w;
            if (w >= least) mine += w;
          }
          const bool here = b == bin && kept;
          if (here) in += w;
          x.list(here, 1 + turn, o, w);
        });
      };
      if (by_k) pass(std::true_type{});
      else pass(std::false_type{});
      mine = warp_sum(mine);
      if (lane == 0) *cluster.map_shared_rank(&s.warp_sum[rank * SMP_WARPS + warp], 0) = mine;
      double sums[3] = {x.block_sum(all), x.block_sum(above), x.block_sum(in)};
#pragma unroll
      for (int y = 0; y < 3; ++y) x.tell(s.part[turn & 1][y], sums[y]);
      cluster.sync();
#pragma unroll
      for (int y = 0; y < 3; ++y) {
        sums[y] = 0;
        for (int b = 0; b < blocks; ++b) sums[y] += s.part[turn & 1][y][b];
      }
      target = p * sums[0];
      above = sums[1];
      // Not the bin: another one that holds anything, by the counts again and what
      // is known of this one. (None: rounding.)
      const bool high = !(above < target), short_of = above + sums[2] < target;
      if ((high || short_of) && turn + 1 < SMP_TRIES) {
        const int was_from = from, was_to = to;
        if (high) to = bin - 1;
        else from = bin + 1;
        bool other = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) other |= count[e] && 4 * tid + e >= from && 4 * tid + e <= to;
        if (!__syncthreads_or(other)) {
          from = was_from;
          to = was_to;
        } else {
          // `above` is the sum up to the bin's beginning.
          if (tid == bin / 4) {
            double run_to = upto - own;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (e < bin % 4) run_to += est[e];
            s.red[0] = above - run_to;
          }
          __syncthreads();
          fix = s.red[0];
          continue;
        }
      }
      const int members = *cluster.map_shared_rank(&s.listed[1 + turn], 0);
      if (members <= SMP_LIST) {
        if (rank == 0) {
          // In whole units: the order of the list does not matter.
          if (tid == 0) {
            s.best = 0;
            s.least = ~0ull;
          }
          if (tid < blocks * SMP_WARPS) s.add[tid] = 0;
          __syncthreads();
          const double need = (target - above) * SMP_UNIT;
          x.pairs(members, [&](uint64_t o, uint64_t with, uint64_t) {
            atomicMin((unsigned long long*)&s.least, (unsigned long long)o);
            if ((double)with >= need) atomicMax((unsigned long long*)&s.best, (unsigned long long)o);
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
          if (tid < blocks * SMP_WARPS) s.warp_sum[tid] += (double)s.add[tid] / SMP_UNIT;
          __syncthreads();
        }
      } else {
        cut = max(cut, x.halve(bin, cut, target - above, [&](float l) { return x.weight(l); }));
        double add = 0;
        x.each([&](float l, int i) {
          if (x.bin_of(l) == bin && order_of(l, i) >= cut) {
            const double w = x.weight(l);
            if (w >= least) add += w;
          }
        });
        add = warp_sum(add);
        if (lane == 0) *cluster.map_shared_rank(&s.warp_sum[rank * SMP_WARPS + warp], 0) = mine + add;
        cluster.sync();
      }
      break;
    }
  } else {
    x.each([&](float l, int i) {
      if (order_of(l, i) >= cut) {
        const double w = x.weight(l);
        if (w >= least) mine += w;
      }
    });
    mine = warp_sum(mine);
    if (lane == 0) *cluster.map_shared_rank(&s.warp_sum[rank * SMP_WARPS + warp], 0) = mine;
    cluster.sync();
  }

  // ---- the stretch that holds the token, then the token ------------------------------------------------
  if (rank == 0 && warp == 0) {
    constexpr int PER = SMP_CLUSTER * SMP_WARPS / 32;
    double v[PER], own = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      v[e] = PER * lane + e < blocks * SMP_WARPS ? s.warp_sum[PER * lane + e] : 0.0;
      own += v[e];
    }
    double upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const double total = __shfl_sync(0xffffffffu, upto, 31);
    const float u = a.u[row];
    const double want = (double)fminf(u > 0.f ? u : 0.f, 0x1.fffffep-1f) * total;
    // The first stretch past whose end the sum exceeds it; if rounding leaves none,
    // the last that holds anything.
    int at = INT_MAX, last = -1;
    double run = upto - own, left = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      if (v[e] > 0) {
        last = PER * lane + e;
        if (at == INT_MAX && run + v[e] > want) {
          at = last;
          left = want - run;
        }
      }
      run += v[e];
    }
    const int first = __reduce_min_sync(0xffffffffu, at);
    last = __reduce_max_sync(0xffffffffu, last);
    if (first == INT_MAX) left = INFINITY;
    else left = __shfl_sync(0xffffffffu, left, first / PER);
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
    double upto = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
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
