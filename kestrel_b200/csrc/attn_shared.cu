// Attention of one new token per sequence where groups of sequences begin with the
// same pages: what a group has in common is read and computed once for all of it.
//
// The softmax over a sequence's positions splits into that over the common prefix
// and that over its own rest: with maxima m, sums l and results o of both,
//   out = (l_1 2^(m_1 - m) o_1 + l_2 2^(m_2 - m) o_2) / (l_1 2^(m_1 - m) + l_2 2^(m_2 - m)).
// The queries of a group against its prefix are a matrix product of many rows, so
// the prompt kernel computes them on the tensor cores, split over the prefix where
// there are few (attn_prompt.cu, SHARED), and the decode kernel streams the rest
// (attn_decode.cu, SHARED), beside it where SMs are free. This file looks up before
// what is common: the leading pages that the tables of all of a group's sequences
// name alike, and that every one of them goes on behind. Nothing is taken on trust,
// so the result is that of kc_attn_decode_dev whatever the groups are. And it joins
// the parts, a warp per head of an entry. (Joined by the decode kernel's blocks at
// the end of each sequence, one read after the other, 64 entries at 32768 positions
// took 145 us.)
//
// Measured (B200, us a call; what has to be read at 6559 GB/s; each sequence by
// itself), heads of 128: 32 samples of a prompt of 4001, 32 and 4 heads, f32 queries:
// 41, 5.6, 47; 4 groups of 32 at 6000, 32 and 8, bf16: 142, 98, 407; 64 at 32768, 32
// and 4, f16: 93, 21, 485. The first and last are the steps of a chain: the plan 9, the
// prefixes' way to their first scores 9, their products, the join 7; the second is
// bound by what the own parts read, 5.0 TB/s beside the prefixes.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "kv.h"
#include "kv_dev.cuh"

namespace kc {

constexpr int PREP_THREADS = 128;
constexpr int FEW = 8;  // entries of a group that one lane looks through
constexpr int SHARED_SPLITS = 31;  // (a lane each in the join, and one for the own part)
constexpr size_t SHARED_PART_BYTES = (size_t)24 << 20;

size_t attn_shared_part_bytes() { return SHARED_PART_BYTES; }
int attn_shared_counts() { return 1; }

// What the two kernels take, in us, as measured on a B200: until their first
// products and after their last, for a step of 128 (64) positions of a row tile, and
// by the bytes that an SM, and all of them, take in.
constexpr float PREFIX_FIXED = 9.f, ITEM_FIXED = 6.f, PREFIX_STEP = 1.6f, PREFIX_STEP_F32 = 1.8f;
constexpr float OWN_FIXED = 16.f, DECODE_FIXED = 9.f, PREP_AND_JOIN = 12.f, NEXT_JOIN = 6.f;
constexpr float BESIDE_BYTES = 2.8e4f, SM_BYTES = 4.2e4f, ALL_BYTES = 5.8e6f, SEEN_BYTES = 8.5e6f;  // (of pages that L2 has seen before)

// The plan, by one warp: a lane per number of SMs that the prefixes get, the last
// one for all SMs to both in turn. False: not shared it takes no longer.
// (Whole numbers: the same plan whichever warp adds its sums first.)
typedef unsigned long long plan_sum;
struct PlanSums {
  int units;       // row tiles of the prefixes, over the heads
  int longest;     // tiles of the longest prefix
  plan_sum steps;  // tiles of all units
  plan_sum prefix, own, all;  // positions: of the prefixes, the own parts, and not shared
};
// `launches` that the entries take (as many at a time as the workspace has
// room for), each with its own start, join and rounds.
__device__ __forceinline__ bool shared_plan(const PlanSums& t, const KvView& c, bool f32, int sms, int most, int launches,
                                            int32_t* plan) {
  const int lane = threadIdx.x & 31;
  const float bytes = 4.f * c.hd * c.nkv, of_prefix = t.prefix, of_own = t.own;
  const bool turns = lane == 31;
  const int g = turns ? sms : max(1, (lane + 1) * sms / 32), rest = turns ? sms : sms - g;
  // A step alone, or with its part of the memory rate, which row tiles that read the
  // same positions share.
  float step = f32 ? PREFIX_STEP_F32 : PREFIX_STEP;
  if (!turns) step = fmaxf(step, __fdividef(of_prefix * bytes, (float)t.steps * BESIDE_BYTES));
  // Items (units by parts) go over the g SMs in rounds.
  int splits = 1;
  float prefix = INFINITY;
  const float times = launches, units = t.units, longest = t.longest, per = __fdividef(1.f, g * times);
  for (int p = 1; p <= min(most, max(1, t.longest / 2)); ++p) {
    const float took = times * (PREFIX_FIXED + ceilf(units * p * per - 1e-3f) * (ITEM_FIXED + step * ceilf(__fdividef(longest, (float)p))));
    if (took < prefix) {
      prefix = took;
      splits = p;
    }
  }
  prefix = fmaxf(prefix, times * PREFIX_FIXED + of_prefix * bytes / ALL_BYTES);
  // (Side by side they share the memory rate.)
  const float own = times * OWN_FIXED + fmaxf(of_own * bytes / (rest * SM_BYTES), (of_own + (turns ? 0.f : of_prefix)) * bytes / ALL_BYTES);
  const float both = PREP_AND_JOIN + (times - 1) * NEXT_JOIN + (turns ? prefix + own : fmaxf(prefix, own));
  const unsigned best = __reduce_min_sync(0xffffffffu, __float_as_uint(both));
  const unsigned who = __ballot_sync(0xffffffffu, __float_as_uint(both) == best);
  if (lane == __ffs(who) - 1) {
    plan[PLAN_SPLITS] = splits;
    plan[PLAN_PREFIX] = g;
    plan[PLAN_OWN] = rest;
  }
  // (Not shared, a position is read once from memory, and again from L2.)
  const float once = of_own + of_prefix, again = (float)t.all - once;
  return __uint_as_float(best) < DECODE_FIXED + once * bytes / ALL_BYTES + again * bytes / SEEN_BYTES;
}

// A block per entry: the pages that its table has in common with that of the first
// of its group that holds anything. The last block takes the least of each group.
__global__ void __launch_bounds__(PREP_THREADS) shared_prep_kernel(KvView c, const int32_t* __restrict__ seqs, int n,
                                                                   const int32_t* __restrict__ group_start,
                                                                   int n_groups, int32_t* of_entry, int32_t* of_group,
                                                                   int32_t* lead, int* done, int group, bool f32,
                                                                   int sms, int most, int launches, bool always, int32_t* plan) {
  pdl_enter();
  __shared__ int differ, last, wrong, shares, large;
  __shared__ PlanSums sums;
  const int i = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const auto seq = [&](int e) { return seqs ? seqs[e] : e; };
  const auto holds = [&](int s) { return s >= 0 && s < c.n_seq ? kv_len(c, s) : 0; };
  if (tid == 0) {
    wrong = large = 0;
    sums = PlanSums{};
  }
  {
    const int s = seq(i), len = holds(s), g = kv_row_owner(group_start, n_groups, i);
    int pages = 0;
    if (g >= 0 && len > 0) {
      int first = max(group_start[g], 0);
      while (first < i && holds(seq(first)) == 0) ++first;
      const int s0 = seq(first);
      pages = (min(len, holds(s0)) - 1) >> c.page_log2;  // (a position behind them is left)
      if (tid == 0) differ = pages;
      __syncthreads();
      const int32_t *x = c.table + (int64_t)s0 * c.max_pages, *y = c.table + (int64_t)s * c.max_pages;
      for (int p0 = 0; p0 < pages; p0 += 8 * PREP_THREADS) {
        int at = INT_MAX;
#pragma unroll
        for (int u = 7; u >= 0; --u) {
          const int p = p0 + u * PREP_THREADS + tid;
          if (p < pages) {
            const int a = x[p], b = y[p];
            if (a != b || a < 0 || a >= c.n_pages) at = p;
          }
        }
        if (at != INT_MAX) atomicMin(&differ, at);
        if (__syncthreads_or(at != INT_MAX)) break;
      }
      __syncthreads();
      pages = differ;
    }
    if (tid == 0) of_entry[i] = g < 0 ? 0 : len > 0 ? pages << c.page_log2 : -1;
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) last = atomicAdd(done, 1) == n - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (tid == 0) {
    *done = 0;
    plan[PLAN_SPLITS] = most;
    plan[PLAN_PREFIX] = plan[PLAN_OWN] = sms;
  }
  // Groups that do not ascend within the entries: nothing is common.
  for (int g = tid; g <= n_groups; g += PREP_THREADS) {
    const int at = group_start[g];
    if (at < (g ? group_start[g - 1] : 0) || at > n) wrong = 1;
  }
  __syncthreads();
  if (wrong) {
    if (tid == 0) report(c.status, KC_ERR_ARG | (W_KV_ROWS << 8));
    for (int e = tid; e < n; e += PREP_THREADS) of_entry[e] = 0;
    for (int g = tid; g < n_groups; g += PREP_THREADS) of_group[g] = 0;
    return;
  }
  // What group g's entries lo .. hi - 1 have in common, of those that hold anything
  // (`held` of them, the first `first`).
  const auto settle = [&](int g, int lo, int hi, int least, int first, int held) {
    const int both = held > 1 ? least : 0;
    of_group[g] = both;
    lead[g] = held ? seq(first) : 0;
    if (both) {
      const int units = (int)(((int64_t)(hi - lo) * group + 127) / 128) * c.nkv, nt = (both + shared_tile(c.hd) - 1) / shared_tile(c.hd);
      atomicAdd(&sums.units, units);
      atomicMax(&sums.longest, nt);
      atomicAdd(&sums.steps, (plan_sum)units * nt);
      atomicAdd(&sums.prefix, (plan_sum)both);
    }
    return both;
  };
  const auto by_warp = [&](int g, int lo, int hi) {
    int least = INT_MAX, first = INT_MAX, held = 0;
    for (int e = lo + lane; e < hi; e += 32) {
      const int of = __ldcg(of_entry + e);
      if (of < 0) continue;
      least = min(least, of);
      first = min(first, e);
      ++held;
    }
    least = __reduce_min_sync(0xffffffffu, least);
    first = __reduce_min_sync(0xffffffffu, first);
    held = __reduce_add_sync(0xffffffffu, held);
    const int both = held > 1 ? least : 0;
    for (int e = lo + lane; e < hi; e += 32) of_entry[e] = __ldcg(of_entry + e) < 0 ? 0 : both;
    if (lane == 0) settle(g, lo, hi, least, first, held);
  };
  if (n_groups <= 32) {
    for (int g = warp; g < n_groups; g += PREP_THREADS / 32) by_warp(g, group_start[g], group_start[g + 1]);
  } else {
    // Many groups: the small ones a lane each, since a warp's look-ups wait for each
    // other; the others a warp each. (2000 entries in groups of their own: a call of
    // 516 us so, of 915 with a warp for each.)
    for (int g = tid; g < n_groups; g += PREP_THREADS) {
      const int lo = group_start[g], hi = group_start[g + 1];
      if (hi - lo > FEW) {
        large = 1;
        continue;
      }
      int of[FEW], least = INT_MAX, first = INT_MAX, held = 0;
#pragma unroll
      for (int k = 0; k < FEW; ++k) of[k] = lo + k < hi ? __ldcg(of_entry + lo + k) : -1;
#pragma unroll
      for (int k = 0; k < FEW; ++k)
        if (of[k] >= 0) {
          least = min(least, of[k]);
          first = min(first, lo + k);
          ++held;
        }
      const int both = settle(g, lo, hi, least, first, held);
#pragma unroll
      for (int k = 0; k < FEW; ++k)
        if (lo + k < hi) of_entry[lo + k] = of[k] < 0 ? 0 : both;
    }
    __syncthreads();
    for (int g0 = 0, ones = 0; large && g0 < n_groups; g0 += 32) {
      const int g = g0 + lane, lo = g < n_groups ? group_start[g] : 0, hi = g < n_groups ? group_start[g + 1] : 0;
      for (unsigned left = __ballot_sync(0xffffffffu, hi - lo > FEW); left; left &= left - 1) {
        const int who = __ffs(left) - 1, its_lo = __shfl_sync(0xffffffffu, lo, who), its_hi = __shfl_sync(0xffffffffu, hi, who);
        if (ones++ % (PREP_THREADS / 32) == warp) by_warp(g0 + who, its_lo, its_hi);
      }
    }
  }
  __syncthreads();
  plan_sum own = 0, all = 0;
#pragma unroll 4
  for (int e = tid; e < n; e += PREP_THREADS) {
    const int len = holds(seq(e));
    own += len - __ldcg(of_entry + e);
    all += len;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    own += __shfl_xor_sync(0xffffffffu, own, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if (lane == 0) {
    atomicAdd(&sums.own, own);
    atomicAdd(&sums.all, all);
  }
  __syncthreads();
  if (warp == 0) {
    const bool yes = sums.units > 0 && shared_plan(sums, c, f32, sms, most, launches, plan);
    if (lane == 0) shares = yes || always;
  }
  __syncthreads();
  if (shares) return;
  for (int e = tid; e < n; e += PREP_THREADS) of_entry[e] = 0;
  for (int g = tid; g < n_groups; g += PREP_THREADS) of_group[g] = 0;
  if (tid == 0) {
    plan[PLAN_SPLITS] = plan[PLAN_PREFIX] = 1;
    plan[PLAN_OWN] = sms;
  }
}

// A warp per (entry, head): the parts' maxima and sums a lane each, then their
// values, 16 bytes a lane, eight parts under way. (What it waits for is the decode
// kernel alone, the launch before it; that the prefixes' kernel is through too rests on
// every block of the decode kernel waiting for it before it leaves.)
template <typename T>
__global__ void __launch_bounds__(PREP_THREADS) shared_join_kernel(const AttnArgs a, const SharedArgs sh) {
  pdl_enter();
  const KvView& c = a.c;
  const int lane = threadIdx.x & 31, ld = shared_row_floats(c.hd), n = sh.e1 - sh.e0;
  const int64_t row = (int64_t)blockIdx.x * (PREP_THREADS / 32) + (threadIdx.x >> 5);
  if (row >= (int64_t)n * a.nh) return;
  const int i = (int)(row / a.nh), s = a.seqs ? a.seqs[sh.e0 + i] : sh.e0 + i;
  if (s < 0 || s >= c.n_seq) return;
  const int both = sh.of_entry[sh.e0 + i], splits = both > 0 ? shared_splits(both, c.hd, sh.plan[PLAN_SPLITS]) : 0;
  const int64_t step = (int64_t)n * a.nh * ld;
  // Lane p: part p of the prefix; lane `splits`: the own one.
  const float* mine = sh.part + row * ld + (lane < splits ? lane : sh.splits) * step;
  // (The first values are asked for beside the maxima and sums.)
  const auto ask = [&](int p0, int y, float4(&u)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (p0 + k <= splits && y < c.hd)
        u[k] = __ldcg(reinterpret_cast<const float4*>(sh.part + row * ld + (p0 + k < splits ? p0 + k : sh.splits) * step + y));
  };
  float4 u[8];
  ask(0, 4 * lane, u);
  const float2 ml = lane <= splits ? __ldcg(reinterpret_cast<const float2*>(mine + ld - 8)) : make_float2(-INFINITY, 0.f);
  float top = ml.y == 0.f ? -INFINITY : ml.x;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float share = ml.y == 0.f ? 0.f : exp2f(ml.x - (top == -INFINITY ? 0.f : top)) * ml.y, sum = share;
  const unsigned some = __ballot_sync(0xffffffffu, ml.y != 0.f);  // parts that saw a position
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  share = sum == 0.f ? 0.f : __fdiv_rn(share, sum);
  T* out = static_cast<T*>(a.out) + (int64_t)(sh.e0 + i) * a.out_stride + (row - (int64_t)i * a.nh) * c.hd;
  for (int y0 = 0; y0 < c.hd; y0 += 128) {
    const int y = y0 + 4 * lane;
    const bool mine_y = y < c.hd;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = 0; p0 <= splits; p0 += 8) {
      if (y0 || p0) ask(p0, y, u);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float w = __shfl_sync(0xffffffffu, share, min(p0 + k, 31));
        // (What is infinite stays so, however little its part weighs.)
        const auto of = [w](float x) { return fabsf(x) < INFINITY ? w : 1.f; };
        if (p0 + k <= splits && mine_y && (some >> (p0 + k) & 1)) {
          v.x = __fmaf_rn(of(u[k].x), u[k].x, v.x);
          v.y = __fmaf_rn(of(u[k].y), u[k].y, v.y);
          v.z = __fmaf_rn(of(u[k].z), u[k].z, v.z);
          v.w = __fmaf_rn(of(u[k].w), u[k].w, v.w);
        }
      }
    }
    if (!mine_y) continue;
    out[y] = (T)v.x;
    out[y + 1] = (T)v.y;
    out[y + 2] = (T)v.z;
    out[y + 3] = (T)v.w;
  }
}

int launch_attn_shared(const AttnArgs& a, SharedArgs sh, const KvMaps& rows16, const KvMaps& tiles, float* part,
                       int* count, float* shared_part, cudaStream_t st) {
  const KvView& c = a.c;
  const int64_t row = (int64_t)a.nh * shared_row_floats(c.hd), room = (int64_t)(SHARED_PART_BYTES / sizeof(float)) / row;
  // Where the entries cannot hold so much that reading it takes longer than a plan, a
  // prefix kernel's start and a join, there is nothing to plan. (4 at 300, 8 and 2
  // heads of 64: 11.6 us, planned and shared 25.)
  const double most = 4.0 * c.hd * c.nkv * a.n * std::min((int64_t)c.max_pages * c.page, (int64_t)c.n_pages * c.page);
  const bool small = most / SEEN_BYTES < PREP_AND_JOIN + ITEM_FIXED;
  if (a.n < 2 || sh.n_groups < 1 || room < 4 || (small && !sh.always))
    return launch_attn_decode(a, rows16, part, count, st);
  // Few row tiles: the prefixes are split over the SMs, within the workspace.
  const int64_t group = a.nh / c.nkv, units = (a.n * group + 127) / 128 * c.nkv;
  sh.splits = (int)std::max<int64_t>(1, std::min<int64_t>({num_sms() / units, SHARED_SPLITS, room / a.n - 1}));
  sh.part = shared_part;
  int* done = count + std::max(num_sms(), attn_prompt_counts());
  // As many entries at a time as the workspace has room for.
  const int step = (int)std::min<int64_t>(a.n, room / (sh.splits + 1));
  launch_k(shared_prep_kernel, a.n, PREP_THREADS, 0, st, c, a.seqs, a.n, sh.group_start, sh.n_groups, sh.of_entry,
           sh.of_group, sh.lead, done, (int)group, a.t_q == T_F32, num_sms(), sh.splits, (a.n + step - 1) / step, sh.always, sh.plan);
  const int64_t el = a.t_q == T_F32 ? 4 : 2;
  for (sh.e0 = 0; sh.e0 < a.n; sh.e0 += step) {
    sh.e1 = std::min(a.n, sh.e0 + step);
    AttnArgs p = a, own = a;
    p.seqs = nullptr;
    p.row_start = sh.group_start;
    p.n = sh.n_groups;
    p.n_rows = a.n;
    int rc = launch_attn_prefix(p, sh, tiles, part, count, st);
    if (rc != KC_OK) return rc;
    own.seqs = a.seqs ? a.seqs + sh.e0 : nullptr;
    own.n = own.n_rows = sh.e1 - sh.e0;
    own.q = static_cast<const uint8_t*>(a.q) + sh.e0 * a.q_stride * el;
    own.out = static_cast<uint8_t*>(a.out) + sh.e0 * a.out_stride * el;
    rc = launch_attn_own(own, sh, rows16, part, count, st);
    if (rc != KC_OK) return rc;
    const int64_t rows = (int64_t)own.n * a.nh;
    const int grid = (int)((rows + PREP_THREADS / 32 - 1) / (PREP_THREADS / 32));
    if (a.t_q == T_F32) launch_k(shared_join_kernel<float>, grid, PREP_THREADS, 0, st, a, sh);
    else if (a.t_q == T_F16) launch_k(shared_join_kernel<__half>, grid, PREP_THREADS, 0, st, a, sh);
    else launch_k(shared_join_kernel<__nv_bfloat16>, grid, PREP_THREADS, 0, st, a, sh);
  }
  return KC_OK;
}

}  // namespace kc
