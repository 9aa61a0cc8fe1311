// Attention of prompt rows over the paged key-value cache on the tensor cores.
//
// For query row r of a sequence with c rows and len positions, i = len - c + r
// and over its visible positions j (j <= i, and j > i - window or j < sinks):
//   s_j = scale * q . k_j,  m = max s_j,  p_j = exp(s_j - m),
//   out = sum p_j v_j / sum p_j;  zeros where nothing is visible.
// One pass over the positions with the running maximum and sum of each row.
//
// The rows of a key-value head (tokens outermost, then the heads of its group)
// are cut into tiles of 128, the M of an MMA, so that the group shares every
// key and value. Positions pass in tiles of BN. One block per SM takes items
// (row tiles of a head) as it comes to them, those that see most first (in the
// list's order where it has more than 32 entries). Roles:
//   softmax warps  four per stream, a thread per row: scores from TMEM, the
//                  mask where the tile needs it, weights back to TMEM as the
//                  16-bit A operand of the second product. The accumulator is
//                  rescaled only when a row's weights have grown too large.
//   a TMA warp     K and V tiles, a box per page, through one ring.
//   an MMA warp    S = Q K^T (both in shared memory), O += P V (P in TMEM).
//   two more       find the next item and bring its queries, while the others
//                  are at the last one.
// Two streams take turns on the tensor cores, so that one's exponentials run
// beside the other's products (the two of a tile, 128 x 128 x 128 each, take as
// long as its 16384 exponentials, 1024 cycles): either two row tiles over the same positions, or
// one row tile whose position tiles alternate, joined at the end. With fewer
// items than SMs their positions are split further, over several blocks; the
// block that finishes last joins the parts in their order.
//
// f32 queries are carried by two f16 operands (value and rest), and so are
// their weights: twice the products, f32-grade results over a 16-bit cache (at
// most 8e-6 off however long it is, 4e-6 for values of mean 0, where f32
// arithmetic is 1e-6: the tensor cores cut their sums off, see KEEP). Weights
// under 16-bit queries are rounded to the cache's type; their sum is not. (Those of
// shared prefixes have their rests too: what is shared goes by the time that it is
// expected to take, and should not show in the results. 64 entries at 32768 positions,
// 32 and 4 heads of 128, f16: 78 us without, 91 so, 2.9e-4 and 2.1e-4 off.)
//
// Measured on a B200, 32 query and 4 key-value heads of 128, f16: 8192 rows from
// the first (550 GFLOP) in 533 us kept up (1.03 PFLOP/s, under the power cap,
// where the measured matrix rate is 1.43); two prompts of 6001 and 7400 rows with 8
// heads under a window of 2048, bf16 (422 GFLOP of visible pairs) in 476 us. At 4096 rows the tensor pipe is
// busy for 52% of the active cycles, and so is the unit of the exponentials: a
// stream's tile takes its warps about 2600 cycles beside the other stream's,
// and the two products and their hand-overs 1550 a step. Tried and not kept: a
// share of the exponentials as cubics on the FMA pipes (a quarter: 4% slower),
// the MMA warp's code per stream or run by the whole warp (5% slower).
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "attn_dev.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv.h"
#include "kv_dev.cuh"
#include "tc_dev.cuh"

namespace kc {

constexpr int PM = 128;  // rows of a tile
constexpr int P_STAGES_MAX = 8;
constexpr int P_SPLITS_MAX = 8;  // blocks an item's positions are split over, at most
constexpr int KEPT_COLUMNS = 264;  // of both streams, or one, and their maxima
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
static_assert(2 * kSoftmaxRegs + kOtherRegs == 3 * 168, "within the registers of the launch");

template <typename TQ, int NB, bool TWO, bool SHARED>
struct PromptShape {
  static constexpr bool kSplit = sizeof(TQ) == 4;   // queries of two operands
  static constexpr bool kRests = kSplit || SHARED;  // weights of two
  static constexpr int HD = 64 * NB;               // padded head size
  static constexpr int BN = NB <= 2 ? 128 : 64;    // positions of a tile
  static constexpr int NS = NB <= 2 ? 2 : 1;       // streams
  static constexpr int QT = TWO ? 2 : 1;           // row tiles
  static constexpr int QB = PM * 128 * NB;         // bytes of a query operand
  static constexpr int Q_ALL = QT * (kSplit ? 2 : 1) * QB;
  static constexpr int KV = BN * 128 * NB;         // bytes of a K or V tile
  static constexpr int CAP = (NB <= 2 ? 221 : 225) * 1024;  // beside up to 6 (1.5) KB of static arrays
  static constexpr int FIT = (CAP - 1024 - Q_ALL) / KV;
  static constexpr int ST = FIT < P_STAGES_MAX ? FIT : P_STAGES_MAX;
  static constexpr int SMEM = Q_ALL + ST * KV + 1024;
  // Two streams: three warpgroups of 168 registers a thread at launch, of which
  // the third (loads, MMAs) gives the softmax warps 32 a thread.
  static constexpr int THREADS = 128 * NS + 128;
  // TMEM columns. Two streams with 16-bit weights share the scores' columns:
  // they are free again as soon as they are in registers, so that the next
  // scores are there when a softmax ends and its warps never wait for their own
  // products (8192 rows of 32 heads: 478 us with scores and weights in the same
  // columns, 464 so). Weights of two operands leave no room for that.
  static constexpr bool kShared = NS == 2 && !kRests;
  static constexpr int T_S = kShared ? 0 : 128;    // scores of stream w at T_S w
  static constexpr int T_P = kShared ? 128 : 0;    // its weights at T_P + (kShared ? 64 : 128) w
  static constexpr int T_PW = kShared ? 64 : 128;
  static constexpr int T_O = 256;                  // its accumulator at T_O + HD w
  // A split item's part: per four columns the rows' values ([HD / 4][PM][4]),
  // then the rows' maxima and sums ([PM][2]).
  static constexpr int PART = PM * (HD + 2);
  // An accumulator begins anew after so many tiles, and what it held is kept in
  // memory: the tensor cores cut a sum's last bits off with every 16 positions
  // (and operand), always towards zero, about 2^-24.5 of the final sum a step when
  // nothing cancels. 1024 rows at 131072 positions, f32: 3.4e-4 off when they go
  // on adding, 8e-6 with 12 tiles (192 steps), 5.4e-6 with 8, 1.1e-5 with 16. 6 x
  // 256 rows at 300 to 4000 take 129 us without, 134, 139 and 131 so, the 1024 at
  // 131072 3.8 ms without and 4.2 with 12 or 16. Where results are rounded to 16
  // bits, 2048 steps, 1e-4.
  static constexpr int KEEP = (kSplit ? 1536 : 32768) / BN;
  // What a stream keeps: the maxima that the values count from (every fourth
  // place), then the values, as in a part.
  static constexpr int KEPT = PM * (HD + 4);
  static_assert(!TWO || kShared, "two row tiles: two streams of 16-bit weights");
  static_assert(ST >= 2 && T_O + NS * HD <= 512 && NS * (HD + 4) <= KEPT_COLUMNS, "fits");
};

// Keeps a branch's code out of the way of what runs for every tile.
__device__ __forceinline__ bool rarely(bool c) { return __builtin_expect(c, 0); }

// 16 values times f; whether any of them is NaN. (An infinity is one that the row
// sees, with a weight: beyond its mask it would be NaN, 0 times it.)
__device__ __forceinline__ bool normalise16(float (&v)[16], float f) {
  uint64_t odd = 0;  // infinite and NaN values times 0 are NaN
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    const uint64_t x = f2(v[e], v[e + 1]);
    odd = fma2(x, f2(0.f, 0.f), odd);
    const float2 y = f2(mul2(x, f2(f, f)));
    v[e] = y.x;
    v[e + 1] = y.y;
  }
  bool nan = false;
  if (rarely(f2(odd).x + f2(odd).y != 0.f)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) nan |= v[e] != v[e];
  }
  return nan;
}

// The lowest n bits (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
}

// Row f of an item: its token among the entry's rows, its head of the group.
// (x * magic) >> 16 = x / group for x < 512, group <= 128.
struct RowMap {
  int tok0, rem, group;
  uint32_t magic;
  __device__ RowMap(int row0, int g) : tok0(row0 / g), rem(row0 - row0 / g * g), group(g), magic(65536u / g + 1) {}
  __device__ int token(int f) const { return tok0 + (int)(((uint32_t)(rem + f) * magic) >> 16); }
  __device__ int64_t offset(int f, int64_t stride, int hd) const {
    const int t = token(f);
    return t * stride + (int64_t)(rem + f - (t - tok0) * group) * hd;
  }
};

// An item: the rows row0 .. row0 + rows - 1 ((token, head) pairs) of head kvh
// of entry i, over position tiles t0 .. t1-1 of those they see. Tile t begins
// at position BN * (t < head ? t : t - head + w0): `head` tiles of the first
// tokens, then those of the window.
struct Item {
  int valid, s, len, count, start, row0, rows, kvh;
  int head, w0, nt, t0, t1;
  int unit, split, splits;
  __device__ int pos(int t, int bn) const { return (t < head ? t : t - head + w0) * bn; }
};

// One row computed by a warp, 32 positions at a time: what the products cannot
// give when a value that the row does not see is not finite (0 * NaN). A lane
// takes one position's score, then eight columns of every fourth position's
// values, so that the loads of 64 columns are all under way together (32 rows
// at 8192 positions, 8 heads of 64, all of them so: 18 ms; position by position
// 219). Columns col0 .. col1-1 are written. `alive` is the time at which it last
// moved on, for those who wait for it.
// Positions `from` .. `at` (SHARED: a part of a prefix, whose maximum, in exponents
// of 2, and sum go to `state` with column 0).
template <typename TQ, typename TKV, typename TO, bool SHARED>
__device__ __noinline__ void prompt_row(const AttnArgs& a, int s, int kvh, int from, int at, const TQ* q, TO* out,
                                        int col0, int col1, float* state, volatile uint64_t* alive) {
  const KvView c = a.c;
  const int lane = threadIdx.x & 31, sub = lane & 7, lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
  const float scale = a.scale;
  float x[8], o[4][8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int u = 0; u < 8; ++u) x[u] = lane + 32 * u < c.hd ? (float)q[lane + 32 * u] : 0.f;
#pragma unroll
  for (int g = 0; g < 4; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) o[g][i] = 0.f;
  for (int j0 = SHARED ? from : 0, steps = 0; j0 <= at; j0 += 32) {
    if (j0 + 32 <= lo && j0 >= a.sinks) {
      j0 = lo / 32 * 32 - 32;
      continue;
    }
    const int j = j0 + lane;
    bool see = j <= at && (j >= lo || j < a.sinks);
    long long e = 0;
    if (see) {
      const int id = c.table[(int64_t)s * c.max_pages + (j >> c.page_log2)];
      see = id >= 0 && id < c.n_pages;
      if (see) e = ((((int64_t)a.layer * c.n_pages + id) * c.nkv + kvh) * c.page + (j & (c.page - 1))) * (int64_t)c.hd;
    }
    const unsigned seen = __ballot_sync(0xffffffffu, see);
    float t = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (64 * g < c.hd) {
        uint4 k[8];
#pragma unroll
        for (int w = 0; w < 8; ++w)
          k[w] = see && 64 * g + 8 * w < c.hd
                     ? reinterpret_cast<const uint4*>(reinterpret_cast<const TKV*>(c.k) + e)[8 * g + w]
                     : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          alignas(16) TKV y[8];
          *reinterpret_cast<uint4*>(y) = k[w];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            t = __fmaf_rn(__shfl_sync(0xffffffffu, x[2 * g + (w >> 2)], 8 * (w & 3) + i), (float)y[i], t);
        }
      }
    t = see ? t * scale : -INFINITY;
    if (__any_sync(0xffffffffu, !(t < INFINITY))) {  // a score of NaN or infinity: every result is NaN
      l = NAN;
      break;
    }
    float top = t;
#pragma unroll
    for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float mn = fmaxf(m, top), shrink = mn == -INFINITY ? 1.f : expf(m - mn);
    const float p = mn == -INFINITY ? 0.f : expf(t - mn);
    float sum = p;
#pragma unroll
    for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    m = mn;
    l = __fmaf_rn(l, shrink, sum);
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (64 * g < c.hd) {
        uint4 v[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const int from = 4 * y + (lane >> 3);
          const long long e_y = __shfl_sync(0xffffffffu, e, from);
          v[y] = seen >> from & 1 && 64 * g + 8 * sub < c.hd
                     ? reinterpret_cast<const uint4*>(reinterpret_cast<const TKV*>(c.v) + e_y)[8 * g + sub]
                     : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) o[g][i] *= shrink;
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const float p_y = __shfl_sync(0xffffffffu, p, 4 * y + (lane >> 3));
          alignas(16) TKV z[8];
          *reinterpret_cast<uint4*>(z) = v[y];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[g][i] = __fmaf_rn(p_y, (float)z[i], o[g][i]);
        }
      }
    if (!(++steps & 31) && lane == 0) *alive = globaltimer();
  }
#pragma unroll
  for (int g = 0; g < 4; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float r = o[g][i];
      r += __shfl_xor_sync(0xffffffffu, r, 8);
      r += __shfl_xor_sync(0xffffffffu, r, 16);
      const int col = 64 * g + 8 * sub + i;
      if (lane < 8 && col >= col0 && col < col1) out[col] = (TO)(l == 0.f ? 0.f : l != l ? l : __fdiv_rn(r, l));
    }
  if (SHARED && col0 == 0 && lane == 0) *reinterpret_cast<float2*>(state) = make_float2(m * 1.4426950408889634f, l);
}

// mbar_wait whose limit counts from the last time that a row computed by itself
// moved on (it takes as long as it is).
__device__ __forceinline__ bool prompt_wait(uint64_t* bar, uint32_t parity, int* status,
                                            const volatile uint64_t* alive) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity)) {
    const uint64_t now = globaltimer();
    if (now - t0 > kWaitLimitNs && (int64_t)(now - *alive) > (int64_t)kWaitLimitNs) {
      report(status, KC_ERR_TIMEOUT | (W_ATT_PROMPT << 8));
      return false;
    }
  }
  return true;
}

// A row's accumulator (hd16 columns at o_t of TMEM; reference m) and what is kept
// of it in memory (its reference, values from 4 * PM on): put there, added to it,
// or added back to the accumulator. Whole warps; out of the way of the tiles that
// do not need it.
enum { KEEP_FIRST, KEEP_ADD, KEEP_RETURN };
__device__ __noinline__ void keep_sums(uint32_t o_t, int hd16, float* kept, float m, int how) {
  const float before = how == KEEP_FIRST ? m : __ldcg(kept), shrink = before == m ? 1.f : exp2_fast(before - m);
  for (int e0 = 0; e0 < hd16; e0 += 16) {
    float4* at = reinterpret_cast<float4*>(kept + (e0 + 4) * PM);
    float4 y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = how == KEEP_FIRST ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldcg(at + e * PM);
    float o[16];
    tmem_ld16(o_t + e0, o);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e].x = __fmaf_rn(y[e].x, shrink, o[4 * e]);
      y[e].y = __fmaf_rn(y[e].y, shrink, o[4 * e + 1]);
      y[e].z = __fmaf_rn(y[e].z, shrink, o[4 * e + 2]);
      y[e].w = __fmaf_rn(y[e].w, shrink, o[4 * e + 3]);
      if (how != KEEP_RETURN) __stcg(at + e * PM, y[e]);
    }
    if (how == KEEP_RETURN) tmem_st16(o_t + e0, reinterpret_cast<const float*>(y));
  }
  if (how != KEEP_RETURN) __stcg(kept, m);
  tmem_wait_st();
}

struct PromptArgs {
  AttnArgs a;
  int splits;   // blocks an item's positions may be split over
  float* part;  // [unit][split][PART]
  float* kept;  // [block][stream][KEPT]
  int* count;   // per unit, zero between launches
  int* next;    // [2] items dealt beyond one per block, blocks done: zero between launches
  bool q_map;   // queries come by TMA
  SharedArgs sh;  // SHARED
};

// SHARED: an entry is a group of sequences, its rows one query of each; every row
// sees all positions that the group has in common, and what comes of them is left
// for the join (attn_shared.cu).
template <typename TQ, typename TKV, int NB, bool TWO, bool SHARED>
__global__ void __launch_bounds__(PromptShape<TQ, NB, TWO, SHARED>::THREADS, 1)
    attn_prompt_kernel(const PromptArgs d, const __grid_constant__ KvMaps maps, const __grid_constant__ KvMap q_map) {
  using S = PromptShape<TQ, NB, TWO, SHARED>;
  constexpr int BN = S::BN, NS = S::NS, ST = S::ST;
  constexpr bool kSplit = S::kSplit, kRests = S::kRests;
  // Weights are 2^lift for a score at the reference, so that small ones of f16
  // keep their bits; f16's range ends at 2^16, and rescaling starts from sums of
  // kMost. (Two f16 operands: rescaling starts 2^8 past the reference.)
  constexpr bool kF16 = std::is_same_v<TKV, __half>;
  constexpr float kLift = !kF16 ? 0.f : kRests ? 7.f : 3.f;
  constexpr float kMost = kF16 ? 32768.f : 1.1e9f;
  constexpr int W_TMA = 4 * NS, W_MMA = W_TMA + 1, W_AUX = W_TMA + 2;  // W_AUX: and the next
  constexpr bool kShared = S::kShared;
  // (SHARED: many rows see a prefix whole, where a prompt's last ones do; f32, four
  // groups of 9 at 50587, 32 and 4 heads of 128: 3.8e-6 off in 145 us with 12 tiles,
  // 2.3e-6 in 163 with 6, 1.7e-6 in 171 with 4.)
  constexpr int KEEP = SHARED && kSplit ? S::KEEP / 2 : S::KEEP;
  constexpr int AHEAD = NS;  // K tiles loaded before the first V
  if (threadIdx.x < 3) prefetch_map(threadIdx.x == 0 ? &maps.k : threadIdx.x == 1 ? &maps.v : &q_map);
  pdl_enter();
  extern __shared__ uint8_t prompt_raw[];
  __shared__ __align__(8) uint64_t kv_full[ST], kv_empty[ST], s_full[NS], s_free[NS], p_full[NS], pv_done[NS],
      o_empty[NS];
  __shared__ __align__(8) uint64_t q_raw, q_full, q_empty, item_full[2], item_empty[2];
  __shared__ uint32_t tmem_sh;
  __shared__ Item items[2];
  __shared__ __align__(8) uint64_t drained, join_full, part_full, last_full;
  __shared__ float factor_sh[2][S::QT][PM];  // what a row's queries were multiplied with (f32 queries)
  __shared__ float2 join_sh[2][NS][PM];      // maximum and sum of a stream's rows
  __shared__ int last_sh;
  __shared__ uint64_t alive_sh;  // (prompt_row)
  const AttnArgs& a = d.a;
  const KvView& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // SHARED: as many blocks and parts of a prefix as the device has planned.
  const int splits = SHARED ? d.sh.plan[PLAN_SPLITS] : d.splits;
  const int blocks = SHARED ? min((int)gridDim.x, d.sh.plan[PLAN_PREFIX]) : gridDim.x;
  if (SHARED && blockIdx.x >= blocks) return;
  const int group = a.nh / c.nkv;
  const int hd16 = (c.hd + 15) / 16 * 16;  // columns of the products that are computed
  const float flip = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f;  // into the queries: score factors are positive
  uint8_t* q_sm = prompt_raw + ((1024 - (smem_u32(prompt_raw) & 1023)) & 1023);
  uint8_t* ring = q_sm + S::Q_ALL;
  if (tid == 0) {
    alive_sh = 0;
    for (int i = 0; i < ST; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int w = 0; w < NS; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&p_full[w], 128);
      mbar_init(&s_free[w], 128);
      mbar_init(&pv_done[w], 1);
      mbar_init(&o_empty[w], TWO ? 128 : 128 * NS);
    }
    mbar_init(&q_raw, 1);
    mbar_init(&q_full, kSplit && d.q_map ? 4 * NS : 2);
    mbar_init(&q_empty, 1);
    mbar_init(&drained, 1);
    mbar_init(&join_full, 128 * NS);
    mbar_init(&part_full, 128 * NS);
    mbar_init(&last_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 4 * NS + 3);
    }
    fence_mbar_init();
  }
  if (warp == W_MMA) tmem_alloc(&tmem_sh, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh;
  bool ok = true;
  // Item n of this block, for every role but the one that finds it. A role
  // gives it back once it has read what it needs of it.
  auto item_wait = [&](int n) -> bool {
    if (ok && !prompt_wait(&item_full[n & 1], (n >> 1) & 1, c.status, &alive_sh)) ok = false;
    return ok;
  };
  auto wait = [&](uint64_t* bar, int phase) {
    if (ok && !prompt_wait(bar, phase & 1, c.status, &alive_sh)) ok = false;
  };

  // Eight values of each 64 of a query row, lane `part` of the row's eight, to
  // the operands of row tile `tile`.
  constexpr int TILE_Q = (kSplit ? 2 : 1) * S::QB;
  auto operands = [&](const float (&v)[NB][8], int rr, int tile, int part, int buf) {
    float f = 1.f;
    if constexpr (kSplit) {
      // A power of two puts the row's largest value in [2^14, 2^15).
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[j][e]));
#pragma unroll
      for (int o = 4; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      f = pow2_factor(amax);
      if (part == 0) factor_sh[buf][tile][rr] = f;
    }
    f *= flip;
    uint8_t* to = q_sm + tile * TILE_Q + rr * 128 + ((part ^ (rr & 7)) << 4);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      uint32_t hi[4], rest[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z0 = v[j][2 * e] * f, z1 = v[j][2 * e + 1] * f;
        hi[e] = pack2<TKV>(z0, z1);
        if constexpr (kSplit) rest[e] = rest2<TKV>(z0, z1, hi[e]);
      }
      *reinterpret_cast<uint4*>(to + j * PM * 128) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if constexpr (kSplit)
        *reinterpret_cast<uint4*>(to + S::QB + j * PM * 128) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
    }
  };

  if (warp >= W_TMA) {
    if constexpr (NS == 2) regs_down<kOtherRegs>();  // a warpgroup at a time
  }
  if (warp == W_TMA) {
    // ---- K and V tiles: K 0 .. AHEAD-1, then V t, K t + AHEAD ----------------
    const int piece = min(c.page, BN), pieces = BN / piece;
    int it = 0;
    for (int n = 0; ok; ++n) {
      item_wait(n);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const Item x = items[n & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[n & 1]);
      if (!x.valid) break;
      auto page_at = [&](int t) {
        if (lane >= pieces || t >= x.t1) return -1;
        const int p = x.pos(t, BN) + lane * piece;
        if (p >= x.len) return -1;
        // (Looked at where it is used: the look-ups of the tiles ahead are under way
        // together.)
        return c.table[(int64_t)x.s * c.max_pages + (p >> c.page_log2)];
      };
      auto load = [&](const KvMap* map, int t, int id) {
        const int st = it % ST;
        if (it >= ST) wait(&kv_empty[st], it / ST - 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        uint8_t* to = ring + st * S::KV;
        if (lane == 0) mbar_expect_tx(&kv_full[st], S::KV);
        __syncwarp();
        if (lane < pieces) {
          const int p = x.pos(t, BN) + lane * piece;
          const bool in_pool = id >= 0 && id < c.n_pages;
          if (!in_pool && p < x.len) report(c.status, KC_ERR_ARG | (W_KV_PAGE << 8));
          const int lp = in_pool ? a.layer * c.n_pages + id : c.n_layer * c.n_pages;  // past the pool: zeros
#pragma unroll
          for (int b = 0; b < NB; ++b)
            kv_load(to + b * BN * 128 + lane * piece * 128, map, 64 * b, p & (c.page - 1), x.kvh, lp, &kv_full[st]);
        }
        ++it;
      };
      int kid[AHEAD + 1];  // pages of tiles t .. t + AHEAD
      for (int u = 0; u < AHEAD; ++u) kid[u] = page_at(x.t0 + u);
      for (int u = 0; u < AHEAD && x.t0 + u < x.t1 && ok; ++u) load(&maps.k, x.t0 + u, kid[u]);
      for (int t = x.t0; t < x.t1 && ok; ++t) {
        kid[AHEAD] = page_at(t + AHEAD);
        load(&maps.v, t, kid[0]);
        if (ok && t + AHEAD < x.t1) load(&maps.k, t + AHEAD, kid[AHEAD]);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) kid[u] = kid[u + 1];
      }
    }
    // Every load lands before the block may end.
    for (int i = max(0, it - ST); i < it; ++i) mbar_wait(&kv_full[i % ST], (i / ST) & 1, c.status, W_ATT_PROMPT);
  } else if (warp == W_MMA) {
    if (elect_one()) {
      const uint32_t id_s = tc_idesc<TKV>(BN, false), id_o = tc_idesc<TKV>(hd16, true);
      const int ksteps = hd16 / 16;
      const uint32_t qa = smem_u32(q_sm), ra = smem_u32(ring);
      int ring_at = 0;  // loads before this item's
      int kp[NS];       // weight tiles of each stream so far
      int used = 0;     // items with products so far
#pragma unroll
      for (int w = 0; w < NS; ++w) kp[w] = 0;
      auto stage = [&](int it) {
        wait(&kv_full[it % ST], it / ST);
        tc_fence_after();
        return ra + (it % ST) * S::KV;
      };
      // One instruction covers 16 of K; descriptors step in units of 16 bytes.
      // (Unrolled with constant steps: computing each descriptor in a loop
      // takes longer than the product it is for.)
      auto scores = [&](int w, uint32_t k) {
        const uint64_t kd = sw128_desc(k);
        // Rests first: the tensor cores cut a sum's last bits off at every step,
        // which costs the less the smaller the sum still is (f32 results over
        // 4096 positions are 1.9e-6 off otherwise).
#pragma unroll
        for (int part = kSplit ? 1 : 0; part >= 0; --part) {
          const uint64_t qd = sw128_desc(qa + ((TWO ? w : 0) * (kSplit ? 2 : 1) + part) * S::QB);
#pragma unroll
          for (int ks = 0; ks < 4 * NB; ++ks)
            if (ks < ksteps)
              tc_mma(tmem + S::T_S * w, qd + ((ks >> 2) * PM * 128 + 32 * (ks & 3)) / 16,
                     kd + ((ks >> 2) * BN * 128 + 32 * (ks & 3)) / 16, id_s,
                     part < (kSplit ? 1 : 0) || ks > 0);
        }
        tc_commit(&s_full[w]);
      };
      auto values = [&](int w, int k, uint32_t v, bool add) {
        const uint64_t vd = sw128_desc_mn(v, BN * 128);
        wait(&p_full[w], k);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int part = 0; part < (kRests ? 2 : 1); ++part)
#pragma unroll
          for (int ks = 0; ks < BN / 16; ++ks)
            tc_mma_ts(tmem + S::T_O + w * S::HD, tmem + S::T_P + S::T_PW * w + part * (BN / 2) + 8 * ks,
                      vd + ks * 2048 / 16, id_o, add || part > 0 || ks > 0);
        tc_commit(&pv_done[w]);
      };
      // Before an item's first products into an accumulator: the last item's
      // results have been read from it.
      auto results_read = [&](int w) {
        if (used > 0) wait(&o_empty[w], used - 1);
        tc_fence_after();
      };
      int claims = 0, claim_w = 0, claim_k = 0;  // the scores issued last: whose they are
      for (int n = 0; ok; ++n) {
        if (!item_wait(n)) break;
        const int valid = items[n & 1].valid, nt = items[n & 1].t1 - items[n & 1].t0;
        mbar_arrive(&item_empty[n & 1]);
        if (!valid) break;
        if (nt <= 0) continue;
        wait(&q_full, used);
        if (!ok) break;
        tc_fence_after();
        // Loads come as K 0, K 1, V 0, K 2, V 1 ...
        auto k_at = [&](int t) { return ring_at + (NS == 2 ? max(2 * t - 1, 0) : 2 * t); };
        auto v_at = [&](int t) { return ring_at + (NS == 2 ? min(2 * t + 2, 2 * nt - 1) : 2 * t + 1); };
        if constexpr (kShared) {
          // Steps: (tile, stream) pairs in turn. Scores of step i + 1, then the
          // products of step i - 1.
          const int steps = TWO ? 2 * nt : nt;
          for (int i = -1; i <= steps && ok; ++i) {
            if (i + 1 < steps) {
              const int w = (i + 1) & 1, t = TWO ? (i + 1) >> 1 : i + 1;
              const uint32_t k = stage(k_at(t));
              // The last scores have been read.
              if (claims++ > 0) wait(&s_free[claim_w], claim_k);
              if (!ok) break;
              tc_fence_after();
              scores(w, k);
              claim_w = w;
              claim_k = kp[w] + (TWO ? t : t >> 1);
              if (!TWO || w == 1) tc_commit(&kv_empty[k_at(t) % ST]);
              if (i + 2 == steps) tc_commit(&q_empty);
            }
            if (i >= 1) {
              const int w = (i - 1) & 1, t = TWO ? (i - 1) >> 1 : i - 1, k = TWO ? t : t >> 1;
              const uint32_t v = stage(v_at(t));
              if (k == 0) results_read(w);
              values(w, kp[w] + k, v, k % KEEP != 0);
              if (!ok) break;
              if (!TWO || w == 1) tc_commit(&kv_empty[v_at(t) % ST]);
            }
          }
          if (!TWO && nt == 1) results_read(1);  // (each item's phase is waited for)
#pragma unroll
          for (int w = 0; w < NS; ++w) kp[w] += TWO ? nt : (nt - w + 1) >> 1;
        } else {
          auto step_scores = [&](int t) {
            const uint32_t k = stage(k_at(t));
            if (!ok) return;
            scores(t % NS, k);
            tc_commit(&kv_empty[k_at(t) % ST]);
            if (t + 1 == nt) tc_commit(&q_empty);
          };
          for (int t = 0; t < NS && t < nt && ok; ++t) step_scores(t);
#pragma unroll
          for (int w = 0; w < NS; ++w) results_read(w);
          for (int t = 0; t < nt && ok; ++t) {
            const int w = t % NS;
            const uint32_t v = stage(v_at(t));
            values(w, kp[w] + t / NS, v, t / NS % KEEP != 0);
            if (!ok) break;
            tc_commit(&kv_empty[v_at(t) % ST]);
            if (t + NS < nt) step_scores(t + NS);
          }
#pragma unroll
          for (int w = 0; w < NS; ++w) kp[w] += (nt - w + NS - 1) / NS;
        }
        ring_at += 2 * nt;
        ++used;
      }
      // The tensor cores are done with TMEM and shared memory.
      tc_commit(&drained);
      mbar_wait(&drained, 0, c.status, W_ATT_PROMPT);
    }
  } else if (warp >= W_AUX) {
    // ---- the next item, and its queries -----------------------------------------
    const bool finder = warp == W_AUX;
    // Row tiles of entry i, the lane's of 32 consecutive ones, in whose order the
    // warp calls this; 0 where its rows are out of order: an entry begins where
    // every earlier one has begun or later, so that no two share a row and the
    // tiles of all of them are no more than the launch reckons with. `last`: the
    // largest beginning before these 32, and then up to them (0 until something is
    // out of order). The first time over the list says whether anything is.
    bool ascend = true, known = false;
    auto tiles_of = [&](int i, int& last, int& lo, int& hi) {
      if constexpr (SHARED) {
        lo = hi = 0;
        if (i < a.n && d.sh.of_group[i] > 0) {
          lo = max(a.row_start[i], d.sh.e0);
          hi = max(lo, min(a.row_start[i + 1], d.sh.e1));
        }
        return (int)(((int64_t)(hi - lo) * group + S::QT * PM - 1) / (S::QT * PM));
      }
      lo = hi = last;
      if (i < a.n) {
        lo = a.row_start[i];
        hi = a.row_start[i + 1];
      }
      bool wrong = lo < last || hi < lo || hi > a.n_rows;
      // (If none is wrong by itself they ascend: each begins where the last ends.)
      if (!ascend || (!known && __any_sync(0xffffffffu, wrong))) {
        ascend = false;
        int top = max(lo, last);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, top, o);
          if (lane >= o) top = max(top, y);
        }
        last = __shfl_sync(0xffffffffu, top, 31);
        wrong |= lo < top;
        if (wrong) {
          if (i < a.n && blockIdx.x == 0) report(c.status, KC_ERR_ARG | (W_KV_ROWS << 8));
          lo = hi = 0;
        }
      }
      return (int)(((int64_t)(hi - lo) * group + S::QT * PM - 1) / (S::QT * PM));
    };
    auto scan = [&](int v) {  // inclusive, over the warp
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
      }
      return v;
    };
    // Up to 32 entries are taken in the order of their positions, most last
    // (items are dealt from the end); this lane holds the lane-th of them.
    int e_i = lane, e_lo = 0, e_hi = 0, e_len = 0, e_sum = 0, tiles = 0, e_lead = 0;  // (e_lead: the lane-th entry's)
    const bool sorted = a.n <= 32;
    if (finder) {
      if (sorted) {
        int len = 0, m = 0;
        if constexpr (SHARED) {
          if (lane < a.n) {
            len = d.sh.of_group[lane];
            e_lead = d.sh.lead[lane];
            e_lo = max(a.row_start[lane], d.sh.e0);
            e_hi = max(e_lo, min(a.row_start[lane + 1], d.sh.e1));
          }
          if (len == 0) e_lo = e_hi = 0;
          m = (int)(((int64_t)(e_hi - e_lo) * group + S::QT * PM - 1) / (S::QT * PM));
        } else {
          const int s = lane < a.n ? (a.seqs ? a.seqs[lane] : lane) : -1;
          len = s >= 0 && s < c.n_seq ? kv_len(c, s) : 0;
        }
        int rank = 0;
        for (int j = 0; j < 32; ++j) {
          const int other = __shfl_sync(0xffffffffu, len, j);
          rank += other < len || (other == len && j < lane);
        }
        for (int j = 0; j < 32; ++j)
          if (__shfl_sync(0xffffffffu, rank, j) == lane) e_i = j;
        int last = 0;
        if constexpr (!SHARED) m = tiles_of(lane, last, e_lo, e_hi);
        e_lo = __shfl_sync(0xffffffffu, e_lo, e_i);
        e_hi = __shfl_sync(0xffffffffu, e_hi, e_i);
        e_len = __shfl_sync(0xffffffffu, len, e_i);
        e_sum = scan(__shfl_sync(0xffffffffu, m, e_i));
        tiles = __shfl_sync(0xffffffffu, e_sum, 31);
      } else {
        int m = 0, last = 0, lo, hi;
        for (int b = 0; b < a.n; b += 32) m += tiles_of(b + lane, last, lo, hi);
        tiles = __shfl_sync(0xffffffffu, scan(m), 31);
      }
    }
    known = true;
    const int64_t total = (int64_t)tiles * c.nkv * splits;
    int used = 0;
    int64_t idx = blockIdx.x;  // the block's first item; the rest as it comes to them
    bool dealt = false;
    for (int n = 0; ok; ++n) {
      Item x{};
      if (finder) {
        while (true) {
          if (dealt) {
            int more = 0;
            if (lane == 0) more = atomicAdd(d.next, 1);
            idx = (int64_t)blocks + __shfl_sync(0xffffffffu, more, 0);
          }
          dealt = true;
          x.valid = idx < total;
          if (!x.valid) break;
          x.split = (int)(idx % splits);
          x.unit = (int)(total / splits - 1 - idx / splits);
          x.kvh = x.unit % c.nkv;
          int t = x.unit / c.nkv, l = 0, i = 0;
          if (sorted) {
            l = __ffs(__ballot_sync(0xffffffffu, t < e_sum)) - 1;
            i = __shfl_sync(0xffffffffu, e_i, l);
            x.start = __shfl_sync(0xffffffffu, e_lo, l);
            x.count = __shfl_sync(0xffffffffu, e_hi, l) - x.start;
            x.len = __shfl_sync(0xffffffffu, e_len, l);
            if (l > 0) t -= __shfl_sync(0xffffffffu, e_sum, l - 1);
          } else {
            int last = 0;
            for (int b = 0; b < a.n; b += 32) {
              int lo, hi;
              const int m = tiles_of(b + lane, last, lo, hi), y = scan(m);
              const unsigned at = __ballot_sync(0xffffffffu, t < y);
              if (at) {
                l = __ffs(at) - 1;
                i = b + l;
                x.start = __shfl_sync(0xffffffffu, lo, l);
                x.count = __shfl_sync(0xffffffffu, hi, l) - x.start;
                t -= __shfl_sync(0xffffffffu, y - m, l);
                break;
              }
              t -= __shfl_sync(0xffffffffu, y, 31);
            }
          }
          x.row0 = t * S::QT * PM;
          if constexpr (SHARED) x.s = sorted ? __shfl_sync(0xffffffffu, e_lead, i & 31) : d.sh.lead[i];
          else x.s = a.seqs ? a.seqs[i] : i;
          if (x.s < 0 || x.s >= c.n_seq) {
            if (lane == 0) report(c.status, KC_ERR_ARG | (W_KV_SEQ << 8));
            continue;
          }
          if (!sorted) x.len = SHARED ? d.sh.of_group[i] : kv_len(c, x.s);
          x.rows = min(S::QT * PM, x.count * group - x.row0);
          // Positions of the first and last row, and the tiles they see.
          const int at0 = SHARED ? x.len - 1 : x.len - x.count + x.row0 / group,
                    at1 = SHARED ? x.len - 1 : x.len - x.count + (x.row0 + x.rows - 1) / group;
          x.head = x.w0 = x.nt = 0;
          if (at1 >= 0) {
            const int lo = a.window > 0 ? max(0, at0 - a.window + 1) : 0;
            x.head = (min(a.sinks, lo) + BN - 1) / BN;
            x.w0 = max(lo / BN, x.head);
            x.nt = x.head + at1 / BN + 1 - x.w0;
          }
          // At least four tiles to a part: a join takes about as long.
          x.splits = SHARED ? shared_splits(x.len, c.hd, splits) : max(1, min(splits, x.nt / 4));
          if (x.split >= x.splits) continue;
          x.t0 = (int)((int64_t)x.nt * x.split / x.splits);
          x.t1 = (int)((int64_t)x.nt * (x.split + 1) / x.splits);
          break;
        }
        if (n >= 2) wait(&item_empty[n & 1], (n >> 1) - 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          items[n & 1] = x;
          mbar_arrive(&item_full[n & 1]);
        }
      } else {
        item_wait(n);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        x = items[n & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[n & 1]);
      }
      if (!x.valid) break;
      if (x.nt <= 0) continue;
      // (Nothing would hold the queries of the items to come back for this warp: a
      // wait that it enters two of them late sees a phase of the same parity under
      // way, and after the last item for good.)
      if (kSplit && d.q_map && !finder) continue;
      if (used > 0) wait(&q_empty, used - 1);
      ++used;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const RowMap rm(x.row0, group);
      const TQ* q = static_cast<const TQ*>(a.q) + (int64_t)x.start * a.q_stride + (int64_t)x.kvh * group * c.hd;
      const int loader = tid - 32 * W_AUX;
      if (d.q_map && finder && lane == 0) {
        // A box per tile and 128 bytes of columns. (Rows past the entry's are
        // another's or zeros; nothing comes of them.)
        uint64_t* bar = kSplit ? &q_raw : &q_full;
        mbar_expect_tx(bar, S::Q_ALL);
        for (int y = 0; y < S::QT; ++y)
#pragma unroll
          for (int b = 0; b < TILE_Q / (PM * 128); ++b)
            tma_load_3d(q_sm + y * TILE_Q + b * PM * 128, &q_map, 128 / (int)sizeof(TQ) * b, x.kvh * group,
                        x.start + rm.tok0 + y * (PM / group), bar);
      }
      if (!kSplit && d.q_map) {
        if (!finder && lane == 0) mbar_arrive(&q_full);
        continue;
      }
      if (kSplit && d.q_map) continue;  // the softmax warps make operands of them
      {
        // Eight lanes per row, eight values of each 64 a lane.
        const bool wide = !((uintptr_t)a.q % 16) && a.q_stride * sizeof(TQ) % 16 == 0;
        const int part = loader & 7;
        constexpr int BATCH = NB > 2 ? 1 : kSplit ? 2 : 4;  // rows of a lane under way
        for (int f0 = loader >> 3; f0 < S::QT * PM; f0 += 8 * BATCH) {
          float v[BATCH][NB][8];
#pragma unroll
          for (int y = 0; y < BATCH; ++y) {
            const int f = f0 + 8 * y;
            const TQ* from = q + rm.offset(f < x.rows ? f : 0, a.q_stride, c.hd) + 8 * part;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
              const bool real = f < x.rows && 64 * j + 8 * part < c.hd;
              if (real && wide) {
                load8(from + 64 * j, v[y][j]);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[y][j][e] = real ? (float)from[64 * j + e] : 0.f;
              }
            }
          }
#pragma unroll
          for (int y = 0; y < BATCH; ++y)
            operands(v[y], (f0 + 8 * y) & (PM - 1), (f0 + 8 * y) >> 7, part, (used - 1) & 1);
        }
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full);
    }
    // Every load lands before the block may end.
    if (kSplit && finder && d.q_map && used > 0) mbar_wait(&q_raw, (used - 1) & 1, c.status, W_ATT_PROMPT);
    // The last block to find nothing left puts the counters back.
    if (finder && lane == 0 && atomicAdd(d.next + 1, 1) == blocks - 1) d.next[0] = d.next[1] = 0;
  } else {
    if constexpr (NS == 2) regs_up<kSoftmaxRegs>();
    // ---- softmax: stream w, a thread per row ---------------------------------
    const int w = warp >> 2, r = tid & 127, my_tile = TWO ? w : 0;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    float* kept = d.kept + (int64_t)(blockIdx.x * NS + w) * S::KEPT + 4 * r;
    const uint32_t s_t = tmem + lanes + S::T_S * w, p_t = tmem + lanes + S::T_P + S::T_PW * w;
    const float unit = flip == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
    int ks = 0, used = 0, ring_at = 0;  // score tiles, items with products, loads before this item's
    int done[NS] = {}, parts = 0;       // tiles of each stream, split items before this one's
    for (int n = 0;; ++n) {
      item_wait(n);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const Item& x = items[n & 1];  // (given back at the end: read from there as needed, it takes no registers)
      if (!x.valid) break;
      const RowMap rm(x.row0, group);
      const int f = my_tile * PM + r, nt = x.t1 - x.t0, at_base = x.len - x.count;
      const bool real = f < x.rows;
      const int at = !real ? -1 : SHARED ? x.len - 1 : at_base + rm.token(f);
      const int lo = a.window > 0 ? at - a.window + 1 : 0;
      if constexpr (kSplit) {
        if (d.q_map && nt > 0) {
          // The rows that TMA brought lie where their two operands go, row for
          // row: a warp reads its rows whole before it writes them. Eight lanes
          // per row, eight values of each 64 a lane. (By two warps, beside the
          // last item's end: 33 rows at 545 took 28 us from a cold L2, 26 so, 256
          // at 4096 68 and 62, 8192 from the first 852 and 845.)
          wait(&q_raw, used);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const int part = tid & 7;
          constexpr int STEP = 16 * NS;                   // rows of all threads at a time
          constexpr int BATCH = NB <= 2 ? PM / STEP : 1;  // those of a thread under way
          for (int f0 = tid >> 3; f0 < PM; f0 += STEP * BATCH) {
            float v[BATCH][NB][8];
#pragma unroll
            for (int y = 0; y < BATCH; ++y)
#pragma unroll
              for (int j = 0; j < NB; ++j) {
                const int row = f0 + STEP * y, c0 = 2 * (part & 3), sw = row & 7, flip_c = part >> 2;  // (bank order)
                const uint8_t* raw = q_sm + (2 * j + (part >> 2)) * PM * 128 + row * 128;
                const float4 u = *reinterpret_cast<const float4*>(raw + (((c0 + flip_c) ^ sw) << 4));
                const float4 z = *reinterpret_cast<const float4*>(raw + (((c0 + 1 - flip_c) ^ sw) << 4));
                const float4 lo4 = flip_c ? z : u, hi4 = flip_c ? u : z;
                v[y][j][0] = lo4.x; v[y][j][1] = lo4.y; v[y][j][2] = lo4.z; v[y][j][3] = lo4.w;
                v[y][j][4] = hi4.x; v[y][j][5] = hi4.y; v[y][j][6] = hi4.z; v[y][j][7] = hi4.w;
              }
            __syncwarp();
#pragma unroll
            for (int y = 0; y < BATCH; ++y) operands(v[y], f0 + STEP * y, 0, part, used & 1);
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full);
        }
      }
      // Tiles whose positions every row of this tile sees need no mask.
      const int t_at0 = SHARED ? x.len - 1 : at_base + rm.token(my_tile * PM);
      const int t_lo1 = a.window > 0 ? at_base + rm.token(min(x.rows, (my_tile + 1) * PM) - 1) - a.window + 1 : 0;
      float m = -INFINITY, l = 0.f;
      // Stream w's k-th tile is k (two row tiles) or NS k + w.
      const int mine = TWO ? nt : (nt - w + NS - 1) / NS;
      // Base-2 exponents per score unit (a zero scale has zero queries instead,
      // so that a masked score's -inf survives the product).
      float cq = unit;
      const uint32_t o_t = tmem + lanes + S::T_O + w * S::HD;
      for (int k = 0; k < mine; ++k, ++ks) {
        const int t = TWO ? k : NS * k + w, j0 = x.pos(x.t0 + t, BN);
        wait(&s_full[w], ks);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (rarely(k > 0 && k % KEEP == 0)) {
          // The products so far are complete (with the scores, or are waited for),
          // and the next ones do not add to them.
          if constexpr (kShared) {
            wait(&pv_done[w], ks - 1);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            tc_fence_after();
          }
          keep_sums(o_t, hd16, kept, m, k == KEEP ? KEEP_FIRST : KEEP_ADD);
        }
        if constexpr (kSplit)
          if (k == 0) cq = __fdiv_rn(unit, factor_sh[used & 1][my_tile][r]);
        float s[BN];
#pragma unroll
        for (int e = 0; e < BN; e += 32) tmem_ld32(s_t + e, s + e);
        tmem_wait_ld();
        if constexpr (kShared) {
          tc_fence_before();
          mbar_arrive(&s_free[w]);
        }
        if (rarely(j0 + BN - 1 > t_at0 || (j0 < t_lo1 && j0 + BN > a.sinks))) {
          // A bit per position: up to the row's own, and not before its window
          // unless among the first tokens.
          const int hi = at - j0, from = lo - j0, first = a.sinks - j0;
#pragma unroll
          for (int y = 0; y < BN; y += 32) {
            const uint32_t see = low_bits(hi + 1 - y) & (~low_bits(from - y) | low_bits(first - y));
#pragma unroll
            for (int e = 0; e < 32; ++e) s[y + e] = see >> e & 1 ? s[y + e] : -INFINITY;
          }
        }
        if (rarely(j0 + BN > x.len)) {
          // Rows past the sequence's end hold whatever the page held before:
          // zeros in their place (only the last tile has such rows; its V is
          // the item's last load).
          const int v_it = ring_at + 2 * nt - 1, st = v_it % ST;
          wait(&kv_full[st], v_it / ST);
          uint8_t* v = ring + st * S::KV;
          for (int y = r; y < BN * 8 * NB; y += 128)
            if (j0 + ((y >> 3) & (BN - 1)) >= x.len) *reinterpret_cast<uint4*>(v + y * 16) = make_uint4(0, 0, 0, 0);
          fence_async_shared();
        }
        // Weights of half the tile's positions against maximum mx.
        auto weigh = [&](int half, float mx, uint32_t* p, uint32_t* rest) {
          const float base = kLift - (mx == -INFINITY ? 0.f : mx);
          const uint64_t cq2 = f2(cq, cq), base2 = f2(base, base);
          uint64_t sums[4] = {0, 0, 0, 0};
          // In stretches of independent steps, so that none waits for the last.
#pragma unroll
          for (int e0 = 0; e0 < BN / 4; e0 += 4) {
            float2 y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = half * (BN / 2) + 2 * (e0 + e);
              y[e] = f2(fma2(f2(s[i], s[i + 1]), cq2, base2));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = make_float2(exp2_fast(y[e].x), exp2_fast(y[e].y));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sums[e & 3] = add2(sums[e & 3], f2(y[e].x, y[e].y));
              p[e0 + e] = pack2<TKV>(y[e].x, y[e].y);
              if constexpr (kRests) rest[e0 + e] = rest2<TKV>(y[e].x, y[e].y, p[e0 + e]);
            }
          }
          const float2 sum = f2(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
          return sum.x + sum.y;
        };
        auto put = [&](int half, const uint32_t* p, const uint32_t* rest) {
#pragma unroll
          for (int e = 0; e < BN / 4; e += 16) {
            tmem_st16(p_t + half * (BN / 4) + e, p + e);
            if constexpr (kRests) tmem_st16(p_t + BN / 2 + half * (BN / 4) + e, rest + e);
          }
        };
        // Largest of the row's scores, in exponents of 2.
        auto largest = [&]() {
          float tops[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) tops[e] = s[e];
#pragma unroll
          for (int e = 8; e < BN; e += 2) tops[e / 2 & 7] = max3(tops[e / 2 & 7], s[e], s[e + 1]);
          const float top =
              max3(max3(tops[0], tops[1], tops[2]), max3(tops[3], tops[4], tops[5]), fmaxf(tops[6], tops[7]));
          return top == -INFINITY ? top : top * cq;
        };
        // A larger reference: what has been summed so far is rescaled. The
        // products so far are complete, and the next ones wait for weights: the
        // accumulator is this warp's.
        auto rescale = [&](float top, bool grow) {
          tc_fence_after();
          const float shrink = grow ? exp2_fast(m - top) : 1.f;
          if (grow) m = top;
          l *= shrink;
          for (int e0 = 0; e0 < hd16; e0 += 16) {
            float o[16];
            tmem_ld16(o_t + e0, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= shrink;
            tmem_st16(o_t + e0, o);
          }
        };
        uint32_t p[BN / 4], rest[kRests ? BN / 4 : 1];
        float sum;
        if constexpr (kRests) {
          const float top = largest();
          if (k == 0) m = top;
          const bool grow = top > m + 8.f;
          if (__any_sync(0xffffffffu, grow)) rescale(top, grow);
          sum = weigh(0, m, p, rest);
          put(0, p, rest);
          sum += weigh(1, m, p, rest);
        } else {
          // No maximum is looked for after the first tile: while a tile's weights
          // add up to less than kMost, none of them is past the 16-bit type's
          // range, and any reference does. (8192 rows of 32 heads: 471 us with
          // every tile's maximum, 461 so.) The weights are handed over once: in two
          // halves, whose first products could start earlier, it took 4% more.
          if (rarely(k == 0)) m = largest();
          sum = weigh(0, m, p, rest);
          // The weights' columns are free once the last products are complete.
          if (kShared && ks > 0) wait(&pv_done[w], ks - 1);
          put(0, p, rest);
          sum += weigh(1, m, p, rest);
          if (rarely(__any_sync(0xffffffffu, !(sum < kMost) || m == -INFINITY))) {
            const float top = largest();
            const bool grow = top > m && (!(sum < kMost) || m == -INFINITY);
            if (__any_sync(0xffffffffu, grow)) {
              if (!kShared && ks > 0) wait(&pv_done[w], ks - 1);
              rescale(top, grow);
              sum = weigh(0, m, p, rest);
              put(0, p, rest);
              sum += weigh(1, m, p, rest);
            }
          }
        }
        put(1, p, rest);
        l += sum;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[w]);
      }

      // ---- the item's result -------------------------------------------------------
      // Of one row tile both streams' warps write half the columns each, from
      // both accumulators (a warp reads the lanes of its quarter, whoever's).
      constexpr bool kJoin = NS == 2 && !TWO;
      const int half = kJoin ? (hd16 / 16 + 1) / 2 * 16 : hd16;
      const int col0 = kJoin && w == 1 ? half : 0, col1 = kJoin && w == 0 ? half : hd16;
      float scale_of[NS];  // what each accumulator counts
#pragma unroll
      for (int v = 0; v < NS; ++v) scale_of[v] = 1.f;
      if (nt > 0) {
#pragma unroll
        for (int v = 0; v < NS; ++v)
          if (TWO ? v == w : v < nt) {
            done[v] += TWO ? nt : (nt - v + NS - 1) / NS;
            wait(&pv_done[v], done[v] - 1);
          }
        if (rarely(mine > KEEP)) {
          // What was kept goes back to the accumulator.
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after();
          if (ok) keep_sums(o_t, hd16, kept, m, KEEP_RETURN);
          tc_fence_before();
        }
        if constexpr (kJoin) {
          join_sh[used & 1][w][r] = make_float2(m, l);
          mbar_arrive(&join_full);
          wait(&join_full, used);
          const float2 o = join_sh[used & 1][w ^ 1][r];
          const float mn = fmaxf(m, o.x);
          const float mine_f = mn == -INFINITY ? 0.f : exp2_fast(m - mn);
          const float their_f = mn == -INFINITY ? 0.f : exp2_fast(o.x - mn);
          // The same order of operations on both sides.
          l = w == 0 ? __fmaf_rn(l, mine_f, o.y * their_f) : __fmaf_rn(o.y, their_f, l * mine_f);
          m = mn;
          scale_of[w] = mine_f;
          scale_of[w ^ 1] = their_f;
        }
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      const bool split = !SHARED && x.splits > 1;
      TQ* out = static_cast<TQ*>(a.out) + (int64_t)x.start * a.out_stride + (int64_t)x.kvh * group * c.hd;
      const uint32_t grain = (uint32_t)((uintptr_t)a.out | (uint64_t)a.out_stride * sizeof(TQ) | c.hd * sizeof(TQ));
      float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
      bool bad = l != l || l == INFINITY;
      TQ* to_row = out + rm.offset(real ? f : 0, a.out_stride, c.hd);
      float* part_row = d.part + ((int64_t)x.unit * d.splits + x.split) * S::PART + 4 * r;
      // SHARED: the row of its (split, entry, head) for the join.
      constexpr int JOIN_LD = S::HD + 8, JOIN_GRAIN = JOIN_LD * 4;  // (rows of whole sectors)
      float* join_row = nullptr;
      if constexpr (SHARED)
        join_row = d.sh.part + (((int64_t)x.split * (d.sh.e1 - d.sh.e0) + x.start - d.sh.e0) * a.nh + x.kvh * group) * JOIN_LD +
                   rm.offset(real ? f : 0, (int64_t)a.nh * JOIN_LD, JOIN_LD);
      for (int e0 = col0; e0 < col1; e0 += 32) {
        float o[2][16];
        const uint32_t o_0 = tmem + lanes + S::T_O + (TWO ? w : 0) * S::HD + e0;
        const bool both = e0 + 16 < col1;
        if (nt > 0 && ok) {
          tmem_ld16(o_0, o[0]);
          if (both) tmem_ld16(o_0 + 16, o[1]);
          if (kJoin && nt > 1) {
            float o1[2][16];
            tmem_ld16(o_0 + S::HD, o1[0]);
            if (both) tmem_ld16(o_0 + S::HD + 16, o1[1]);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e >> 4][e & 15] = __fmaf_rn(o[e >> 4][e & 15], scale_of[0], o1[e >> 4][e & 15] * scale_of[NS - 1]);
          }
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e >> 4][e & 15] = 0.f;
        }
        if (!real) continue;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (y && !both) break;
          const int e1 = e0 + 16 * y;
          if constexpr (SHARED) {
            bad |= normalise16(o[y], inv);
            store16(join_row + e1, o[y], 16, JOIN_GRAIN);
            if (e1 == 0) *reinterpret_cast<float2*>(join_row + S::HD) = make_float2(m - kLift, l);
            continue;
          }
          if (split) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<float4*>(part_row + (e1 + e) * PM) =
                  make_float4(o[y][e], o[y][e + 1], o[y][e + 2], o[y][e + 3]);
            if (e1 == 0) *reinterpret_cast<float2*>(part_row + S::HD * PM - 2 * r) = make_float2(m, l);
            continue;
          }
          bad |= normalise16(o[y], inv);
          store16(to_row + e1, o[y], c.hd - e1, grain);
        }
      }
      if (nt > 0) {
        tc_fence_before();
#pragma unroll
        for (int v = 0; v < NS; ++v)
          if (!TWO || v == w) mbar_arrive(&o_empty[v]);
        ++used;
        ring_at += 2 * nt;
      }
      bool write = !split;
      if (split) {
        // The parts in their order, by the block that brings the last one.
        __threadfence();
        mbar_arrive(&part_full);
        if (tid == 0) {
          wait(&part_full, parts);
          last_sh = ok && atomicAdd(d.count + x.unit, 1) == x.splits - 1;
          if (last_sh) d.count[x.unit] = 0;
          __threadfence();
          mbar_arrive(&last_full);
        }
        wait(&last_full, parts);
        ++parts;
        ok = __all_sync(0xffffffffu, ok);
        write = ok && last_sh;
        if (write) {
          __threadfence();
          const float* from = d.part + (int64_t)x.unit * d.splits * S::PART + 4 * r;
          float share[P_SPLITS_MAX], top = -INFINITY;
          l = 0.f;
          {
            float2 ml[P_SPLITS_MAX];
#pragma unroll
            for (int p = 0; p < P_SPLITS_MAX; ++p) {
              ml[p] = p < x.splits ? __ldcg(reinterpret_cast<const float2*>(from + p * S::PART + S::HD * PM - 2 * r))
                                   : make_float2(-INFINITY, 0.f);
              top = fmaxf(top, ml[p].x);
            }
#pragma unroll
            for (int p = 0; p < P_SPLITS_MAX; ++p) {
              share[p] = top == -INFINITY ? 0.f : exp2_fast(ml[p].x - top);
              l = __fmaf_rn(share[p], ml[p].y, l);
            }
          }
          inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
          bad = l != l || l == INFINITY;
          for (int e0 = col0; e0 < col1 && real; e0 += 16) {
            float o[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0.f;
#pragma unroll
            for (int p = 0; p < P_SPLITS_MAX; ++p) {
              if (p >= x.splits) break;
#pragma unroll
              for (int e = 0; e < 16; e += 4) {
                const float4 y = __ldcg(reinterpret_cast<const float4*>(from + p * S::PART + (e0 + e) * PM));
                o[e] = __fmaf_rn(share[p], y.x, o[e]);
                o[e + 1] = __fmaf_rn(share[p], y.y, o[e + 1]);
                o[e + 2] = __fmaf_rn(share[p], y.z, o[e + 2]);
                o[e + 3] = __fmaf_rn(share[p], y.w, o[e + 3]);
              }
            }
            bad |= normalise16(o, inv);
            store16(to_row + e0, o, c.hd - e0, grain);
          }
        }
      }
      // A row that a value beyond its mask has spoilt (or that sees a NaN, or an
      // infinity against a weight's rest) is computed again by itself.
      for (unsigned again = __ballot_sync(0xffffffffu, ok && write && real && bad); again; again &= again - 1) {
        const int f1 = my_tile * PM + 32 * (warp & 3) + __ffs(again) - 1;
        const TQ* q_row = static_cast<const TQ*>(a.q) + (int64_t)x.start * a.q_stride + (int64_t)x.kvh * group * c.hd +
                          rm.offset(f1, a.q_stride, c.hd);
        if constexpr (SHARED) {
          // (x.head is 0: position tile t begins at t BN.)
          float* to = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, (unsigned long long)join_row, __ffs(again) - 1));
          prompt_row<TQ, TKV, float, true>(a, x.s, x.kvh, x.t0 * BN, min(x.t1 * BN, x.len) - 1, q_row, to, col0,
                                           min(col1, c.hd), to + S::HD, &alive_sh);
        } else {
          prompt_row<TQ, TKV, TQ, false>(a, x.s, x.kvh, 0, at_base + rm.token(f1), q_row,
                                         out + rm.offset(f1, a.out_stride, c.hd), col0, min(col1, c.hd), nullptr,
                                         &alive_sh);
        }
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[n & 1]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == W_MMA) tmem_free(tmem, 512);
}

// Parts of split items: what 192 items of 128 rows take at a head size of 128.
constexpr size_t PROMPT_PART_BYTES = (size_t)192 * PM * (128 + 2) * sizeof(float);
constexpr int PROMPT_MAX_UNITS = 192;
// Behind them, what the streams of every block keep of sums over many tiles.
size_t attn_prompt_part_bytes() {
  return PROMPT_PART_BYTES + (size_t)num_sms() * PM * KEPT_COLUMNS * sizeof(float);
}
int attn_prompt_counts() { return PROMPT_MAX_UNITS + 2; }

template <typename TQ, typename TKV, int NB, bool TWO, bool SHARED>
static int launch_prompt(PromptArgs d, const KvMaps& maps, cudaStream_t st) {
  using S = PromptShape<TQ, NB, TWO, SHARED>;
  const AttnArgs& a = d.a;
  static PerDeviceOnce attr;
  if (smem_attr_once(attr, attn_prompt_kernel<TQ, TKV, NB, TWO, SHARED>, S::SMEM) != cudaSuccess) return KC_ERR_CUDA;
  // Every sequence may leave its last tile partly filled.
  const int64_t rows = (int64_t)a.n_rows * (a.nh / a.c.nkv), tile = S::QT * PM;
  const int64_t most = (rows / tile + std::min(a.n, a.n_rows)) * a.c.nkv;
  if (most > INT32_MAX / 16) return KC_ERR_SHAPE;
  d.splits = SHARED ? d.sh.splits : 1;
  if (!TWO && !SHARED) {
    // Fewer items than SMs: their positions over as many blocks as there are,
    // within the workspace.
    const int64_t likely = std::max<int64_t>((rows + tile - 1) / tile, std::min(a.n, a.n_rows)) * a.c.nkv;
    const int64_t slots = std::min<int64_t>(PROMPT_MAX_UNITS, PROMPT_PART_BYTES / (S::PART * sizeof(float)));
    d.splits = (int)std::max<int64_t>(1, std::min<int64_t>({num_sms() / likely, slots / most, P_SPLITS_MAX}));
  }
  const int grid = (int)std::min<int64_t>(num_sms(), most * d.splits);
  // Queries by TMA where a tile is whole tokens and TMA can address them (16-bit
  // ones go to the tensor cores as they are); otherwise two warps bring them.
  KvMap q_map{};
  const int group = a.nh / a.c.nkv;
  d.q_map = (S::kSplit || a.scale > 0.f) && PM % group == 0 && !((uintptr_t)a.q % 16) &&
            a.q_stride * sizeof(TQ) % 16 == 0 && make_q_map(a, q_map) == KC_OK;
  launch_k(attn_prompt_kernel<TQ, TKV, NB, TWO, SHARED>, grid, S::THREADS, S::SMEM, st, d, maps, q_map);
  return KC_OK;
}

template <typename TQ, typename TKV, bool SHARED>
static int launch_prompt_hd(const PromptArgs& d, const KvMaps& maps, cudaStream_t st) {
  // Two row tiles per item read every key and value once for both; with few
  // rows, or f32 queries (two operands each), an item is one. f16, 32 and 4 heads
  // of 128, two tiles and one, us: 5 x 256 rows at 2048 (160 pairs) 69 and 66, 6 x
  // 256 at 300 to 4000 (192) 85 and 74, 8 x 256 at 2048 (256) 73 and 88, 10 x 256
  // (320) 103 and 109, 2048 from the first (256) 56 and 63, 8192 (1024) 527 and 606.
  // (Below two rounds of pairs one tile evens the rounds out better; the rule does
  // not count them.)
  const AttnArgs& a = d.a;
  const int64_t pairs = ((int64_t)a.n_rows * (a.nh / a.c.nkv) + 2 * PM - 1) / (2 * PM) * a.c.nkv;
  const bool two = sizeof(TQ) == 2 && !SHARED && pairs >= num_sms();
  switch ((a.c.hd + 63) / 64) {
    case 1:
      if constexpr (sizeof(TQ) == 2)
        if (two) return launch_prompt<TQ, TKV, 1, true, false>(d, maps, st);
      return launch_prompt<TQ, TKV, 1, false, SHARED>(d, maps, st);
    case 2:
      if constexpr (sizeof(TQ) == 2)
        if (two) return launch_prompt<TQ, TKV, 2, true, false>(d, maps, st);
      return launch_prompt<TQ, TKV, 2, false, SHARED>(d, maps, st);
    case 3: return launch_prompt<TQ, TKV, 3, false, SHARED>(d, maps, st);
    default: return launch_prompt<TQ, TKV, 4, false, SHARED>(d, maps, st);
  }
}

int attn_prompt_box_rows(int page, int hd) { return std::min(page, hd <= 128 ? 128 : 64); }

template <bool SHARED>
static int launch_prompt_types(const PromptArgs& d, const KvMaps& maps, cudaStream_t st) {
  if (d.a.c.type == T_BF16) return launch_prompt_hd<__nv_bfloat16, __nv_bfloat16, SHARED>(d, maps, st);
  if (d.a.t_q == T_F32) return launch_prompt_hd<float, __half, SHARED>(d, maps, st);
  return launch_prompt_hd<__half, __half, SHARED>(d, maps, st);
}

int launch_attn_prompt(const AttnArgs& a, const KvMaps& maps, float* part, int* count, cudaStream_t st) {
  return launch_prompt_types<false>(
      PromptArgs{a, 1, part, part + PROMPT_PART_BYTES / sizeof(float), count, count + PROMPT_MAX_UNITS, false, {}}, maps,
      st);
}

int launch_attn_prefix(const AttnArgs& a, const SharedArgs& sh, const KvMaps& maps, float* part, int* count,
                       cudaStream_t st) {
  return launch_prompt_types<true>(
      PromptArgs{a, 1, part, part + PROMPT_PART_BYTES / sizeof(float), count, count + PROMPT_MAX_UNITS, false, sh}, maps,
      st);
}

}  // namespace kc
