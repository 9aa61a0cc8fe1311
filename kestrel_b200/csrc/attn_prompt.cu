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
// key and value. Positions pass in tiles of BN. Roles:
//   softmax warps  four per stream, a thread per row: scores from TMEM, the
//                  mask where the tile needs it, weights back to TMEM as the
//                  16-bit A operand of the second product. The accumulator is
//                  rescaled only when a row's maximum has grown by 2^8.
//   a TMA warp     K and V tiles, a box per page, through one ring.
//   an MMA warp    S = Q K^T (both in shared memory), O += P V (P in TMEM).
// Two streams take turns on the tensor cores, so that one's exponentials run
// beside the other's products (an MMA tile of 128 x 128 x 128 takes as long as
// its 16384 exponentials): either two row tiles over the same positions, or
// one row tile whose position tiles alternate, joined at the end.
//
// f32 queries are carried by two f16 operands (value and rest), and so are
// their weights: twice the products, f32-grade results over a 16-bit cache.
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
// One pair of weights in this many takes its exponentials from exp2_cubic.
constexpr int kCubicEvery = 4;
constexpr int kSoftmaxRegs = 200, kOtherRegs = 104;
static_assert(2 * kSoftmaxRegs + kOtherRegs == 3 * 168, "within the registers of the launch");

template <typename TQ, int NB, bool TWO>
struct PromptShape {
  static constexpr bool kSplit = sizeof(TQ) == 4;
  static constexpr int HD = 64 * NB;               // padded head size
  static constexpr int BN = NB <= 2 ? 128 : 64;    // positions of a tile
  static constexpr int NS = NB <= 2 ? 2 : 1;       // streams
  static constexpr int QT = TWO ? 2 : 1;           // row tiles
  static constexpr int QB = PM * 128 * NB;         // bytes of a query operand
  static constexpr int Q_ALL = QT * (kSplit ? 2 : 1) * QB;
  static constexpr int KV = BN * 128 * NB;         // bytes of a K or V tile
  static constexpr int CAP = 226 * 1024;
  static constexpr int FIT = (CAP - 1024 - Q_ALL) / KV;
  static constexpr int ST = FIT < P_STAGES_MAX ? FIT : P_STAGES_MAX;
  static constexpr int SMEM = Q_ALL + ST * KV + 1024;
  // Two streams: three warpgroups of 168 registers a thread at launch, of which
  // the third (loads, MMAs, two idle warps) gives the softmax warps 32 each.
  static constexpr int THREADS = NS == 2 ? 384 : 192;
  static constexpr int T_O = 256;                  // TMEM columns: S of stream w at 128 w, its O at T_O + HD w
  static constexpr int JOIN_LD = HD + 4;           // floats of a row handed over between the streams
  static_assert(!TWO || NS == 2, "two row tiles need two streams");
  static_assert(ST >= 2 && T_O + NS * HD <= 512, "fits");
  // Shared memory after the last product: the join, then the rows going out.
  static constexpr int OUT_AT = TWO || NS == 1 ? 0 : (PM * JOIN_LD * 4 + 1023) / 1024 * 1024;
  static_assert(TWO || OUT_AT + PM * HD * (int)sizeof(TQ) <= Q_ALL + ST * KV, "join and output fit");
};

// The position tiles that a row tile reads: `head` tiles of the first tokens,
// then tiles w0 .. (n tiles in all).
struct TileSpan {
  int head, w0, n;
  __device__ int start(int t, int bn) const { return (t < head ? t : t - head + w0) * bn; }
};

// The lowest n bits (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
}

struct RowTile {
  int i, s, len, count, start;  // entry, sequence, its positions, its rows, its first row
  int row0;                     // first (token, head) row of the block's tiles
};

// One row computed position by position by a warp: what the products cannot
// give when a value that the row does not see is not finite (0 * NaN).
template <typename TQ, typename TKV>
__device__ __noinline__ void prompt_row(const AttnArgs& a, int s, int kvh, int at, const TQ* q, TQ* out) {
  const KvView& c = a.c;
  const int lane = threadIdx.x & 31, lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
  float x[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    x[u] = lane + 32 * u < c.hd ? (float)q[lane + 32 * u] : 0.f;
    o[u] = 0.f;
  }
  for (int j = 0; j <= at; ++j) {
    if (j < lo && j >= a.sinks) {
      j = lo - 1;
      continue;
    }
    const int id = c.table[(int64_t)s * c.max_pages + (j >> c.page_log2)];
    if (id < 0 || id >= c.n_pages) continue;
    const int64_t e =
        ((((int64_t)a.layer * c.n_pages + id) * c.nkv + kvh) * c.page + (j & (c.page - 1))) * (int64_t)c.hd;
    const TKV* k = reinterpret_cast<const TKV*>(c.k) + e;
    const TKV* v = reinterpret_cast<const TKV*>(c.v) + e;
    float t = 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (lane + 32 * u < c.hd) t = __fmaf_rn(x[u], (float)k[lane + 32 * u], t);
#pragma unroll
    for (int w = 16; w; w >>= 1) t += __shfl_xor_sync(0xffffffffu, t, w);
    t *= a.scale;
    if (t != t) {  // every result is NaN
      l = t;
      break;
    }
    const float mn = fmaxf(m, t), shrink = mn == -INFINITY ? 1.f : expf(m - mn);
    const float p = mn == -INFINITY ? 0.f : expf(t - mn);
    m = mn;
    l = __fmaf_rn(l, shrink, p);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (lane + 32 * u < c.hd) o[u] = __fmaf_rn(p, (float)v[lane + 32 * u], o[u] * shrink);
  }
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (lane + 32 * u < c.hd) out[lane + 32 * u] = (TQ)(l == 0.f ? 0.f : l != l ? l : __fdiv_rn(o[u], l));
}

template <typename TQ, typename TKV, int NB, bool TWO>
__global__ void __launch_bounds__(PromptShape<TQ, NB, TWO>::THREADS, 1)
    attn_prompt_kernel(const AttnArgs a, const __grid_constant__ KvMaps maps) {
  using S = PromptShape<TQ, NB, TWO>;
  constexpr int BN = S::BN, NS = S::NS, ST = S::ST;
  constexpr bool kSplit = S::kSplit;
  // Weights reach 2^(lift + 8): small ones of f16 keep their bits.
  constexpr float kLift = std::is_same_v<TKV, __half> ? 7.f : 0.f;
  constexpr float kGrow = 8.f;
  pdl_enter();
  extern __shared__ uint8_t prompt_raw[];
  __shared__ __align__(8) uint64_t kv_full[ST], kv_empty[ST], s_full[NS], p_half[NS], p_full[NS], o_full[NS];
  __shared__ __align__(8) uint64_t q_full, drained;
  __shared__ uint32_t tmem_sh;
  __shared__ RowTile rt_sh;
  __shared__ float factor_sh[S::QT][PM];  // what a row's queries were multiplied with (f32 queries)
  const KvView& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int W_TMA = 4 * NS, W_MMA = W_TMA + 1;
  const int group = a.nh / c.nkv;
  const int block = gridDim.x - 1 - blockIdx.x;  // later rows see more: they begin first
  const int kvh = block % c.nkv;

  // ---- the block's rows ------------------------------------------------------
  if (warp == 0) {
    RowTile r{};
    r.i = -1;
    int t = block / c.nkv;
    for (int b = 0; b < a.n && r.i < 0; b += 32) {
      int lo = 0, hi = 0;
      if (b + lane < a.n) {
        lo = a.row_start[b + lane];
        hi = a.row_start[b + lane + 1];
        if (lo < 0 || hi < lo || hi > a.n_rows) {
          if (block == 0) report(c.status, KC_ERR_ARG | (W_KV_ROWS << 8));
          lo = hi = 0;
        }
      }
      const int n = (int)(((int64_t)(hi - lo) * group + S::QT * PM - 1) / (S::QT * PM));
      int x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const unsigned mine = __ballot_sync(0xffffffffu, t >= x - n && t < x);
      if (mine) {
        const int l = __ffs(mine) - 1;
        r.i = b + l;
        r.start = __shfl_sync(0xffffffffu, lo, l);
        r.count = __shfl_sync(0xffffffffu, hi - lo, l);
        r.row0 = (t - __shfl_sync(0xffffffffu, x - n, l)) * S::QT * PM;
      }
      t -= __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) {
      if (r.i >= 0) {
        r.s = a.seqs ? a.seqs[r.i] : r.i;
        if (r.s < 0 || r.s >= c.n_seq) {
          report(c.status, KC_ERR_ARG | (W_KV_SEQ << 8));
          r.i = -1;
        } else {
          r.len = kv_len(c, r.s);
        }
      }
      rt_sh = r;
      for (int i = 0; i < ST; ++i) {
        mbar_init(&kv_full[i], 1);
        mbar_init(&kv_empty[i], 1);
      }
      for (int w = 0; w < NS; ++w) {
        mbar_init(&s_full[w], 1);
        mbar_init(&p_half[w], 128);
        mbar_init(&p_full[w], 128);
        mbar_init(&o_full[w], 1);
      }
      mbar_init(&q_full, 128 * NS);
      mbar_init(&drained, 1);
      fence_mbar_init();
    }
  }
  __syncthreads();
  const RowTile rt = rt_sh;
  if (rt.i < 0) return;
  if (warp == W_MMA) tmem_alloc(&tmem_sh, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_sh;
  uint8_t* q_sm = prompt_raw + ((1024 - (smem_u32(prompt_raw) & 1023)) & 1023);
  uint8_t* ring = q_sm + S::Q_ALL;
  const int rows = min(S::QT * PM, rt.count * group - rt.row0);
  // Positions of the first and last row, and the tiles they read.
  const int at0 = rt.len - rt.count + rt.row0 / group, at1 = rt.len - rt.count + (rt.row0 + rows - 1) / group;
  TileSpan span{0, 0, 0};
  if (at1 >= 0) {
    const int lo = a.window > 0 ? max(0, at0 - a.window + 1) : 0;
    span.head = (min(a.sinks, lo) + BN - 1) / BN;
    span.w0 = max(lo / BN, span.head);
    span.n = span.head + at1 / BN + 1 - span.w0;
  }
  const int nt = span.n;
  const int hd16 = (c.hd + 15) / 16 * 16;  // columns of the products that are computed
  // Stream w's k-th tile is k (two row tiles) or NS k + w.
  auto tiles_of = [&](int w) { return TWO ? nt : (nt - w + NS - 1) / NS; };
  constexpr int AHEAD = TWO ? 1 : NS;  // K tiles loaded before the first V
  bool ok = true;

  if (warp >= W_TMA) {
    if constexpr (NS == 2) regs_down<kOtherRegs>();  // with the idle warps: a warpgroup at a time
  }
  if (warp == W_TMA) {
    // ---- K and V tiles: K 0 .. AHEAD-1, then V t, K t + AHEAD ----------------
    const int piece = min(c.page, BN), pieces = BN / piece;
    int it = 0;
    auto page_at = [&](int t) {
      if (lane >= pieces || t >= nt) return -1;
      const int p = span.start(t, BN) + lane * piece;
      if (p >= rt.len) return -1;
      const int id = c.table[(int64_t)rt.s * c.max_pages + (p >> c.page_log2)];
      if (id < 0 || id >= c.n_pages) {
        report(c.status, KC_ERR_ARG | (W_KV_PAGE << 8));
        return -1;
      }
      return id;
    };
    auto load = [&](const KvMap* map, int t, int id) {
      const int st = it % ST;
      if (it >= ST && !mbar_wait(&kv_empty[st], (it / ST - 1) & 1, c.status, W_ATT_PROMPT)) ok = false;
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      uint8_t* to = ring + st * S::KV;
      if (lane == 0) mbar_expect_tx(&kv_full[st], S::KV);
      __syncwarp();
      if (lane < pieces) {
        const int p = span.start(t, BN) + lane * piece;
        const int lp = id >= 0 ? a.layer * c.n_pages + id : c.n_layer * c.n_pages;  // past the pool: zeros
#pragma unroll
        for (int b = 0; b < NB; ++b)
          kv_load(to + b * BN * 128 + lane * piece * 128, map, 64 * b, p & (c.page - 1), kvh, lp, &kv_full[st]);
      }
      ++it;
    };
    int kid[AHEAD + 1];  // pages of tiles t .. t + AHEAD
    for (int t = 0; t < AHEAD; ++t) kid[t] = page_at(t);
    for (int t = 0; t < AHEAD && t < nt && ok; ++t) load(&maps.k, t, kid[t]);
    for (int t = 0; t < nt && ok; ++t) {
      kid[AHEAD] = page_at(t + AHEAD);
      load(&maps.v, t, kid[0]);
      if (ok && t + AHEAD < nt) load(&maps.k, t + AHEAD, kid[AHEAD]);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) kid[u] = kid[u + 1];
    }
    // Every load lands before the block may end.
    for (int i = max(0, it - ST); i < it; ++i) mbar_wait(&kv_full[i % ST], (i / ST) & 1, c.status, W_ATT_PROMPT);
  } else if (warp == W_MMA) {
    if (nt > 0 && elect_one()) {
      const uint32_t id_s = tc_idesc<TKV>(BN, false), id_o = tc_idesc<TKV>(hd16, true);
      const int ksteps = hd16 / 16;
      const uint32_t qa = smem_u32(q_sm), ra = smem_u32(ring);
      int it = 0;  // next stage of the ring, in the order of its loads
      auto stage_wait = [&]() {
        if (ok && !mbar_wait(&kv_full[it % ST], (it / ST) & 1, c.status, W_ATT_PROMPT)) ok = false;
        tc_fence_after();
        return ra + (it % ST) * S::KV;
      };
      // One instruction covers 16 of K; descriptors step in units of 16 bytes.
      // (Unrolled with constant steps: computing each descriptor in a loop
      // takes longer than the product it is for.)
      auto scores = [&](int w, uint32_t k) {
        const uint64_t kd = sw128_desc(k);
#pragma unroll
        for (int part = 0; part < (kSplit ? 2 : 1); ++part) {
          const uint64_t qd = sw128_desc(qa + ((TWO ? w : 0) * (kSplit ? 2 : 1) + part) * S::QB);
#pragma unroll
          for (int ks = 0; ks < 4 * NB; ++ks)
            if (ks < ksteps)
              tc_mma(tmem + 128 * w, qd + ((ks >> 2) * PM * 128 + 32 * (ks & 3)) / 16,
                     kd + ((ks >> 2) * BN * 128 + 32 * (ks & 3)) / 16, id_s, part > 0 || ks > 0);
        }
        tc_commit(&s_full[w]);
      };
      // The weights come in two halves, so that the first half's products run
      // beside the exponentials of the second.
      auto values = [&](int w, int k, uint32_t v, bool add) {
        const uint64_t vd = sw128_desc_mn(v, BN * 128);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (ok && !mbar_wait(half ? &p_full[w] : &p_half[w], k & 1, c.status, W_ATT_PROMPT)) ok = false;
          if (!ok) return;
          tc_fence_after();
#pragma unroll
          for (int part = 0; part < (kSplit ? 2 : 1); ++part)
#pragma unroll
            for (int ks = half * (BN / 32); ks < (half + 1) * (BN / 32); ++ks)
              tc_mma_ts(tmem + S::T_O + w * S::HD, tmem + 128 * w + part * (BN / 2) + 8 * ks, vd + ks * 2048 / 16,
                        id_o, add || half > 0 || part > 0 || ks > 0);
        }
      };
      if (!mbar_wait(&q_full, 0, c.status, W_ATT_PROMPT)) ok = false;
      if constexpr (TWO) {
        uint32_t k = stage_wait();
        if (ok) {
          scores(0, k);
          scores(1, k);
          tc_commit(&kv_empty[it % ST]);
        }
        ++it;
        for (int t = 0; t < nt && ok; ++t) {
          const int v_it = it;
          const uint32_t v = stage_wait();
          ++it;
          const bool more = t + 1 < nt;
          k = 0;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            values(w, t, v, t > 0);
            if (!ok) break;
            if (w == 1) tc_commit(&kv_empty[v_it % ST]);
            if (!more) {
              tc_commit(&o_full[w]);
              continue;
            }
            if (w == 0) k = stage_wait();
            if (!ok) break;
            scores(w, k);
          }
          if (ok && more) tc_commit(&kv_empty[it % ST]);
          if (more) ++it;
        }
      } else {
        for (int w = 0; w < NS && w < nt && ok; ++w) {
          const uint32_t k = stage_wait();
          if (!ok) break;
          scores(w, k);
          tc_commit(&kv_empty[it % ST]);
          ++it;
        }
        for (int t = 0; t < nt && ok; ++t) {
          const int w = t % NS;
          const uint32_t v = stage_wait();
          values(w, t / NS, v, t >= NS);
          if (!ok) break;
          tc_commit(&kv_empty[it % ST]);
          ++it;
          if (t + NS < nt) {
            const uint32_t k = stage_wait();
            if (!ok) break;
            scores(w, k);
            tc_commit(&kv_empty[it % ST]);
            ++it;
          } else {
            tc_commit(&o_full[w]);
          }
        }
      }
      // The tensor cores are done with TMEM and shared memory.
      tc_commit(&drained);
      mbar_wait(&drained, 0, c.status, W_ATT_PROMPT);
    }
  } else if (warp < W_TMA) {
    if constexpr (NS == 2) regs_up<kSoftmaxRegs>();
    // ---- softmax: stream w, a thread per row ---------------------------------
    const int w = warp >> 2, r = tid & 127, my_tile = TWO ? w : 0;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_t = tmem + lanes + 128 * w, o_t = tmem + lanes + S::T_O + w * S::HD;
    const TQ* q = static_cast<const TQ*>(a.q);
    const float flip = a.scale > 0.f ? 1.f : a.scale < 0.f ? -1.f : 0.f;  // score factors are positive: see below
    // Row f of the block: its token among the sequence's rows, its head of the
    // group ((x * magic) >> 16 = x / group for x < 512, group <= 128).
    const int tok0 = rt.row0 / group, rem = rt.row0 - tok0 * group;
    const uint32_t magic = 65536u / group + 1;
    auto token = [&](int f) { return tok0 + (int)(((uint32_t)(rem + f) * magic) >> 16); };
    auto row_of = [&](int f, int64_t stride) {
      const int t = token(f);
      return (int64_t)(rt.start + t) * stride + (int64_t)(kvh * group + rem + f - (t - tok0) * group) * c.hd;
    };
    // ---- queries into shared memory ------------------------------------------
    constexpr int LOADERS = TWO ? 128 : 128 * NS;
    const int loader = TWO ? r : tid;
    bool copied = false;
    if constexpr (!kSplit) {
      copied = flip == 1.f && !((uintptr_t)a.q % 16) && a.q_stride % 8 == 0;
      if (copied) {
#pragma unroll 8
        for (int y = loader; y < PM * 8 * NB; y += LOADERS) {
          const int rr = y / (8 * NB), p = y - rr * 8 * NB, f = my_tile * PM + rr;
          const bool real = f < rows && 8 * p < c.hd;
          copy16_async(smem_u32(q_sm + my_tile * S::QB) + (p >> 3) * PM * 128 + (rr >> 3) * 1024 + (rr & 7) * 128 +
                           (((p & 7) ^ (rr & 7)) << 4),
                       real ? q + row_of(f, a.q_stride) + 8 * p : q, real);
        }
        copies_wait();
      }
    }
    if (!copied) {
      // A warp per row, four values a lane.
      const bool wide = !((uintptr_t)a.q % (4 * sizeof(TQ))) && a.q_stride % 4 == 0;
      constexpr int H = NB <= 2 ? 1 : 2, BATCH = 8, ROWS = 32 * PM / LOADERS;  // rows of a warp
      const int first = loader / 32 * ROWS;
      for (int x0 = 0; x0 < ROWS; x0 += BATCH) {
        float v[BATCH][H][4];
#pragma unroll
        for (int y = 0; y < BATCH; ++y) {
          const int f = my_tile * PM + first + x0 + y;
          const TQ* from = q + row_of(f < rows ? f : 0, a.q_stride);
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const int d = 4 * lane + 128 * h;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[y][h][e] = 0.f;
            if (f < rows && d < c.hd) {
              if (wide) {
                load4(from + d, v[y][h]);
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[y][h][e] = (float)from[d + e];
              }
            }
          }
        }
#pragma unroll
        for (int y = 0; y < BATCH; ++y) {
          const int rr = first + x0 + y;
          float f = 1.f;
          if constexpr (kSplit) {
            // A power of two puts the row's largest value in [2^14, 2^15).
            float amax = 0.f;
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
              for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(v[y][h][e]));
#pragma unroll
            for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            f = pow2_factor(amax);
            if (lane == 0) factor_sh[my_tile][rr] = f;
          }
          f *= flip;
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const int d = 4 * lane + 128 * h;
            if (d >= S::HD) continue;
            uint8_t* to = q_sm + my_tile * (kSplit ? 2 : 1) * S::QB + (d >> 6) * PM * 128 + (rr >> 3) * 1024 +
                          (rr & 7) * 128 + ((((d & 63) >> 3) ^ (rr & 7)) << 4) + (d & 7) * 2;
            float z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = v[y][h][e] * f;
            const uint32_t h0 = pack2<TKV>(z[0], z[1]), h1 = pack2<TKV>(z[2], z[3]);
            *reinterpret_cast<uint2*>(to) = make_uint2(h0, h1);
            if constexpr (kSplit)
              *reinterpret_cast<uint2*>(to + S::QB) = make_uint2(rest2<TKV>(z[0], z[1], h0), rest2<TKV>(z[2], z[3], h1));
          }
        }
      }
    }
    fence_async_shared();
    mbar_arrive(&q_full);
    const int f = my_tile * PM + r;
    const bool real = f < rows;
    const int at = real ? rt.len - rt.count + token(f) : -1;
    const int lo = a.window > 0 ? at - a.window + 1 : 0;
    // Tiles whose positions every row of this tile sees need no mask.
    const int t_at0 = rt.len - rt.count + token(my_tile * PM);
    const int t_lo1 =
        a.window > 0 ? rt.len - rt.count + token(min(rows, (my_tile + 1) * PM) - 1) - a.window + 1 : 0;
    float cq = 0.f, m = -INFINITY, l = 0.f;
    const int mine = tiles_of(w);
    if (mine > 0 && !mbar_wait(&q_full, 0, c.status, W_ATT_PROMPT)) ok = false;
    // Base-2 exponents per score unit (a zero scale has zero queries instead,
    // so that a masked score's -inf survives the product).
    cq = flip == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
    if constexpr (kSplit) cq = __fdiv_rn(cq, factor_sh[my_tile][r]);
    for (int k = 0; k < mine; ++k) {
      const int t = TWO ? k : NS * k + w, j0 = span.start(t, BN);
      if (ok && !mbar_wait(&s_full[w], k & 1, c.status, W_ATT_PROMPT)) ok = false;
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float s[BN];
#pragma unroll
      for (int x = 0; x < BN; x += 32) tmem_ld32(s_t + x, s + x);
      tmem_wait_ld();
      if (j0 + BN - 1 > t_at0 || (j0 < t_lo1 && j0 + BN > a.sinks)) {
        // A bit per position: up to the row's own, and not before its window
        // unless among the first tokens.
        const int hi = at - j0, from = lo - j0, first = a.sinks - j0;
#pragma unroll
        for (int x = 0; x < BN; x += 32) {
          const uint32_t see = low_bits(hi + 1 - x) & (~low_bits(from - x) | low_bits(first - x));
#pragma unroll
          for (int e = 0; e < 32; ++e) s[x + e] = see >> e & 1 ? s[x + e] : -INFINITY;
        }
      }
      float tops[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) tops[x] = s[x];
#pragma unroll
      for (int x = 8; x < BN; x += 2) tops[x / 2 & 7] = max3(tops[x / 2 & 7], s[x], s[x + 1]);
      float top = max3(max3(tops[0], tops[1], tops[2]), max3(tops[3], tops[4], tops[5]), fmaxf(tops[6], tops[7]));
      top = top == -INFINITY ? top : top * cq;
      if (k == 0) {
        m = top;
      } else {
        const bool grow = top > m + kGrow;
        if (__any_sync(0xffffffffu, grow)) {
          // The products before these scores are complete, and the next ones
          // wait for these weights: the accumulator is this warp's for now.
          const float shrink = grow ? exp2_fast(m - top) : 1.f;
          if (grow) m = top;
          l *= shrink;
          for (int x = 0; x < hd16; x += 16) {
            float o[16];
            tmem_ld16(o_t + x, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= shrink;
            tmem_st16(o_t + x, o);
          }
          tmem_wait_st();
        }
      }
      if (t == nt - 1 && j0 + BN > rt.len) {
        // Rows past the sequence's end hold whatever the page held before:
        // zeros in their place (the last V is the last load of the ring).
        const int v_it = 2 * nt - 1, st = v_it % ST;
        if (!mbar_wait(&kv_full[st], (v_it / ST) & 1, c.status, W_ATT_PROMPT)) ok = false;
        uint8_t* v = ring + st * S::KV;
        for (int y = r; y < BN * 8 * NB; y += 128)
          if (j0 + ((y >> 3) & (BN - 1)) >= rt.len) *reinterpret_cast<uint4*>(v + y * 16) = make_uint4(0, 0, 0, 0);
        fence_async_shared();
      }
      const float base = kLift - (m == -INFINITY ? 0.f : m);
      const uint64_t cq2 = f2(cq, cq), base2 = f2(base, base);
      uint64_t sum = 0;
#pragma unroll
      for (int x = 0; x < BN; x += 32) {
        uint32_t p[16], rest[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float2 y = f2(fma2(f2(s[x + 2 * e], s[x + 2 * e + 1]), cq2, base2));
          if (!kSplit && e % kCubicEvery == kCubicEvery - 1) {
            y = exp2_cubic(y);
          } else {
            y.x = exp2_fast(y.x);
            y.y = exp2_fast(y.y);
          }
          sum = add2(sum, f2(y.x, y.y));
          p[e] = pack2<TKV>(y.x, y.y);
          if constexpr (kSplit) rest[e] = rest2<TKV>(y.x, y.y, p[e]);
        }
        tmem_st16(s_t + x / 2, p);
        if constexpr (kSplit) tmem_st16(s_t + BN / 2 + x / 2, rest);
        if (x == BN / 2 - 32 || x == BN - 32) {
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(x == BN - 32 ? &p_full[w] : &p_half[w]);
        }
      }
      l += f2(sum).x + f2(sum).y;
    }
    if (ok && mine > 0 && !mbar_wait(&o_full[w], 0, c.status, W_ATT_PROMPT)) ok = false;
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();

    // ---- the streams' join, and the result -------------------------------------
    float* join = reinterpret_cast<float*>(q_sm);
    float mine_f = 1.f, their_f = 0.f;
    const bool two = NS == 2 && !TWO && nt > 1;
    if (two) {
      // Both streams' products are complete (each waited for its own) when
      // both have come to the first barrier: shared memory is free.
      named_sync(1, 256);
      if (w == 1) {
        join[r * S::JOIN_LD + S::HD] = m;
        join[r * S::JOIN_LD + S::HD + 1] = l;
        for (int x = 0; x < hd16; x += 16) {
          float o[16];
          tmem_ld16(o_t + x, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4*>(join + r * S::JOIN_LD + x + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      }
      named_sync(1, 256);
      if (w == 0) {
        const float m1 = join[r * S::JOIN_LD + S::HD], l1 = join[r * S::JOIN_LD + S::HD + 1], mn = fmaxf(m, m1);
        if (mn != -INFINITY) {
          mine_f = exp2_fast(m - mn);
          their_f = exp2_fast(m1 - mn);
        }
        l = __fmaf_rn(l, mine_f, l1 * their_f);
      }
    }
    if (TWO || w == 0) {
      // Rows go out through shared memory (this warp's 32, 16-byte pieces
      // swizzled), so that a warp's stores cover whole lines.
      const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);
      constexpr int PIECES = S::HD * sizeof(TQ) / 16, PER = 16 / sizeof(TQ);
      uint8_t* stage = q_sm + (TWO ? my_tile * S::QB : S::OUT_AT) +
                       (warp & 3) * 32 * PIECES * 16;
      bool bad = l != l || l == INFINITY;
      for (int x = 0; x < hd16; x += 16) {
        float o[16];
        if (ok && mine > 0) {
          tmem_ld16(o_t + x, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0.f;
        }
        if (two)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __fmaf_rn(o[e], mine_f, join[r * S::JOIN_LD + x + e] * their_f);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          bad |= !(fabsf(o[e]) <= 3.4028234e38f);
          o[e] = l == 0.f ? 0.f : o[e] * inv;
        }
#pragma unroll
        for (int p = 0; p < 16 / PER; ++p)
          store_piece(reinterpret_cast<TQ*>(stage + (lane * PIECES + ((x / PER + p) ^ (lane & 7))) * 16), o + p * PER);
      }
      __syncwarp();
      const bool wide = !((uintptr_t)a.out % 16) && a.out_stride * sizeof(TQ) % 16 == 0;
      const int first = my_tile * PM + 32 * (warp & 3);  // the warp's first row
#pragma unroll 4
      for (int y = lane; y < 32 * PIECES; y += 32) {
        const int row = y / PIECES, p = y - row * PIECES;
        if (first + row >= rows || p * PER >= c.hd) continue;
        TQ* to = static_cast<TQ*>(a.out) + row_of(first + row, a.out_stride) + p * PER;
        const uint8_t* from = stage + (row * PIECES + (p ^ (row & 7))) * 16;
        if (wide) {
          *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
        } else {
#pragma unroll
          for (int e = 0; e < PER; ++e) to[e] = reinterpret_cast<const TQ*>(from)[e];
        }
      }
      __syncwarp();
      // A row that a value beyond its mask has spoilt (or that sees one that is
      // not finite) is computed again by itself.
      for (unsigned again = __ballot_sync(0xffffffffu, ok && real && bad); again; again &= again - 1) {
        const int f1 = first + __ffs(again) - 1;
        prompt_row<TQ, TKV>(a, rt.s, kvh, rt.len - rt.count + token(f1), q + row_of(f1, a.q_stride),
                            static_cast<TQ*>(a.out) + row_of(f1, a.out_stride));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == W_MMA) tmem_free(tmem, 512);
}

template <typename TQ, typename TKV, int NB, bool TWO>
static int launch_prompt(const AttnArgs& a, const KvMaps& maps, cudaStream_t st) {
  using S = PromptShape<TQ, NB, TWO>;
  static PerDeviceOnce attr;
  if (smem_attr_once(attr, attn_prompt_kernel<TQ, TKV, NB, TWO>, S::SMEM) != cudaSuccess) return KC_ERR_CUDA;
  // Every sequence may leave its last tile partly filled.
  const int64_t tiles = (int64_t)a.n_rows * (a.nh / a.c.nkv) / (S::QT * PM) + std::min(a.n, a.n_rows);
  if (tiles * a.c.nkv > INT32_MAX) return KC_ERR_SHAPE;
  launch_k(attn_prompt_kernel<TQ, TKV, NB, TWO>, dim3((unsigned)(tiles * a.c.nkv)), S::THREADS, S::SMEM, st, a, maps);
  return KC_OK;
}

template <typename TQ, typename TKV>
static int launch_prompt_hd(const AttnArgs& a, const KvMaps& maps, cudaStream_t st) {
  // Two row tiles per block read every key and value once for both; with few
  // rows, or f32 queries (two operands each), a block takes one.
  const int64_t pairs = ((int64_t)a.n_rows * (a.nh / a.c.nkv) + 2 * PM - 1) / (2 * PM) * a.c.nkv;
  const bool two = sizeof(TQ) == 2 && pairs >= num_sms();
  switch ((a.c.hd + 63) / 64) {
    case 1:
      if constexpr (sizeof(TQ) == 2)
        if (two) return launch_prompt<TQ, TKV, 1, true>(a, maps, st);
      return launch_prompt<TQ, TKV, 1, false>(a, maps, st);
    case 2:
      if constexpr (sizeof(TQ) == 2)
        if (two) return launch_prompt<TQ, TKV, 2, true>(a, maps, st);
      return launch_prompt<TQ, TKV, 2, false>(a, maps, st);
    case 3: return launch_prompt<TQ, TKV, 3, false>(a, maps, st);
    default: return launch_prompt<TQ, TKV, 4, false>(a, maps, st);
  }
}

int attn_prompt_box_rows(int page, int hd) { return std::min(page, hd <= 128 ? 128 : 64); }

int launch_attn_prompt(const AttnArgs& a, const KvMaps& maps, cudaStream_t st) {
  if (a.c.type == T_BF16) return launch_prompt_hd<__nv_bfloat16, __nv_bfloat16>(a, maps, st);
  if (a.t_q == T_F32) return launch_prompt_hd<float, __half>(a, maps, st);
  return launch_prompt_hd<__half, __half>(a, maps, st);
}

}  // namespace kc
