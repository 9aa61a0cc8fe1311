// Attention of one new token per sequence over the paged key-value cache,
// split over the cache's length and joined (formulas: attn_prompt.cu).
//
// A decode step reads every visible key and value once and computes 4 flops a
// byte and query head: it is bound by the memory rate, and what matters is that
// all SMs read all the time, however unequal the sequences are. So the work is
// one line of 16-position chunks, sequence after sequence and head after head,
// cut into equal ranges for one block per SM and its warps; a range may begin
// and end inside a sequence. Each warp runs its own ring of chunks (TMA boxes of
// one page's rows, 128-byte swizzle, up to 192 KB in flight per SM) and its own
// softmax state, writes what it has whole, and meets the others once, at the
// end: the parts of a block are joined in shared memory, and those of a sequence
// that several blocks hold in a workspace, by the block that finishes last. Both
// go in the order of the line, so the sums do not depend on timing.
//
// The eight heads of a group share each chunk as the rows of one m16n8k16
// product. f32 queries and the f32 weights are each carried by two 16-bit rows
// (value and rest, 22 bits for f16), which fill the product's other eight rows
// at no cost: results are f32-grade although the cache is 16-bit. Groups of
// more than eight heads with 16-bit queries use all sixteen rows for heads (their
// weights are rounded to the cache's type).
//
// Measured on a B200 (plain copy 6.46 TB/s): 96 sequences of 1500 to 8192 under
// a window of 4096, 8 key-value heads of 128, 1.37 GB in 234 us (5.9 TB/s); one
// of 131071, 4 heads, 268 MB in 56 us (4.8); 32 of 200 to 4096, 126 MB in 34.6 us
// (3.6). Past one round of a block's threads (256 sequences; 128 at head sizes
// past 128) every block walks the list of lengths twice: 1000 of 64, 131 MB in 40
// us (3.3). What is not reading: about 5 us until the first chunks are asked for
// (launch, lengths, ranges, page ids) and 5 to 8 at the end (the last warp, the
// parts, their join through L2).
#include <algorithm>
#include <type_traits>

#include "attn_dev.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv.h"
#include "kv_dev.cuh"

namespace kc {

constexpr int DC = 16;  // positions per chunk: the smallest page
constexpr int DEC_MAX_PARTS = 160;  // most blocks of a launch

template <int NB, int HT>
struct DecShape {
  static constexpr int HD = 64 * NB;                           // padded head size
  static constexpr int W = NB <= 2 ? 8 : 4;                    // warps
  static constexpr int CHUNK = 2 * NB * DC * 128;              // K and V of one chunk
  static constexpr int LD = HD + 4;                            // a head's part: values, maximum, sum, (16-byte rows)
  static constexpr int FIRST = W * HT * LD * 4;                // a part per warp, kept beside the ring
  static constexpr int FIT = (225 * 1024 - FIRST) / (W * CHUNK);
  static constexpr int ST = FIT < 6 ? FIT : 6;                 // ring stages per warp
  static constexpr int SMEM = W * ST * CHUNK + FIRST + 1024;
  // After the chunks: a warp's last part where its ring was, and behind warp
  // 0's what each part counts for, and each unit's maxima and sums.
  static_assert(HT * LD * 4 + 2 * W * HT * 12 <= ST * CHUNK, "fits");
  static_assert(2 * HT <= 32, "a thread per part and head");
};

struct DecArgs {
  AttnArgs a;
  float* part;  // [grid][2][HT][LD]
  int* count;   // [grid], zero between launches
  SharedArgs sh;  // of calls with prefixes that are computed elsewhere
};

// Entry i's sequence, and the positions before its own part (SHARED).
template <bool SHARED>
__device__ __forceinline__ int dec_seq(const DecArgs& d, int i) {
  return d.a.seqs ? d.a.seqs[i] : SHARED ? d.sh.e0 + i : i;
}
template <bool SHARED>
__device__ __forceinline__ int dec_before(const DecArgs& d, int i) {
  return SHARED ? d.sh.of_entry[d.sh.e0 + i] : 0;
}

// Chunks of the visible positions of a sequence of `len` positions as seen from
// its last one: `head` chunks of the first tokens, then those from w0 on.
struct Span {
  int head, w0, n, lo;
};
template <bool SHARED>
__device__ __forceinline__ Span dec_span(int len, int window, int sinks, int before) {
  Span s;
  if constexpr (SHARED) {
    // (A prefix is whole pages, and of a sequence that goes on behind it.)
    s.lo = s.head = 0;
    s.w0 = before / DC;
  } else {
    s.lo = window > 0 ? max(0, len - window) : 0;
    s.head = (min(sinks, s.lo) + DC - 1) / DC;
    s.w0 = max(s.lo / DC, s.head);
  }
  s.n = len > 0 ? s.head + (len + DC - 1) / DC - s.w0 : 0;
  return s;
}

// a / b for a >= 0, b > 0: in 32 bits where they fit (a 64-bit division takes
// several times as long, and half a dozen stand before the first load).
__device__ __forceinline__ long long div_ll(long long a, long long b) {
  return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

// A warp's range of the line, segment by segment (one segment: consecutive
// chunks of one unit, a unit being a sequence's key-value head and head tile).
struct SegIter {
  long long pos, end, base;  // base: line position of sequence i's first unit
  int i, pad;                // pad: chunks each unit takes of the line (0: as many as it has)
  int s, len;
  Span span;
  // the segment
  int unit, c0, c1, n_unit;
  long long unit_at;  // line position of the unit's first chunk
};

template <bool SHARED>
__device__ __forceinline__ void seg_sequence(SegIter& t, const DecArgs& d) {
  const AttnArgs& a = d.a;
  t.s = dec_seq<SHARED>(d, t.i);
  t.len = t.s >= 0 && t.s < a.c.n_seq ? kv_len(a.c, t.s) : 0;
  t.span = dec_span<SHARED>(t.len, a.window, a.sinks, dec_before<SHARED>(d, t.i));
}
template <bool SHARED>
__device__ __forceinline__ bool seg_next(SegIter& t, const DecArgs& d, int units) {
  const AttnArgs& a = d.a;
  while (t.pos < t.end) {
    const int np = t.pad ? t.pad : t.span.n;
    const long long off = t.pos - t.base;  // (a sequence's stretch fits 31 bits: the host sees to it)
    if (off >= np * units) {
      t.base += np * units;
      if (++t.i >= a.n) return false;
      seg_sequence<SHARED>(t, d);
      continue;
    }
    t.unit = (int)((uint32_t)off / (uint32_t)np);
    t.c0 = (int)off - t.unit * np;
    const int take = (int)min(t.end - t.pos, (long long)(np - t.c0));
    t.unit_at = t.pos - t.c0;
    t.c1 = min(t.c0 + take, t.span.n);
    t.n_unit = t.span.n;
    t.pos += take;
    if (t.c0 < t.c1) return true;
  }
  return false;
}

// What a warp has of a unit that it does not hold whole.
struct DecPart {
  int have, i, unit, n_unit;
  long long unit_at;
};

// SHARED: results go to the join (attn_shared.cu) as f32 rows, behind the parts of
// the prefix: the values, then at HD the maximum (in exponents of 2) and sum.
template <int HD>
__device__ __forceinline__ float* own_row(const DecArgs& d, int i, int head) {
  return d.sh.part + (((int64_t)d.sh.splits * (d.sh.e1 - d.sh.e0) + i) * d.a.nh + head) * (HD + 8);
}

template <typename TQ, typename TKV, int NB, int HT, bool SHARED>
__global__ void __launch_bounds__(32 * DecShape<NB, HT>::W, 1)
    attn_decode_kernel(const DecArgs d, const __grid_constant__ KvMaps maps) {
  using S = DecShape<NB, HT>;
  constexpr int W = S::W, ST = S::ST, RH = HT / 8, LD = S::LD;
  constexpr bool kSplit = HT == 8;               // rows 8 .. 15 carry the rests
  constexpr bool kHalf = std::is_same_v<TKV, __half>;
  constexpr float kLift = kHalf ? 15.f : 0.f;    // f16 weights up to 2^15: small ones keep their bits
  // SHARED: beside the prefixes' kernel, whose blocks have all seen the end of what
  // came before it when these start (the fence: nor does this SM hold anything older);
  // it is waited for at the end.
  if constexpr (SHARED) {
    pdl_trigger();
    __threadfence();
  } else {
    pdl_enter();
  }
  extern __shared__ uint8_t dec_raw[];
  __shared__ __align__(8) uint64_t full[W][ST];
  __shared__ long long red[3][W], found_at[W];
  __shared__ int found[W];
  __shared__ DecPart parts_sh[2 * W];  // per warp: of its range's first segment, and of its last
  __shared__ int last_sh[2];
  const AttnArgs& a = d.a;
  const KvView& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ring = dec_raw + ((1024 - (smem_u32(dec_raw) & 1023)) & 1023);
  float* firsts = reinterpret_cast<float*>(ring + W * ST * S::CHUNK);
  const int group = a.nh / c.nkv, tiles = (group + HT - 1) / HT, units = c.nkv * tiles;
  // SHARED: the other blocks' SMs are the prefixes'.
  const int blocks = SHARED ? min((int)gridDim.x, d.sh.plan[PLAN_OWN]) : gridDim.x;
  if (SHARED && blockIdx.x >= blocks) {
    pdl_wait();
    return;
  }
  if (lane == 0) {
    for (int s = 0; s < ST; ++s) mbar_init(&full[warp][s], 1);
    fence_mbar_init();
  }

  // ---- the line, and this block's range of it --------------------------------
  // Chunks of all sequences, and the longest one. On the way the rows of
  // sequences that hold nothing become zeros. One round of the block's threads
  // covers 32 W sequences; `here` and `before` are of the last round.
  long long sum = 0, before = 0;
  int most = 0, here = 0;
  for (int i0 = 32 * warp; i0 < a.n; i0 += 32 * W) {
    const int i = i0 + lane;
    here = 0;
    bool none = false;
    if (i < a.n) {
      const int s = dec_seq<SHARED>(d, i);
      const bool real = s >= 0 && s < c.n_seq;
      if (real) here = dec_span<SHARED>(kv_len(c, s), a.window, a.sinks, dec_before<SHARED>(d, i)).n;
      else if (blockIdx.x == 0) report(c.status, KC_ERR_ARG | (W_KV_SEQ << 8));
      none = real && here == 0 && i % blocks == blockIdx.x;
    }
    for (unsigned rows = __ballot_sync(0xffffffffu, none); rows; rows &= rows - 1) {
      if constexpr (SHARED) {
        for (int h = lane; h < a.nh; h += 32)
          *reinterpret_cast<float2*>(own_row<S::HD>(d, i0 + __ffs(rows) - 1, h) + S::HD) = make_float2(-INFINITY, 0.f);
        continue;
      }
      TQ* out = static_cast<TQ*>(a.out) + (int64_t)(i0 + __ffs(rows) - 1) * a.out_stride;
      for (int x = lane; x < a.nh * c.hd; x += 32) out[x] = (TQ)0.f;
    }
    sum += here;
    most = max(most, here);
  }
  {
    // Sequences before this thread's among its warp's, and the warp's sum.
    long long x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    before = x - here;
#pragma unroll
    for (int o = 16; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 31) red[0][warp] = x;
    if (lane == 0) {
      red[1][warp] = most;
      found[warp] = a.n;  // (a range past the line has no sequence)
    }
  }
  __syncthreads();
  long long line = 0;
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += red[0][w];
    line += red[0][w];
    most = max(most, (int)red[1][w]);
  }
  line *= units;
  if (line == 0) {
    if constexpr (SHARED) pdl_wait();
    return;
  }
  // Equal ranges of at least one chunk per warp. When the units are few, each
  // is cut into the same whole number of parts instead (its stretch of the line
  // padded to `pad` chunks) where that is not slower: ranges that begin with
  // their unit have one segment instead of two or three, and a unit in one part
  // needs no join. (A segment's end and a join take about as long as two and
  // four more rounds of chunks: 32 sequences of 2048 positions took 37 us in
  // equal ranges and 29 in one part each.)
  long long per = max(div_ll(line + blocks - 1, blocks), (long long)W);
  per = (per + W - 1) / W * W;
  const long long all = (long long)a.n * units;
  int pad = 0;
  if (all <= blocks) {
    const int parts = (int)((uint32_t)blocks / (uint32_t)all);
    const int q = ((most + parts - 1) / parts + W - 1) / W * W;
    if (q <= per + (parts == 1 ? 6 : 2) * W) {
      per = q;
      pad = q * ((most + q - 1) / q);
      line = all * pad;
    }
  }
  const long long block_at = blockIdx.x * per, block_end = min(line, block_at + per), share_of = per / W;
  if (block_at >= block_end) {
    if constexpr (SHARED) pdl_wait();
    return;
  }
  SegIter at;
  // A block of one unit's part deals its chunks to the warps in turn (so that
  // they read side by side: 131071 positions took 56.5 us, in stretches 57.2);
  // otherwise each warp has a stretch of the range.
  const int stride = pad ? W : 1, mine = pad ? warp : 0;
  at.pos = pad ? block_at : min(block_end, block_at + warp * share_of);
  at.end = pad ? block_end : min(block_end, at.pos + share_of);
  at.pad = pad;
  // The sequence in which each warp's range begins: the last whose first chunk
  // is at or before it.
  if (pad) {
    at.i = (int)div_ll(at.pos, (long long)pad * units);
    at.base = (long long)at.i * pad * units;
  } else {
    // Exactly one sequence holds each position.
    auto look = [&](int i, long long first, int n) {
      for (int w = 0; w < W; ++w) {
        const long long pos = block_at + w * share_of - first * units;
        if (pos >= 0 && pos < (long long)n * units) {
          found[w] = i;
          found_at[w] = first * units;
        }
      }
    };
    if (a.n <= 32 * W) {
      look(tid, before, here);
    } else {
      long long base = 0;  // chunks of the sequences before the 32 * W at hand
      for (int b = 0; b < a.n && base * units < block_end; b += 32 * W) {
        const int i = b + tid;
        int n = 0;
        if (i < a.n) {
          const int s = dec_seq<SHARED>(d, i);
          if (s >= 0 && s < c.n_seq) n = dec_span<SHARED>(kv_len(c, s), a.window, a.sinks, dec_before<SHARED>(d, i)).n;
        }
        long long x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) red[2][warp] = x;
        __syncthreads();
        long long mine = base + x - n;
        for (int w = 0; w < W; ++w) {
          if (w < warp) mine += red[2][w];
          base += red[2][w];
        }
        look(i, mine, n);
      }
    }
    __syncthreads();
    at.i = found[warp];
    at.base = found_at[warp];
    if (at.i >= a.n) at.pos = at.end;
  }
  if (at.pos < at.end) seg_sequence<SHARED>(at, d);

  // ---- queries ------------------------------------------------------------------
  // A segment's, as this lane holds them in A fragments (row r0, and r0 + 8 in
  // the form of 16 heads; columns cc, cc + 1 of each 8). They are asked for a
  // segment ahead, where there are registers for it: behind the chunks under way
  // a load takes as long as those.
  const int r0 = lane >> 2, cc = 2 * (lane & 3);  // fragment row and first column
  constexpr bool kAhead = NB <= 2;
  alignas(8) TQ raw[RH][4 * NB][4];
  using Pair = std::conditional_t<sizeof(TQ) == 4, float2, uint32_t>;
  const bool pairs = !((uintptr_t)a.q % sizeof(Pair)) && a.q_stride % 2 == 0;  // two columns a load
  auto ask = [&](const SegIter& g) {
    const int kvh = g.unit / tiles, h0 = (g.unit - kvh * tiles) * HT;
    const TQ* q = static_cast<const TQ*>(a.q) + (int64_t)g.i * a.q_stride + (int64_t)(kvh * group + h0) * c.hd;
#pragma unroll
    for (int rr = 0; rr < RH; ++rr) {
      const bool real = h0 + r0 + 8 * rr < group;
      const TQ* row = q + (real ? (int64_t)(r0 + 8 * rr) * c.hd : 0) + cc;
      if (pairs) {
#pragma unroll
        for (int ks = 0; ks < 4 * NB; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            Pair v{};
            if (real && 16 * ks + 8 * e + cc < c.hd) v = *reinterpret_cast<const Pair*>(row + 16 * ks + 8 * e);
            *reinterpret_cast<Pair*>(&raw[rr][ks][2 * e]) = v;
          }
      } else {
#pragma unroll
        for (int ks = 0; ks < 4 * NB; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int x = 16 * ks + (e & 1) + 8 * (e >> 1);
            raw[rr][ks][e] = real && x + cc < c.hd ? row[x] : (TQ)0.f;
          }
      }
    }
  };
  SegIter ahead = at;  // what is loaded next
  bool more = seg_next<SHARED>(ahead, d, units), have = more;
  SegIter to_come = ahead;  // the segment after the one at hand
  if (kAhead && have) ask(to_come);

  // ---- this warp's ring ---------------------------------------------------------
  int next = ahead.c0 + mine, issued = 0, used = 0;
  bool ok = true;
  uint8_t* slots = ring + warp * ST * S::CHUNK;
  // The next chunk: first position, sequence and head. False when there is none.
  auto plan = [&](int& p, int& s, int& head) {
    while (more && next >= ahead.c1) {
      more = seg_next<SHARED>(ahead, d, units);
      next = ahead.c0 + mine;
    }
    if (!more) return false;
    p = (next < ahead.span.head ? next : next - ahead.span.head + ahead.span.w0) * DC;
    s = ahead.s;
    head = ahead.unit / tiles;
    next += stride;
    ++issued;
    return true;
  };
  auto load = [&](int st, int p, int s, int head) {
    const int id = c.table[(int64_t)s * c.max_pages + (p >> c.page_log2)];
    int lp = a.layer * c.n_pages + id;
    if (id < 0 || id >= c.n_pages) {
      report(c.status, KC_ERR_ARG | (W_KV_PAGE << 8));
      lp = c.n_layer * c.n_pages;  // past the pool: zeros
    }
    uint8_t* to = slots + st * S::CHUNK;
    mbar_expect_tx(&full[warp][st], S::CHUNK);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      kv_load(to + b * DC * 128, &maps.k, 64 * b, p & (c.page - 1), head, lp, &full[warp][st]);
      kv_load(to + (NB + b) * DC * 128, &maps.v, 64 * b, p & (c.page - 1), head, lp, &full[warp][st]);
    }
  };
  if (lane < 2) parts_sh[2 * warp + lane].have = 0;
  __syncwarp();
  {
    // The first ones at once, a lane per stage.
    int p = 0, s = 0, head = 0;
    bool go = false;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      int p1, s1, head1;
      if (plan(p1, s1, head1) && lane == st) {
        p = p1;
        s = s1;
        head = head1;
        go = true;
      }
    }
    if (go) load(lane, p, s, head);
  }
  __syncwarp();

  const float log2e = 1.4426950408889634f;
  while (have) {
    at = to_come;
    if (!kAhead) ask(at);
    const int kvh = at.unit / tiles, h0 = (at.unit - kvh * tiles) * HT;
    uint32_t qa[4 * NB][4];
    float cq[RH];  // base-2 exponents per score unit
#pragma unroll
    for (int rr = 0; rr < RH; ++rr) {
      float f = 1.f;
      if constexpr (sizeof(TQ) == 4) {
        // A power of two puts the row's largest value in [2^14, 2^15).
        float amax = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4 * NB; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf((float)raw[rr][ks][e]));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        f = pow2_factor(amax);
      }
      cq[rr] = __fdiv_rn(a.scale * log2e, f);
#pragma unroll
      for (int ks = 0; ks < 4 * NB; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float x = (float)raw[rr][ks][2 * e] * f, y = (float)raw[rr][ks][2 * e + 1] * f;
          const uint32_t hi = pack2<TKV>(x, y);
          if constexpr (kSplit) {
            qa[ks][2 * e] = hi;
            qa[ks][2 * e + 1] = sizeof(TQ) == 4 ? rest2<TKV>(x, y, hi) : 0u;
          } else {
            qa[ks][2 * e + rr] = hi;
          }
        }
    }
    have = seg_next<SHARED>(to_come, d, units);
    if (kAhead && have) ask(to_come);
    float m[RH], l[RH], o[8 * NB][4];
#pragma unroll
    for (int rr = 0; rr < RH; ++rr) {
      m[rr] = -INFINITY;
      l[rr] = 0.f;
    }
#pragma unroll
    for (int t = 0; t < 8 * NB; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][e] = 0.f;

    for (int x = at.c0 + mine; x < at.c1; x += stride) {
      const int st = used % ST;
      if (ok && !mbar_wait(&full[warp][st], (used / ST) & 1, c.status, W_ATT_DEC)) ok = false;
      if (!ok) break;
      ++used;
      const uint32_t kb = smem_u32(slots + st * S::CHUNK), vb = kb + NB * DC * 128;
      const int ch = x < at.span.head ? x : x - at.span.head + at.span.w0, p0 = ch * DC;
      // Scores: 16 rows x 16 positions (two column tiles).
      float sc[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[t][e] = 0.f;
      {
        // ldmatrix: lanes 8 g .. 8 g + 7 address the rows of matrix g: positions
        // 8 (g / 2) .., dims 8 (g % 2) ..
        const int pr = (lane & 7) + 8 * (lane >> 4), g = (lane >> 3) & 1;
#pragma unroll
        for (int ks = 0; ks < 4 * NB; ++ks) {
          const int u = 2 * (ks & 3) + g;
          uint32_t b[4];
          ldsm4(b, kb + (ks >> 2) * DC * 128 + pr * 128 + ((u ^ (pr & 7)) << 4));
          mma16816<TKV>(sc[0], qa[ks], b[0], b[1]);
          mma16816<TKV>(sc[1], qa[ks], b[2], b[3]);
        }
      }
      // Rows of this thread: rr; its positions: p0 + 8 t + cc + e.
      float tt[RH][4];
#pragma unroll
      for (int rr = 0; rr < RH; ++rr)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            tt[rr][2 * t + e] = (kSplit ? with_rest(sc[t][e], sc[t][e + 2]) : sc[t][e + 2 * rr]) * cq[rr];
      const bool edge = p0 + DC > at.len || (p0 < at.span.lo && p0 + DC > a.sinks);
      if (edge) {
        // Positions that the row does not see: no weight, and zeros in place of
        // their values (what a page holds there may be NaN).
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = p0 + 8 * t + cc + e;
            if (j >= at.len || (j < at.span.lo && j >= a.sinks))
#pragma unroll
              for (int rr = 0; rr < RH; ++rr) tt[rr][2 * t + e] = -INFINITY;
          }
        for (int y = lane; y < DC * 8 * NB; y += 32) {
          const int r = (y >> 3) & (DC - 1), j = p0 + r;
          if (j >= at.len || (j < at.span.lo && j >= a.sinks))
            *reinterpret_cast<uint4*>(slots + st * S::CHUNK + NB * DC * 128 + y * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_shared();  // before the slot's next load
        __syncwarp();
      }
      uint32_t pa[4];
#pragma unroll
      for (int rr = 0; rr < RH; ++rr) {
        float top = fmaxf(fmaxf(tt[rr][0], tt[rr][1]), fmaxf(tt[rr][2], tt[rr][3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (__any_sync(0xffffffffu, top > m[rr])) {
          const float mn = fmaxf(m[rr], top), shrink = mn == -INFINITY ? 1.f : exp2_fast(m[rr] - mn);
          m[rr] = mn;
          l[rr] *= shrink;
#pragma unroll
          for (int t = 0; t < 8 * NB; ++t) {
            o[t][2 * rr] *= shrink;
            o[t][2 * rr + 1] *= shrink;
            if constexpr (kSplit) {
              o[t][2] *= shrink;
              o[t][3] *= shrink;
            }
          }
        }
        const float base = (m[rr] == -INFINITY ? 0.f : m[rr]) - kLift;
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = exp2_fast(tt[rr][e] - base);
          l[rr] += p[e];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t hi = pack_weights<TKV>(p[2 * t], p[2 * t + 1]);
          if constexpr (kSplit) {
            pa[2 * t] = hi;
            pa[2 * t + 1] = rest2<TKV>(p[2 * t], p[2 * t + 1], hi);
          } else {
            pa[2 * t + rr] = hi;
          }
        }
      }
      {
        const int pr = (lane & 7) + 8 * ((lane >> 3) & 1), g = lane >> 4;
        // Added here, rounded to nearest: products that add to the sum cut its last
        // bits off, 2^-24 of it per chunk, always towards zero (32 sequences of
        // 131071, 1800 chunks a warp: 6e-5 where f32 sums are 2e-7 off, as here).
#pragma unroll
        for (int t = 0; t < 4 * NB; ++t) {
          const int u = 2 * (t & 3) + g;
          uint32_t b[4];
          ldsm4t(b, vb + (t >> 2) * DC * 128 + pr * 128 + ((u ^ (pr & 7)) << 4));
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float d[4];
            mma16816_only<TKV>(d, pa, b[2 * y], b[2 * y + 1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[2 * t + y][e] += d[e];
          }
        }
      }
      __syncwarp();
      {
        int p1, s1, head1;
        const int slot = issued % ST;
        if (plan(p1, s1, head1) && lane == 0) load(slot, p1, s1, head1);
      }
    }

    // ---- the result, or this warp's part of it ------------------------------------
#pragma unroll
    for (int rr = 0; rr < RH; ++rr) {
      l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 1);
      l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 2);
    }
    if constexpr (kSplit)
#pragma unroll
      for (int t = 0; t < 8 * NB; ++t) {
        o[t][0] = with_rest(o[t][0], o[t][2]);
        o[t][1] = with_rest(o[t][1], o[t][3]);
      }
    if (!pad && at.c0 == 0 && at.c1 == at.n_unit) {
      TQ* out = static_cast<TQ*>(a.out) + (int64_t)at.i * a.out_stride + (int64_t)(kvh * group + h0) * c.hd;
#pragma unroll
      for (int rr = 0; rr < RH; ++rr) {
        const int h = r0 + 8 * rr;
        if (h0 + h >= group) continue;
        const float inv = l[rr] == 0.f ? 0.f : __fdiv_rn(1.f, l[rr]);
        if constexpr (SHARED) {
          float* row = own_row<S::HD>(d, at.i, kvh * group + h0 + h);
#pragma unroll
          for (int t = 0; t < 8 * NB; ++t)
            *reinterpret_cast<float2*>(row + 8 * t + cc) = make_float2(o[t][2 * rr] * inv, o[t][2 * rr + 1] * inv);
          if ((lane & 3) == 0) *reinterpret_cast<float2*>(row + S::HD) = make_float2(m[rr] - kLift, l[rr]);
          continue;
        }
#pragma unroll
        for (int t = 0; t < 8 * NB; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (8 * t + cc + e < c.hd) out[(int64_t)h * c.hd + 8 * t + cc + e] = (TQ)(o[t][2 * rr + e] * inv);
      }
      continue;
    }
    // The last segment's part goes where the ring was: its loads have all come.
    const int which = have ? 0 : 1;
    float* to = which ? reinterpret_cast<float*>(slots) : firsts + warp * HT * LD;
#pragma unroll
    for (int rr = 0; rr < RH; ++rr) {
      float* row = to + (r0 + 8 * rr) * LD;
#pragma unroll
      for (int t = 0; t < 8 * NB; ++t)
        *reinterpret_cast<float2*>(row + 8 * t + cc) = make_float2(o[t][2 * rr], o[t][2 * rr + 1]);
      if ((lane & 3) == 0) *reinterpret_cast<float2*>(row + S::HD) = make_float2(m[rr], l[rr]);
    }
    if (lane == 0) parts_sh[2 * warp + which] = DecPart{1, at.i, at.unit, at.n_unit, at.unit_at};
  }
  // A failed wait leaves loads in flight: they land before the block goes on.
  if (!ok)
    for (; used < issued; ++used) mbar_wait(&full[warp][used % ST], (used / ST) & 1, c.status, W_ATT_DEC);

  // ---- the block's parts, unit by unit in the order of the line --------------------
  __syncthreads();
  auto part_at = [&](int x) {
    return x & 1 ? reinterpret_cast<const float*>(ring + (x >> 1) * ST * S::CHUNK) : firsts + (x >> 1) * HT * LD;
  };
  // What each part counts for in its unit; the unit's maximum and sum (by its
  // first part).
  float2(*unit_sh)[HT] = reinterpret_cast<float2(*)[HT]>(ring + HT * LD * 4);
  float(*share_sh)[HT] = reinterpret_cast<float(*)[HT]>(ring + HT * LD * 4 + 2 * W * HT * 8);
  unsigned held, heads;  // entries that hold a part; that hold their unit's first
  {
    const bool have_part = lane < 2 * W && parts_sh[lane & (2 * W - 1)].have;
    held = __ballot_sync(0xffffffffu, have_part);
    const int before_me = 31 - __clz(held & ((1u << lane) - 1));
    const DecPart* me = parts_sh + (lane & (2 * W - 1));
    const DecPart* prev = parts_sh + max(before_me, 0);
    heads = __ballot_sync(0xffffffffu,
                          have_part && (before_me < 0 || prev->i != me->i || prev->unit != me->unit));
  }
  // Entries of the unit that begins at e: those before the next one's first.
  auto unit_of = [&](int e) {
    const unsigned later = heads & ~((2u << e) - 1);
    return held & ~((1u << e) - 1) & (later ? (later & -later) - 1 : 0xffffffffu);
  };
  if (tid < 2 * W * HT) {  // (whole warps)
    const int e = tid & (2 * W - 1), h = tid / (2 * W);
    const bool mine_held = held >> e & 1;
    const float2 ml = mine_held ? *reinterpret_cast<const float2*>(part_at(e) + h * LD + S::HD)
                                : make_float2(-INFINITY, 0.f);
    const int e0 = 31 - __clz(heads & ((2u << e) - 1));
    const unsigned all_of = mine_held ? unit_of(e0) : 0;
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int k = 0; k < 2 * W; ++k) {
      const float v = __shfl_sync(0xffffffffu, ml.x, k, 2 * W);
      if (all_of >> k & 1) top = fmaxf(top, v);
    }
    const float share = mine_held ? exp2_fast(ml.x - (top == -INFINITY ? 0.f : top)) : 0.f;
#pragma unroll
    for (int k = 0; k < 2 * W; ++k) {
      const float v = __shfl_sync(0xffffffffu, share * ml.y, k, 2 * W);
      if (all_of >> k & 1) total += v;
    }
    if (mine_held) {
      share_sh[e][h] = share;
      if (e == e0) unit_sh[e][h] = make_float2(top, total);
    }
  }
  __syncthreads();
  constexpr int QUADS = HT * S::HD / 4;
  int cut[2] = {-1, -1};  // units that other blocks hold too: their first entry
  for (unsigned left = heads; left; left &= left - 1) {
    const int e = __ffs(left) - 1;
    const unsigned all_of = unit_of(e);
    const DecPart g = parts_sh[e];
    const bool whole = g.unit_at >= block_at && g.unit_at + g.n_unit <= block_at + per;
    const int kvh = g.unit / tiles, h0 = (g.unit - kvh * tiles) * HT;
    TQ* out = static_cast<TQ*>(a.out) + (int64_t)g.i * a.out_stride + (int64_t)(kvh * group + h0) * c.hd;
    // A cut unit's place: 0 if it is the block's first, else 1.
    const int slot = g.unit_at <= block_at ? 0 : 1;
    if (!whole) cut[slot] = e;
    for (int x = tid; x < QUADS; x += 32 * W) {
      const int h = x / (S::HD / 4), y = 4 * (x - h * (S::HD / 4));
      const float2 ml = unit_sh[e][h];
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (unsigned k = all_of; k; k &= k - 1) {
        const int at_k = __ffs(k) - 1;
        const float4 u = *reinterpret_cast<const float4*>(part_at(at_k) + h * LD + y);
        const float w = share_sh[at_k][h];
        v.x = __fmaf_rn(w, u.x, v.x);
        v.y = __fmaf_rn(w, u.y, v.y);
        v.z = __fmaf_rn(w, u.z, v.z);
        v.w = __fmaf_rn(w, u.w, v.w);
      }
      if (whole) {
        if (h0 + h >= group || y >= c.hd) continue;
        const float inv = ml.y == 0.f ? 0.f : __fdiv_rn(1.f, ml.y);
        if constexpr (SHARED) {
          float* row = own_row<S::HD>(d, g.i, kvh * group + h0 + h);
          *reinterpret_cast<float4*>(row + y) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
          if (y == 0) *reinterpret_cast<float2*>(row + S::HD) = make_float2(ml.x - kLift, ml.y);
          continue;
        }
        TQ* to = out + (int64_t)h * c.hd + y;
        to[0] = (TQ)(v.x * inv);
        to[1] = (TQ)(v.y * inv);
        to[2] = (TQ)(v.z * inv);
        to[3] = (TQ)(v.w * inv);
      } else {
        float* to = d.part + ((int64_t)(2 * blockIdx.x + slot) * HT + h) * LD;
        *reinterpret_cast<float4*>(to + y) = v;
        if (y == 0) *reinterpret_cast<float2*>(to + S::HD) = ml;
      }
    }
  }
  if (cut[0] < 0 && cut[1] < 0) {
    if constexpr (SHARED) pdl_wait();
    return;
  }

  // ---- units of several blocks: the last to come joins the parts ---------------------
  __threadfence();
  __syncthreads();
  if (tid < 2) {
    last_sh[tid] = 0;
    if (cut[tid] >= 0) {
      const DecPart g = parts_sh[cut[tid]];
      const int b0 = (int)div_ll(g.unit_at, per), b1 = (int)div_ll(g.unit_at + g.n_unit - 1, per);
      last_sh[tid] = atomicAdd(d.count + b0, 1) == b1 - b0;
      if (last_sh[tid]) d.count[b0] = 0;
    }
  }
  __syncthreads();
  for (int side = 0; side < 2; ++side) {
    if (!last_sh[side]) continue;
    __threadfence();
    const DecPart g = parts_sh[cut[side]];
    const int b0 = (int)div_ll(g.unit_at, per), parts = (int)div_ll(g.unit_at + g.n_unit - 1, per) - b0 + 1;
    const int kvh = g.unit / tiles, h0 = (g.unit - kvh * tiles) * HT;
    TQ* out = static_cast<TQ*>(a.out) + (int64_t)g.i * a.out_stride + (int64_t)(kvh * group + h0) * c.hd;
    // Parts in block order; the unit is the first of every block but b0, where
    // it is unless it begins inside the block's range.
    const int first = 2 * b0 + (g.unit_at == b0 * per ? 0 : 1);
    auto part_of = [&](int p) { return d.part + (int64_t)(p == 0 ? first : 2 * (b0 + p)) * HT * LD; };
    // First every part's share of each head's result (a warp per head, the
    // parts over its lanes), then the sums over the parts.
    float* share = firsts;  // [HT][parts]
    __syncthreads();
    for (int h = warp; h < HT; h += W) {
      float2 ml[DEC_MAX_PARTS / 32];
      float top = -INFINITY, total = 0.f;
#pragma unroll
      for (int u = 0; u < DEC_MAX_PARTS / 32; ++u) {
        const int p = lane + 32 * u;
        ml[u] = p < parts ? __ldcg(reinterpret_cast<const float2*>(part_of(p) + h * LD + S::HD))
                          : make_float2(-INFINITY, 0.f);
        top = fmaxf(top, ml[u].x);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int u = 0; u < DEC_MAX_PARTS / 32; ++u) {
        ml[u].x = exp2_fast(ml[u].x - base);
        total = __fmaf_rn(ml[u].x, ml[u].y, total);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      const float inv = total == 0.f ? 0.f : __fdiv_rn(1.f, total);
      if constexpr (SHARED)
        if (lane == 0 && h0 + h < group)
          *reinterpret_cast<float2*>(own_row<S::HD>(d, g.i, kvh * group + h0 + h) + S::HD) = make_float2(top - kLift, total);
#pragma unroll
      for (int u = 0; u < DEC_MAX_PARTS / 32; ++u)
        if (lane + 32 * u < parts) share[h * parts + lane + 32 * u] = ml[u].x * inv;
    }
    __syncthreads();
    for (int x = tid; x < QUADS; x += 32 * W) {
      const int h = x / (S::HD / 4), y = 4 * (x - h * (S::HD / 4));
      if (h0 + h >= group || y >= c.hd) continue;
      float4 sum4 = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int p0 = 0; p0 < parts; p0 += 16) {  // sixteen parts' loads at once
        float4 v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k)
          v[k] = p0 + k < parts ? __ldcg(reinterpret_cast<const float4*>(part_of(p0 + k) + h * LD + y))
                                : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float w = p0 + k < parts ? share[h * parts + p0 + k] : 0.f;
          sum4.x = __fmaf_rn(w, v[k].x, sum4.x);
          sum4.y = __fmaf_rn(w, v[k].y, sum4.y);
          sum4.z = __fmaf_rn(w, v[k].z, sum4.z);
          sum4.w = __fmaf_rn(w, v[k].w, sum4.w);
        }
      }
      if constexpr (SHARED) {
        *reinterpret_cast<float4*>(own_row<S::HD>(d, g.i, kvh * group + h0 + h) + y) = sum4;
        continue;
      }
      TQ* to = out + (int64_t)h * c.hd + y;
      to[0] = (TQ)sum4.x;
      to[1] = (TQ)sum4.y;
      to[2] = (TQ)sum4.z;
      to[3] = (TQ)sum4.w;
    }
  }
  if constexpr (SHARED) pdl_wait();
}

size_t attn_decode_part_bytes() { return (size_t)num_sms() * 2 * 16 * (256 + 4) * sizeof(float); }

template <typename TQ, typename TKV, int NB, int HT, bool SHARED>
static int launch_decode(const DecArgs& d, const KvMaps& maps, cudaStream_t st) {
  using S = DecShape<NB, HT>;
  static_assert(S::ST >= 2 && S::SMEM <= 226 * 1024, "two stages fit");
  static PerDeviceOnce attr;
  if (smem_attr_once(attr, attn_decode_kernel<TQ, TKV, NB, HT, SHARED>, S::SMEM) != cudaSuccess) return KC_ERR_CUDA;
  const int64_t units = (int64_t)d.a.n * d.a.c.nkv * ((d.a.nh / d.a.c.nkv + HT - 1) / HT);
  const int64_t most = (int64_t)d.a.c.max_pages * d.a.c.page / DC;
  if (most * (units / d.a.n) > INT32_MAX - 8 * num_sms()) return KC_ERR_SHAPE;  // chunks of a sequence, all heads
  // One block per SM, fewer when the tables hold less than a chunk per warp of each.
  const int grid = (int)std::min<int64_t>(std::min(num_sms(), DEC_MAX_PARTS), units * ((most + S::W - 1) / S::W));
  launch_k(attn_decode_kernel<TQ, TKV, NB, HT, SHARED>, grid, 32 * S::W, S::SMEM, st, d, maps);
  return KC_OK;
}

template <typename TQ, typename TKV, int HT, bool SHARED>
static int launch_decode_hd(const DecArgs& d, const KvMaps& maps, cudaStream_t st) {
  switch ((d.a.c.hd + 63) / 64) {
    case 1: return launch_decode<TQ, TKV, 1, HT, SHARED>(d, maps, st);
    case 2: return launch_decode<TQ, TKV, 2, HT, SHARED>(d, maps, st);
    case 3: return launch_decode<TQ, TKV, 3, HT, SHARED>(d, maps, st);
    default: return launch_decode<TQ, TKV, 4, HT, SHARED>(d, maps, st);
  }
}

template <bool SHARED>
static int launch_decode_types(const DecArgs& d, const KvMaps& maps, cudaStream_t st) {
  const AttnArgs& a = d.a;
  const bool many = a.nh / a.c.nkv > 8;
  if (a.c.type == T_BF16)
    return many ? launch_decode_hd<__nv_bfloat16, __nv_bfloat16, 16, SHARED>(d, maps, st)
                : launch_decode_hd<__nv_bfloat16, __nv_bfloat16, 8, SHARED>(d, maps, st);
  if (a.t_q == T_F32) return launch_decode_hd<float, __half, 8, SHARED>(d, maps, st);
  return many ? launch_decode_hd<__half, __half, 16, SHARED>(d, maps, st)
              : launch_decode_hd<__half, __half, 8, SHARED>(d, maps, st);
}

int launch_attn_decode(const AttnArgs& a, const KvMaps& maps, float* part, int* count, cudaStream_t st) {
  return launch_decode_types<false>(DecArgs{a, part, count, {}}, maps, st);
}

int launch_attn_own(const AttnArgs& a, const SharedArgs& sh, const KvMaps& maps, float* part, int* count,
                    cudaStream_t st) {
  return launch_decode_types<true>(DecArgs{a, part, count, sh}, maps, st);
}

}  // namespace kc
