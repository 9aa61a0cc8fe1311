// Rotary positions, on rows of heads and on the way into the pages of a cache.
//
// Pair i of the first dim values of a head at position p turns by p w_i:
//   (a, b) -> gain (a cos - b sin, a sin + b cos).
// The frequencies come as 64-bit fractions of a turn, w_i / 2 pi = turn / 2^64,
// so that the phase is one integer product that drops whole turns by itself: at
// position 2^31 it is still good to 2^-34 of a turn, without 64-bit floating
// point. The quadrant is its top two bits; what is left, within an eighth of a
// turn either way, goes to sincospif, good to its last bits.
//
// Both calls are bound by the memory rate (3 operations a value). A thread takes
// the same columns of several heads of a row, so that their cos and sin are
// computed once for all of these: 8 columns (16 bytes of 16-bit values) at a time
// where dim and head_dim allow it, in both halves if those are paired.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "kv.h"
#include "kv_dev.cuh"
#include "rope.h"

#pragma nv_diag_suppress 20208  // (long double: on the host only)

namespace kc {

constexpr int ROPE_THREADS = 128;

RopeParams make_rope(int dim, bool interleaved, float base, int scaling, float factor, int original, float low,
                     float high, float gain, const float* freq_factors) {
  const long double two_pi = 2 * acosl(-1.0L), s = factor, len = original;
  RopeParams r{};
  r.dim = dim;
  r.interleaved = interleaved;
  r.gain = gain != 0.f ? gain : scaling == ROPE_YARN ? (float)(1 + 0.1L * logl(s)) : 1.f;
  long double from = 0, to = 0;
  if (scaling == ROPE_YARN) {
    const auto pair_of = [&](long double turns) { return dim * logl(len / (two_pi * turns)) / (2 * logl(base)); };
    from = std::max(0.0L, floorl(pair_of(high)));
    to = std::min((long double)dim - 1, ceill(pair_of(low)));
  }
  for (int i = 0; i < dim / 2; ++i) {
    long double w = powl(base, -2.0L * i / dim);
    if (freq_factors) w /= freq_factors[i];
    if (scaling == ROPE_LINEAR) {
      w /= s;
    } else if (scaling == ROPE_YARN) {
      const long double part = std::min(1.0L, std::max(0.0L, (i - from) / std::max(0.001L, to - from)));
      w *= part / s + 1 - part;
    } else if (scaling == ROPE_BANDS) {
      const long double z = std::min(1.0L, std::max(0.0L, (len * w / two_pi - low) / ((long double)high - low)));
      w *= z + (1 - z) / s;
    }
    long double turn = w / two_pi;
    turn -= floorl(turn);  // whole turns a position change nothing
    r.turn[i] = (uint64_t)(int64_t)llrintl(ldexpl(turn - (turn >= 0.5L ? 1 : 0), 64));
  }
  return r;
}

// gain * (cos, sin) of a phase in 64-bit fractions of a turn.
__device__ __forceinline__ float2 cos_sin(uint64_t phase, float gain) {
  const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
  const int64_t rest = (int64_t)(phase - ((uint64_t)quarter << 62));
  float s, c;
  sincospif(__ll2float_rn(rest) * 0x1p-63f, &s, &c);
  const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
  return make_float2((quarter + 1) & 2 ? -x * gain : x * gain, quarter & 2 ? -y * gain : y * gain);
}

template <int VEC, typename S>
__device__ __forceinline__ void load_vec(const S* p, float (&v)[VEC], bool aligned) {
  alignas(16) S in[VEC];
  constexpr int BYTES = VEC * sizeof(S);
  if (aligned && BYTES >= 4) {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(in)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(in) = *reinterpret_cast<const uint2*>(p);
    } else if constexpr (BYTES == 4) {
      *reinterpret_cast<uint32_t*>(in) = *reinterpret_cast<const uint32_t*>(p);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) in[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = (float)in[i];
}
template <int VEC, typename D>
__device__ __forceinline__ void store_vec(D* p, const float (&v)[VEC], bool aligned) {
  alignas(16) D o[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) o[i] = (D)v[i];
  constexpr int BYTES = VEC * sizeof(D);
  if (aligned && BYTES >= 4) {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(o)[i];
    } else if constexpr (BYTES == 8) {
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(o);
    } else if constexpr (BYTES == 4) {
      *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(o);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = o[i];
  }
}

// What a thread has of each head of its chunk: VEC columns from `col` on, and if
// halves are paired VEC more from col2 on (-1: none), turned or as they are.
template <int VEC, bool HALF>
struct RopeLane {
  static constexpr int ANGLES = HALF ? VEC : (VEC + 1) / 2;
  int col, col2;
  bool turns;
  float2 cs[ANGLES];

  // Lanes of a head: those that turn, then those of the columns behind.
  static __host__ __device__ int turning(int dim) { return HALF ? dim / 2 / VEC : dim / VEC; }
  static __host__ __device__ int count(int dim, int hd) { return turning(dim) + (hd - dim) / VEC; }

  __device__ __forceinline__ void place(int lane, int dim) {
    const int t = turning(dim);
    turns = lane < t;
    col = turns ? lane * VEC : dim + (lane - t) * VEC;
    col2 = HALF && turns ? dim / 2 + lane * VEC : -1;
  }
  __device__ __forceinline__ void angles(const RopeParams& r, int position) {
    const int first = HALF ? col : col / 2;
#pragma unroll
    for (int i = 0; i < ANGLES; ++i) cs[i] = cos_sin((uint64_t)(int64_t)position * r.turn[first + i], r.gain);
  }
  template <typename S>
  __device__ __forceinline__ void load(const S* head, float (&x)[VEC], float (&y)[VEC], bool aligned) const {
    load_vec<VEC>(head + col, x, aligned);
    if (HALF && col2 >= 0) load_vec<VEC>(head + col2, y, aligned);
  }
  __device__ __forceinline__ void turn(float (&x)[VEC], float (&y)[VEC]) const {
    if constexpr (HALF) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float a = x[i], b = y[i];
        x[i] = __fmaf_rn(a, cs[i].x, -(b * cs[i].y));
        y[i] = __fmaf_rn(a, cs[i].y, b * cs[i].x);
      }
    } else if constexpr (VEC > 1) {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        const float a = x[i], b = x[i + 1];
        x[i] = __fmaf_rn(a, cs[i / 2].x, -(b * cs[i / 2].y));
        x[i + 1] = __fmaf_rn(a, cs[i / 2].y, b * cs[i / 2].x);
      }
    }
  }
  template <typename D>
  __device__ __forceinline__ void store(D* head, const float (&x)[VEC], const float (&y)[VEC], bool aligned) const {
    store_vec<VEC>(head + col, x, aligned);
    if (HALF && col2 >= 0) store_vec<VEC>(head + col2, y, aligned);
  }
};

// `heads` heads from head(0), head(1) .. to to(0), to(1) ..: loads of two at once.
template <int VEC, bool HALF, typename Head, typename To>
__device__ __forceinline__ void rope_heads(const RopeLane<VEC, HALF>& lane, int heads, bool turns, bool in_aligned,
                                           bool out_aligned, Head head, To to) {
  for (int h = 0; h < heads; h += 2) {
    float x[2][VEC], y[2][VEC];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (h + u < heads) lane.load(head(h + u), x[u], y[u], in_aligned);
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (h + u < heads) {
        if (turns) lane.turn(x[u], y[u]);
        lane.store(to(h + u), x[u], y[u], out_aligned);
      }
  }
}

template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const __grid_constant__ RopeParams r,
                                                            const int32_t* positions, int n_rows, int n_head, int hd,
                                                            int chunk, const T* x, int64_t xs, T* out, int64_t os,
                                                            bool x_aligned, bool out_aligned) {
  pdl_enter();
  const int lanes = RopeLane<VEC, HALF>::count(r.dim, hd), chunks = (n_head + chunk - 1) / chunk;
  const int64_t all = (int64_t)n_rows * chunks * lanes;
  for (int64_t i = (int64_t)blockIdx.x * ROPE_THREADS + threadIdx.x; i < all; i += (int64_t)gridDim.x * ROPE_THREADS) {
    const int64_t part = i / lanes;
    const int row = (int)(part / chunks), h0 = (int)(part - (int64_t)row * chunks) * chunk;
    RopeLane<VEC, HALF> lane;
    lane.place((int)(i - part * lanes), r.dim);
    if (lane.turns) lane.angles(r, positions[row]);
    const T* from = x + row * xs + (int64_t)h0 * hd;
    T* to = out + row * os + (int64_t)h0 * hd;
    rope_heads(lane, min(chunk, n_head - h0), lane.turns, x_aligned, out_aligned,
               [&](int h) { return from + (int64_t)h * hd; }, [&](int h) { return to + (int64_t)h * hd; });
  }
}

// Rows of k and v into the pages as kv_write_kernel puts them (kv.cu), the keys
// turned by their positions, and the queries beside them to rows of their own.
// Chunks of a row: the queries' heads, the keys', the values'.
template <typename S, typename D, int VEC, bool HALF>
__global__ void __launch_bounds__(ROPE_THREADS) kv_append_kernel(const AppendArgs a,
                                                                 const __grid_constant__ RopeParams r, int chunk,
                                                                 bool in_aligned, bool out_aligned, int blocks) {
  pdl_enter();
  const KvView& c = a.c;
  if (blockIdx.x >= blocks) {
    kv_report_repeats<ROPE_THREADS>(c, a.seqs, a.n);
    return;
  }
  const int lanes = RopeLane<VEC, HALF>::count(r.dim, c.hd);
  const int of_q = (a.nh + chunk - 1) / chunk, of_k = (c.nkv + chunk - 1) / chunk, chunks = of_q + 2 * of_k;
  const int64_t all = (int64_t)a.n_rows * chunks * lanes;
  for (int64_t x = (int64_t)blockIdx.x * ROPE_THREADS + threadIdx.x; x < all; x += (int64_t)blocks * ROPE_THREADS) {
    const int64_t part = x / lanes;
    const int row = (int)(part / chunks), l = (int)(x - part * lanes);
    int at = (int)(part - (int64_t)row * chunks);
    const bool tell = at == chunks - 1 && l == 0;  // (one thread a row reports)
    int i = row, back = 1;  // the row is `back` positions from its sequence's end
    if (a.row_start) {
      i = kv_row_owner(a.row_start, a.n, row);
      if (i < 0) {
        if (tell) report(c.status, KC_ERR_ARG | (W_KV_ROWS << 8));
        continue;
      }
      back = a.row_start[i + 1] - row;
    }
    const int s = a.seqs ? a.seqs[i] : i;
    if (s < 0 || s >= c.n_seq) {
      if (tell) report(c.status, KC_ERR_ARG | (W_KV_SEQ << 8));
      continue;
    }
    const int pos = kv_len(c, s) - back;
    if (pos < 0) {
      if (tell) report(c.status, KC_ERR_ARG | (W_KV_ROWS << 8));
      continue;
    }
    RopeLane<VEC, HALF> lane;
    lane.place(l, r.dim);
    const bool is_v = at >= of_q + of_k, turns = lane.turns && !is_v;
    if (turns) lane.angles(r, pos);
    if (at < of_q) {
      const int h0 = at * chunk;
      const S* from = static_cast<const S*>(a.q) + row * a.q_stride + (int64_t)h0 * c.hd;
      S* to = static_cast<S*>(a.q_out) + row * a.out_stride + (int64_t)h0 * c.hd;
      rope_heads(lane, min(chunk, a.nh - h0), turns, in_aligned, out_aligned,
                 [&](int h) { return from + (int64_t)h * c.hd; }, [&](int h) { return to + (int64_t)h * c.hd; });
      continue;
    }
    const int id = c.table[(int64_t)s * c.max_pages + (pos >> c.page_log2)];
    if (id < 0 || id >= c.n_pages) {
      if (tell) report(c.status, KC_ERR_ARG | (W_KV_PAGE << 8));
      continue;
    }
    at -= is_v ? of_q + of_k : of_q;
    const int h0 = at * chunk;
    const S* from = (is_v ? static_cast<const S*>(a.v) + row * a.v_stride : static_cast<const S*>(a.k) + row * a.k_stride) +
                    (int64_t)h0 * c.hd;
    const int64_t step = (int64_t)c.page * c.hd;  // from a head's row to the next one's
    D* to = reinterpret_cast<D*>(is_v ? c.v : c.k) + (((int64_t)a.layer * c.n_pages + id) * c.nkv + h0) * step +
            (int64_t)(pos & (c.page - 1)) * c.hd;
    rope_heads(lane, min(chunk, c.nkv - h0), turns, in_aligned, true,
               [&](int h) { return from + (int64_t)h * c.hd; }, [&](int h) { return to + h * step; });
  }
}

// Columns a thread takes at a time.
static int rope_vec(const RopeParams& r, int hd) {
  const int unit = r.interleaved ? r.dim : r.dim / 2;
  return unit % 8 == 0 && (hd - r.dim) % 8 == 0 ? 8 : unit % 2 == 0 ? 2 : 1;
}

// Heads of a thread: more where there are threads enough without, since their
// angles are computed once.
static int rope_chunk(int64_t threads, int most) {
  int chunk = 1;
  while (chunk < most && chunk < 8 && threads / (2 * chunk) >= (int64_t)num_sms() * 1024) chunk *= 2;
  return chunk;
}
static bool rows_aligned(const void* p, int64_t stride, int hd, size_t el, int vec) {
  const size_t bytes = std::min<size_t>(16, vec * el);
  return (uintptr_t)p % bytes == 0 && stride * el % bytes == 0 && hd * el % bytes == 0;
}

template <int VEC, bool HALF, typename T>
static void rope_run(const RopeParams& r, const int32_t* positions, int n_rows, int n_head, int hd, const void* x,
                     int64_t xs, void* out, int64_t os, cudaStream_t st) {
  const int lanes = RopeLane<VEC, HALF>::count(r.dim, hd);
  const int chunk = rope_chunk((int64_t)n_rows * n_head * lanes, n_head);
  const int64_t all = (int64_t)n_rows * ((n_head + chunk - 1) / chunk) * lanes;
  const int grid = (int)std::min<int64_t>((all + ROPE_THREADS - 1) / ROPE_THREADS, 32 * (int64_t)num_sms());
  launch_k(rope_kernel<T, VEC, HALF>, grid, ROPE_THREADS, 0, st, r, positions, n_rows, n_head, hd, chunk,
           static_cast<const T*>(x), xs, static_cast<T*>(out), os, rows_aligned(x, xs, hd, sizeof(T), VEC),
           rows_aligned(out, os, hd, sizeof(T), VEC));
}

// fn<VEC, HALF>() for a rotation and head size. (Interleaved pairs are at least
// two columns.)
template <class Fn>
static void rope_shape(const RopeParams& r, int hd, Fn&& fn) {
  const int vec = rope_vec(r, hd);
  using std::bool_constant;
  using std::integral_constant;
  if (r.interleaved) {
    if (vec == 8) fn(integral_constant<int, 8>{}, bool_constant<false>{});
    else fn(integral_constant<int, 2>{}, bool_constant<false>{});
  } else {
    if (vec == 8) fn(integral_constant<int, 8>{}, bool_constant<true>{});
    else if (vec == 2) fn(integral_constant<int, 2>{}, bool_constant<true>{});
    else fn(integral_constant<int, 1>{}, bool_constant<true>{});
  }
}

void launch_rope(const RopeParams& r, const int32_t* positions, int n_rows, int n_head, int hd, int t, const void* x,
                 int64_t xs, void* out, int64_t os, cudaStream_t st) {
  rope_shape(r, hd, [&](auto vec, auto half) {
    constexpr int VEC = decltype(vec)::value;
    constexpr bool HALF = decltype(half)::value;
    if (t == T_F32) rope_run<VEC, HALF, float>(r, positions, n_rows, n_head, hd, x, xs, out, os, st);
    else if (t == T_F16) rope_run<VEC, HALF, __half>(r, positions, n_rows, n_head, hd, x, xs, out, os, st);
    else rope_run<VEC, HALF, __nv_bfloat16>(r, positions, n_rows, n_head, hd, x, xs, out, os, st);
  });
}

template <int VEC, bool HALF, typename S, typename D>
static void append_run(const AppendArgs& a, const RopeParams& r, cudaStream_t st) {
  const KvView& c = a.c;
  const int lanes = RopeLane<VEC, HALF>::count(r.dim, c.hd);
  const int chunk = rope_chunk((int64_t)a.n_rows * (a.nh + 2 * c.nkv) * lanes, c.nkv);
  const int chunks = (a.nh + chunk - 1) / chunk + 2 * ((c.nkv + chunk - 1) / chunk);
  const int64_t all = (int64_t)a.n_rows * chunks * lanes;
  const int grid = (int)std::min<int64_t>((all + ROPE_THREADS - 1) / ROPE_THREADS, 32 * (int64_t)num_sms());
  bool aligned = rows_aligned(a.k, a.k_stride, c.hd, sizeof(S), VEC) && rows_aligned(a.v, a.v_stride, c.hd, sizeof(S), VEC);
  if (a.nh) aligned = aligned && rows_aligned(a.q, a.q_stride, c.hd, sizeof(S), VEC);
  launch_k(kv_append_kernel<S, D, VEC, HALF>, grid + (a.seqs && a.n > 1), ROPE_THREADS, 0, st, a, r, chunk, aligned,
           a.nh && rows_aligned(a.q_out, a.out_stride, c.hd, sizeof(S), VEC), grid);
}

void launch_kv_append(const AppendArgs& a, const RopeParams& r, int t, cudaStream_t st) {
  rope_shape(r, a.c.hd, [&](auto vec, auto half) {
    constexpr int VEC = decltype(vec)::value;
    constexpr bool HALF = decltype(half)::value;
    if (a.c.type == T_F16) {
      if (t == T_F32) append_run<VEC, HALF, float, __half>(a, r, st);
      else append_run<VEC, HALF, __half, __half>(a, r, st);
    } else {
      if (t == T_F32) append_run<VEC, HALF, float, __nv_bfloat16>(a, r, st);
      else append_run<VEC, HALF, __nv_bfloat16, __nv_bfloat16>(a, r, st);
    }
  });
}

}  // namespace kc
