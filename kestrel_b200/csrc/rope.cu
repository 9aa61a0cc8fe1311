// Rotary positions, on rows of heads and on the way into the pages of a cache.
//
// Pair i of the first dim values of a head at position p turns by p w_i:
//   (a, b) -> gain (a cos - b sin, a sin + b cos).
// The frequencies come as 64-bit fractions of a turn, w_i / 2 pi = turn / 2^64,
// so that the phase is one integer product that drops whole turns by itself: at
// position 2^31 it is still good to 2^-31 of a turn (rope_turns.h), without 64-bit
// floating point. The quadrant is its top two bits; what is left, within an eighth of a
// turn either way, goes to sincospif, good to its last bits.
//
// The memory rate is the floor of both calls (3 operations a value). A block takes a
// few rows: it looks up where each stands and goes, computes the rows' cos and sin
// once into shared memory, and then streams through their heads, 16 bytes of
// 16-bit values a thread at a time (32 of f32) where dim and head_dim allow it, in
// both halves if those are paired. A thread's first loads go out before all that,
// the next ones before the last are turned.
//
// Measured on a B200 (plain copy 6.56 TB/s): 8192 rows of 36 heads of 128, bf16,
// 151 MB in 29.8 us (5.1 TB/s); 24 x 256 rows of 32 and 4 heads of 128, f32 into
// an f16 cache, 239 MB in 44.8 us (5.3). Angles by each thread for up to eight
// heads of its own took 43.6 and 66.8 us, places by division instead of steps 46.4
// and 47.7, pairs turned one by one instead of two at a time 37.3 and 47.0. As
// interleaved pairs, which are turned one by one, the first takes 33.9 us; where dim / 2
// (interleaved: dim) or what does not turn is no multiple of 8, accesses are of two
// columns: 8192 rows of 58 heads of 80, of which 20 turn, bf16, 152 MB in 83 us (70
// interleaved).
#include <algorithm>
#include <type_traits>

#include "attn_dev.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv.h"
#include "kv_dev.cuh"
#include "rope.h"

namespace kc {

constexpr int ROPE_THREADS = 128;
constexpr int ROPE_ROWS = 8;                 // rows of a block, at most
constexpr int ROPE_PAIRS = ROPE_ROWS * 64;   // and their angles

// gain * (cos, sin) of a phase in 64-bit fractions of a turn.
__device__ __forceinline__ float2 cos_sin(uint64_t phase, float gain) {
  const uint32_t quarter = (uint32_t)((phase + (1ull << 61)) >> 62);
  const int64_t rest = (int64_t)(phase - ((uint64_t)quarter << 62));
  float s, c;
  sincospif(__ll2float_rn(rest) * 0x1p-63f, &s, &c);
  const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
  return make_float2((quarter + 1) & 2 ? -x * gain : x * gain, quarter & 2 ? -y * gain : y * gain);
}

// VEC values as they are in memory.
template <int VEC, typename S>
struct alignas(VEC * sizeof(S) < 16 ? VEC * sizeof(S) : 16) Raw {
  S v[VEC];
};
template <int VEC, typename S>
__device__ __forceinline__ Raw<VEC, S> load_vec(const S* p, bool aligned) {
  Raw<VEC, S> r;
  constexpr int BYTES = VEC * sizeof(S);
  if (aligned) {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      r = *reinterpret_cast<const Raw<VEC, S>*>(p);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = p[i];
  }
  return r;
}
template <int VEC, typename D>
__device__ __forceinline__ void store_vec(D* p, const float (&v)[VEC], bool aligned) {
  Raw<VEC, D> r;
  if constexpr (sizeof(D) == 2 && VEC > 1) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) reinterpret_cast<uint32_t*>(&r)[i] = pack2<D>(v[2 * i], v[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = (D)v[i];
  }
  constexpr int BYTES = VEC * sizeof(D);
  if (aligned) {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&r)[i];
    } else {
      *reinterpret_cast<Raw<VEC, D>*>(p) = r;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = r.v[i];
  }
}

// What a thread has of a head: VEC columns from `col` on, and if halves are paired
// VEC more from col + dim / 2 on. Lanes of a head: those that turn, then those of
// the columns behind.
template <int VEC, bool HALF>
struct RopeLane {
  int col, first;  // first: the pair whose angle the first column has; -1: none
  static __host__ __device__ int turning(int dim) { return HALF ? dim / 2 / VEC : dim / VEC; }
  static __host__ __device__ int count(int dim, int hd) { return turning(dim) + (hd - dim) / VEC; }
  __device__ __forceinline__ RopeLane(int lane, int dim) {
    const int t = turning(dim);
    col = lane < t ? lane * VEC : dim + (lane - t) * VEC;
    first = lane < t ? (HALF ? col : col / 2) : -1;
  }
};

// Two consecutive values as an f32 pair, and back.
template <typename S>
__device__ __forceinline__ uint64_t widen2(const S* p) {
  if constexpr (std::is_same_v<S, __nv_bfloat16>) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    return f2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  } else {
    return f2((float)p[0], (float)p[1]);
  }
}

// One thread's values of a head, as they are in memory.
template <int VEC, bool HALF, typename S>
struct RopeValues {
  Raw<VEC, S> x, y;
  __device__ __forceinline__ void load(const S* head, const RopeLane<VEC, HALF>& l, int half, bool aligned) {
    x = load_vec<VEC>(head + l.col, aligned);
    if (HALF && l.first >= 0) y = load_vec<VEC>(head + l.col + half, aligned);
  }
  // cos, sin: of the row's pairs. Halves of two columns or more are turned two pairs
  // at a time.
  template <typename D>
  __device__ __forceinline__ void put(D* head, const RopeLane<VEC, HALF>& l, int half, bool turns, const float* cos,
                                      const float* sin, bool aligned) const {
    float a[VEC], b[VEC];
    if constexpr (HALF && VEC > 1) {
      const uint64_t minus = f2(-1.f, -1.f);
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        uint64_t p = widen2(x.v + i), q = widen2(y.v + i);
        if (turns) {
          const uint64_t c = *reinterpret_cast<const uint64_t*>(cos + l.first + i),
                         s = *reinterpret_cast<const uint64_t*>(sin + l.first + i);
          const uint64_t u = fma2(p, c, mul2(mul2(q, minus), s));
          q = fma2(p, s, mul2(q, c));
          p = u;
        }
        const float2 pf = f2(p), qf = f2(q);
        a[i] = pf.x;
        a[i + 1] = pf.y;
        b[i] = qf.x;
        b[i + 1] = qf.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        a[i] = (float)x.v[i];
        b[i] = HALF ? (float)y.v[i] : 0.f;
      }
      if (turns) {
        if constexpr (HALF) {
          const float p = a[0], q = b[0], c = cos[l.first], s = sin[l.first];
          a[0] = __fmaf_rn(p, c, -(q * s));
          b[0] = __fmaf_rn(p, s, q * c);
        } else {
          const Raw<VEC / 2, float> c = load_vec<VEC / 2>(cos + l.first, true), s = load_vec<VEC / 2>(sin + l.first, true);
#pragma unroll
          for (int i = 0; i < VEC; i += 2) {
            const float p = a[i], q = a[i + 1];
            a[i] = __fmaf_rn(p, c.v[i / 2], -(q * s.v[i / 2]));
            a[i + 1] = __fmaf_rn(p, s.v[i / 2], q * c.v[i / 2]);
          }
        }
      }
    }
    store_vec<VEC>(head + l.col, a, aligned);
    if (HALF && l.first >= 0) store_vec<VEC>(head + l.col + half, b, aligned);
  }
};

// A launch's rows and how they are cut: `rows` rows a block, a row's heads into
// `cuts` blocks.
struct RopeCut {
  int rows, cuts;
};

// The block's work: heads h0 .. h1-1 of rows r0 .. r1-1, angles by `angles`, from
// from(row, head) by put(row, head, values, lane).
template <int VEC, bool HALF, typename S, class From, class Angles, class Put>
__device__ __forceinline__ void rope_block(int dim, int hd, int rows, int h0, int h1, bool aligned, From from,
                                           Angles angles, Put put) {
  const int lanes = RopeLane<VEC, HALF>::count(dim, hd), heads = h1 - h0, half = dim / 2;
  // A thread's place, and how far the next one is: steps with carries, since
  // divisions would take longer than the rotation.
  const uint32_t part = threadIdx.x / (uint32_t)lanes, step = ROPE_THREADS / (uint32_t)lanes;
  int l = threadIdx.x - part * lanes, row = part / (uint32_t)heads, h = part - row * heads;
  const int dl = ROPE_THREADS - step * lanes, dr = step / (uint32_t)heads, dh = step - dr * heads;
  RopeValues<VEC, HALF, S> now;
  if (row < rows) now.load(from(row, h0 + h), RopeLane<VEC, HALF>(l, dim), half, aligned);
  angles();
  while (row < rows) {
    const int row0 = row, head0 = h0 + h;
    const RopeLane<VEC, HALF> lane(l, dim);
    l += dl;
    h += dh;
    row += dr;
    if (l >= lanes) {
      l -= lanes;
      ++h;
    }
    if (h >= heads) {
      h -= heads;
      ++row;
    }
    RopeValues<VEC, HALF, S> next;
    if (row < rows) next.load(from(row, h0 + h), RopeLane<VEC, HALF>(l, dim), half, aligned);
    put(row0, head0, now, lane);
    now = next;
  }
}

// cos and sin of the block's rows into shared memory: [rows][dim / 2] each.
template <class Position>
__device__ __forceinline__ void rope_angles(const RopeParams& r, int rows, float* cos, float* sin, Position position) {
  const int half = r.dim / 2;
  for (int x = threadIdx.x; x < rows * half; x += ROPE_THREADS) {
    const int row = (uint32_t)x / (uint32_t)half;
    const float2 cs = cos_sin((uint64_t)(int64_t)position(row) * r.turn[x - row * half], r.gain);
    cos[x] = cs.x;
    sin[x] = cs.y;
  }
}

template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const __grid_constant__ RopeParams r,
                                                            const int32_t* positions, int n_rows, int n_head, int hd,
                                                            RopeCut cut, const T* x, int64_t xs, T* out, int64_t os,
                                                            bool x_aligned, bool out_aligned) {
  __shared__ __align__(16) float cos_sh[ROPE_PAIRS], sin_sh[ROPE_PAIRS];
  pdl_enter();
  const int half = r.dim / 2, h0 = (int)((int64_t)n_head * blockIdx.y / cut.cuts),
            h1 = (int)((int64_t)n_head * (blockIdx.y + 1) / cut.cuts);
  const int64_t r0 = (int64_t)blockIdx.x * cut.rows;
  const int rows = (int)min((int64_t)cut.rows, n_rows - r0);
  rope_block<VEC, HALF, T>(
      r.dim, hd, rows, h0, h1, x_aligned, [&](int row, int h) { return x + (r0 + row) * xs + (int64_t)h * hd; },
      [&] {
        rope_angles(r, rows, cos_sh, sin_sh, [&](int row) { return positions[r0 + row]; });
        __syncthreads();
      },
      [&](int row, int h, const RopeValues<VEC, HALF, T>& v, const RopeLane<VEC, HALF>& l) {
        v.put(out + (r0 + row) * os + (int64_t)h * hd, l, half, l.first >= 0, cos_sh + row * half, sin_sh + row * half,
              out_aligned);
      });
}

// Rows of k and v into the pages as kv_write_kernel puts them (kv.cu), the keys
// turned by their positions, and the queries beside them to rows of their own.
// Heads of a row: the queries', the keys', the values'.
template <typename S, typename D, int VEC, bool HALF>
__global__ void __launch_bounds__(ROPE_THREADS) kv_append_kernel(const AppendArgs a,
                                                                 const __grid_constant__ RopeParams r, RopeCut cut,
                                                                 bool in_aligned, bool out_aligned, int blocks) {
  __shared__ __align__(16) float cos_sh[ROPE_PAIRS], sin_sh[ROPE_PAIRS];
  __shared__ int pos_sh[ROPE_ROWS], page_sh[ROPE_ROWS];  // a row's position and page; -1: none
  pdl_enter();
  const KvView& c = a.c;
  if (blockIdx.x >= blocks) {
    if (blockIdx.y == 0) kv_report_repeats<ROPE_THREADS>(c, a.seqs, a.n);
    return;
  }
  const int half = r.dim / 2, heads = a.nh + 2 * c.nkv, h0 = (int)((int64_t)heads * blockIdx.y / cut.cuts),
            h1 = (int)((int64_t)heads * (blockIdx.y + 1) / cut.cuts);
  const int64_t r0 = (int64_t)blockIdx.x * cut.rows;
  const int rows = (int)min((int64_t)cut.rows, a.n_rows - r0);
  rope_block<VEC, HALF, S>(
      r.dim, c.hd, rows, h0, h1, in_aligned,
      [&](int row, int h) {
        const int64_t at = r0 + row;
        if (h < a.nh) return static_cast<const S*>(a.q) + at * a.q_stride + (int64_t)h * c.hd;
        if (h < a.nh + c.nkv) return static_cast<const S*>(a.k) + at * a.k_stride + (int64_t)(h - a.nh) * c.hd;
        return static_cast<const S*>(a.v) + at * a.v_stride + (int64_t)(h - a.nh - c.nkv) * c.hd;
      },
      [&] {
        if (threadIdx.x < rows) {
          const int row = (int)r0 + threadIdx.x;
          int i = row, back = 1, wrong = 0, pos = -1, id = -1;  // the row is `back` positions from its sequence's end
          if (a.row_start) {
            i = kv_row_owner(a.row_start, a.n, row);
            if (i < 0) wrong = W_KV_ROWS;
            else back = a.row_start[i + 1] - row;
          }
          const int s = wrong ? -1 : a.seqs ? a.seqs[i] : i;
          if (!wrong && (s < 0 || s >= c.n_seq)) wrong = W_KV_SEQ;
          if (!wrong) {
            pos = kv_len(c, s) - back;
            if (pos < 0) {
              pos = -1;
              wrong = W_KV_ROWS;
            } else {
              id = c.table[(int64_t)s * c.max_pages + (pos >> c.page_log2)];
              if (id < 0 || id >= c.n_pages) {
                id = -1;
                wrong = W_KV_PAGE;
              }
            }
          }
          if (wrong && blockIdx.y == 0) report(c.status, KC_ERR_ARG | (wrong << 8));
          pos_sh[threadIdx.x] = pos;
          page_sh[threadIdx.x] = id;
        }
        __syncthreads();
        rope_angles(r, rows, cos_sh, sin_sh, [&](int row) { return pos_sh[row]; });
        __syncthreads();
      },
      [&](int row, int h, const RopeValues<VEC, HALF, S>& v, const RopeLane<VEC, HALF>& l) {
        const float *cos = cos_sh + row * half, *sin = sin_sh + row * half;
        const int pos = pos_sh[row], id = page_sh[row];
        if (h < a.nh) {
          if (pos >= 0)
            v.put(static_cast<S*>(a.q_out) + (r0 + row) * a.out_stride + (int64_t)h * c.hd, l, half, l.first >= 0, cos,
                  sin, out_aligned);
          return;
        }
        if (id < 0) return;
        const bool is_v = h >= a.nh + c.nkv;
        D* pool = reinterpret_cast<D*>(is_v ? c.v : c.k);
        const int64_t head = ((int64_t)a.layer * c.n_pages + id) * c.nkv + (h - a.nh - (is_v ? c.nkv : 0));
        v.put(pool + (head * c.page + (pos & (c.page - 1))) * c.hd, l, half, l.first >= 0 && !is_v, cos, sin, true);
      });
}

// Columns a thread takes at a time.
static int rope_vec(const RopeParams& r, int hd) {
  const int unit = r.interleaved ? r.dim : r.dim / 2;
  return unit % 8 == 0 && (hd - r.dim) % 8 == 0 ? 8 : unit % 2 == 0 ? 2 : 1;
}

// Rows a block takes: up to eight loads a thread, while that leaves two blocks an SM
// (8192 rows of 36 heads of 128, bf16: two 30.0 us, four 32.5; 24 x 256 rows of 32 and
// 4 heads, f32 to f16: 45.0 and 46.3; blocks of 256 threads 31.0 and 50.3, of 64 32.3
// and 46.0); a row's heads over several blocks where there are fewer rows than SMs.
static RopeCut rope_cut(int n_rows, int heads, int lanes, int dim) {
  const int per = heads * lanes, sms = num_sms();  // (a row has at most 2^24 values)
  RopeCut c{1, 1};
  while (2 * c.rows <= ROPE_ROWS && 2 * c.rows * (dim / 2) <= ROPE_PAIRS && 2 * c.rows * per <= 8 * ROPE_THREADS &&
         n_rows / (2 * c.rows) >= 2 * sms)
    c.rows *= 2;
  if (n_rows < sms) c.cuts = std::max(1, std::min({sms / n_rows, per / ROPE_THREADS, heads}));
  return c;
}
static bool rows_aligned(const void* p, int64_t stride, int hd, size_t el, int vec) {
  const size_t bytes = std::min<size_t>(16, vec * el);
  return (uintptr_t)p % bytes == 0 && stride * el % bytes == 0 && hd * el % bytes == 0;
}

template <int VEC, bool HALF, typename T>
static void rope_run(const RopeParams& r, const int32_t* positions, int n_rows, int n_head, int hd, const void* x,
                     int64_t xs, void* out, int64_t os, cudaStream_t st) {
  const RopeCut cut = rope_cut(n_rows, n_head, RopeLane<VEC, HALF>::count(r.dim, hd), r.dim);
  launch_k(rope_kernel<T, VEC, HALF>, dim3((n_rows + cut.rows - 1) / cut.rows, cut.cuts), ROPE_THREADS, 0, st, r,
           positions, n_rows, n_head, hd, cut, static_cast<const T*>(x), xs, static_cast<T*>(out), os,
           rows_aligned(x, xs, hd, sizeof(T), VEC), rows_aligned(out, os, hd, sizeof(T), VEC));
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
  const RopeCut cut = rope_cut(a.n_rows, a.nh + 2 * c.nkv, RopeLane<VEC, HALF>::count(r.dim, c.hd), r.dim);
  const int grid = (a.n_rows + cut.rows - 1) / cut.rows;
  bool aligned = rows_aligned(a.k, a.k_stride, c.hd, sizeof(S), VEC) && rows_aligned(a.v, a.v_stride, c.hd, sizeof(S), VEC);
  if (a.nh) aligned = aligned && rows_aligned(a.q, a.q_stride, c.hd, sizeof(S), VEC);
  launch_k(kv_append_kernel<S, D, VEC, HALF>, dim3(grid + (a.seqs && a.n > 1), cut.cuts), ROPE_THREADS, 0, st, a, r,
           cut, aligned, a.nh && rows_aligned(a.q_out, a.out_stride, c.hd, sizeof(S), VEC), grid);
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
