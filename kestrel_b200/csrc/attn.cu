// Attention over the paged key-value cache (kv.h).
//
// For query row r of a sequence with c rows and len positions, i = len - c + r
// and over its visible positions j (j <= i, and j > i - window or j < sinks):
//   s_j = scale * q . k_j,  m = max s_j,  p_j = exp(s_j - m),
//   out = sum p_j v_j / sum p_j;  zeros where nothing is visible.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "kv.h"
#include "kv_dev.cuh"

namespace kc {

// One block per 32 query rows of one key-value head; a row is a (token, query
// head of the group) pair, tokens outermost. Tiles of 32 positions pass
// through shared memory once for all 32 rows, with the running maximum and sum
// of each row kept in f32 (one pass over the cache).
constexpr int AT_ROWS = 32, AT_KEYS = 32, AT_THREADS = 256, AT_HD = 256;

template <typename TQ, typename TKV>
__global__ void __launch_bounds__(AT_THREADS) attn_tile_kernel(AttnArgs a) {
  pdl_enter();
  extern __shared__ float at_smem[];
  const KvView& c = a.c;
  const int hd = c.hd, ld = hd + 1, group = a.nh / c.nkv, kvh = blockIdx.y, tid = threadIdx.x;
  float* qs = at_smem;               // [32][ld]
  float* ks = qs + AT_ROWS * ld;     // [32][ld]
  float* vs = ks + AT_KEYS * ld;     // [32][ld]
  __shared__ float ss[AT_ROWS][AT_KEYS + 1];
  __shared__ int page_of[AT_KEYS];
  // The block's sequence and its first row within it.
  int i = -1, row0 = 0, start = 0, count = 0;
  {
    int t = blockIdx.x;
    for (int e = 0; e < a.n; ++e) {
      const int lo = a.row_start[e], hi = a.row_start[e + 1];
      if (lo < 0 || hi < lo || hi > a.n_rows) {
        if (tid == 0) report(c.status, KC_ERR_ARG | (W_KV_ROWS << 8));
        return;
      }
      const int tiles = ((hi - lo) * group + AT_ROWS - 1) / AT_ROWS;
      if (t < tiles) {
        i = e;
        row0 = t * AT_ROWS;
        start = lo;
        count = hi - lo;
        break;
      }
      t -= tiles;
    }
    if (i < 0) return;
  }
  const int s = a.seqs ? a.seqs[i] : i;
  if (s < 0 || s >= c.n_seq) {
    if (tid == 0) report(c.status, KC_ERR_ARG | (W_KV_SEQ << 8));
    return;
  }
  const int len = kv_len(c, s);
  const int rows = min(AT_ROWS, count * group - row0);
  const int first = len - count + row0 / group, last = len - count + (row0 + rows - 1) / group;  // query positions
  const TQ* q = static_cast<const TQ*>(a.q);
  for (int x = tid; x < AT_ROWS * hd; x += AT_THREADS) {
    const int r = x / hd, d = x - r * hd, f = row0 + r;
    qs[r * ld + d] = r < rows ? (float)q[(int64_t)(start + f / group) * a.q_stride +
                                         (int64_t)(kvh * group + f % group) * hd + d]
                              : 0.f;
  }
  const int r = tid / 8, sub = tid % 8;
  const int at = r < rows ? len - count + (row0 + r) / group : -1;
  float m = -INFINITY, l = 0.f, o[AT_HD / 8];
#pragma unroll
  for (int u = 0; u < AT_HD / 8; ++u) o[u] = 0.f;
  const int lo = a.window > 0 ? max(0, first - a.window + 1) : 0;
  const TKV* kp = reinterpret_cast<const TKV*>(c.k);
  const TKV* vp = reinterpret_cast<const TKV*>(c.v);
  for (int t0 = 0; t0 <= last; t0 += AT_KEYS) {
    if (t0 + AT_KEYS <= lo && t0 >= a.sinks) continue;
    __syncthreads();
    if (tid < AT_KEYS) {
      const int j = t0 + tid;
      int id = j <= last ? c.table[(int64_t)s * c.max_pages + (j >> c.page_log2)] : -1;
      if (j <= last && (id < 0 || id >= c.n_pages)) {
        report(c.status, KC_ERR_ARG | (W_KV_PAGE << 8));
        id = -1;
      }
      page_of[tid] = id;
    }
    __syncthreads();
    for (int x = tid; x < AT_KEYS * hd; x += AT_THREADS) {
      const int j = x / hd, d = x - j * hd, id = page_of[j];
      const int64_t e = ((((int64_t)a.layer * c.n_pages + id) * c.nkv + kvh) * c.page + ((t0 + j) & (c.page - 1))) * hd + d;
      ks[j * ld + d] = id >= 0 ? (float)kp[e] : 0.f;
      vs[j * ld + d] = id >= 0 ? (float)vp[e] : 0.f;
    }
    __syncthreads();
    float top = m;
#pragma unroll
    for (int u = 0; u < AT_KEYS / 8; ++u) {
      const int jj = sub + 8 * u, j = t0 + jj;
      const bool see = j <= at && page_of[jj] >= 0 && (a.window <= 0 || j > at - a.window || j < a.sinks);
      float acc = 0.f;
      for (int d = 0; d < hd; ++d) acc = __fmaf_rn(qs[r * ld + d], ks[jj * ld + d], acc);
      acc = see ? acc * a.scale : -INFINITY;
      ss[r][jj] = acc;
      top = fmaxf(top, acc);
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    __syncwarp();
    const float base = top == -INFINITY ? 0.f : top, shrink = expf(m - base);
    m = top;
    l *= shrink;
#pragma unroll
    for (int u = 0; u < AT_HD / 8; ++u) o[u] *= shrink;
    for (int jj = 0; jj < AT_KEYS; ++jj) {
      const int j = t0 + jj;
      if (!(j <= at && page_of[jj] >= 0 && (a.window <= 0 || j > at - a.window || j < a.sinks))) continue;
      const float p = expf(ss[r][jj] - base);
      l += p;
#pragma unroll
      for (int u = 0; u < AT_HD / 8; ++u)
        if (sub + 8 * u < hd) o[u] = __fmaf_rn(p, vs[jj * ld + sub + 8 * u], o[u]);
    }
  }
  if (r < rows) {
    const int f = row0 + r;
    TQ* out = static_cast<TQ*>(a.out) + (int64_t)(start + f / group) * a.out_stride +
              (int64_t)(kvh * group + f % group) * hd;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int u = 0; u < AT_HD / 8; ++u)
      if (sub + 8 * u < hd) out[sub + 8 * u] = (TQ)(l == 0.f ? 0.f : o[u] * inv);
  }
}

template <typename TQ, typename TKV>
static int launch_tile(const AttnArgs& a, cudaStream_t st) {
  const int group = a.nh / a.c.nkv;
  const int64_t blocks = ((int64_t)a.n_rows * group + AT_ROWS - 1) / AT_ROWS + a.n;
  static PerDeviceOnce attr;
  const size_t smem = (size_t)(AT_ROWS + 2 * AT_KEYS) * (a.c.hd + 1) * 4;
  if (smem_attr_once(attr, attn_tile_kernel<TQ, TKV>, (AT_ROWS + 2 * AT_KEYS) * (AT_HD + 1) * 4) != cudaSuccess)
    return KC_ERR_CUDA;
  launch_k(attn_tile_kernel<TQ, TKV>, dim3((unsigned)blocks, a.c.nkv), AT_THREADS, smem, st, a);
  return KC_OK;
}

int launch_attn_prompt(const AttnArgs& a, cudaStream_t st) {
  if (a.c.type == T_BF16) return launch_tile<__nv_bfloat16, __nv_bfloat16>(a, st);
  if (a.t_q == T_F32) return launch_tile<float, __half>(a, st);
  return launch_tile<__half, __half>(a, st);
}

}  // namespace kc
