// Page operations of the paged key-value cache (kv.h): fork, extend, free,
// compact, copy and the writing of new rows.
//
// The page state (table, len, refs) lives on the device and is changed in
// stream order, so that a decode step needs no host round trip. Allocation is
// deterministic: the lowest free pages, in the order of the call. There is no
// free list to keep in step: a page is free when refs says 0, and the few
// kernels that look for free or live pages scan refs (4 bytes a page).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "kv.h"
#include "kv_dev.cuh"

namespace kc {

constexpr int KV_BLOCK = 1024;  // threads of the single-block metadata kernels

// Exclusive sum of v over the block's threads; `total` gets the sum.
__device__ __forceinline__ long long block_scan(long long v, long long& total) {
  __shared__ long long part[KV_BLOCK / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  if (lane == 31) part[warp] = s;
  __syncthreads();
  if (warp == 0) {
    long long p = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long t = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += t;
    }
    part[lane] = p;
  }
  __syncthreads();
  const long long base = warp ? part[warp - 1] : 0;
  total = part[KV_BLOCK / 32 - 1];
  __syncthreads();
  return base + s - v;
}

__device__ __forceinline__ int held_pages(const KvView& c, int len) { return (len + c.page - 1) >> c.page_log2; }

// ---- fork --------------------------------------------------------------------
// One block per pair. A destination must be empty and appear once, and not
// among the sources; a pair that breaks this is reported and left out.
__global__ void kv_fork_kernel(KvView c, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int n) {
  pdl_enter();
  const int i = blockIdx.x, s = src[i], d = dst[i];
  __shared__ int bad;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  if (s < 0 || s >= c.n_seq || d < 0 || d >= c.n_seq) {
    if (threadIdx.x == 0) report(c.status, KC_ERR_ARG | (W_KV_SEQ << 8));
    return;
  }
  for (int j = threadIdx.x; j < n; j += blockDim.x)
    if (src[j] == d || dst[j] == s || (j < i && dst[j] == d)) bad = 1;
  const int len = kv_len(c, s);
  if (threadIdx.x == 0 && c.len[d] != 0) bad = 1;
  __syncthreads();
  if (bad) {
    if (threadIdx.x == 0) report(c.status, KC_ERR_ARG | (W_KV_FORK << 8));
    return;
  }
  const int32_t* from = c.table + (int64_t)s * c.max_pages;
  int32_t* to = c.table + (int64_t)d * c.max_pages;
  for (int p = threadIdx.x; p < held_pages(c, len); p += blockDim.x) {
    const int id = from[p];
    to[p] = id;
    if (id >= 0 && id < c.n_pages) atomicAdd(c.refs + id, 1);
    else report(c.status, KC_ERR_ARG | (W_KV_PAGE << 8));
  }
  if (threadIdx.x == 0) c.len[d] = len;
}

void launch_kv_fork(const KvView& c, const int32_t* src, const int32_t* dst, int n, cudaStream_t st) {
  launch_k(kv_fork_kernel, n, 128, 0, st, c, src, dst, n);
}

// ---- free --------------------------------------------------------------------
__global__ void kv_free_kernel(KvView c, const int32_t* __restrict__ seqs, const int32_t* __restrict__ keep, int n) {
  pdl_enter();
  const int i = blockIdx.x, s = seqs ? seqs[i] : i;
  __shared__ int bad;
  if (threadIdx.x == 0) bad = s < 0 || s >= c.n_seq;
  __syncthreads();
  if (seqs)
    for (int j = threadIdx.x; j < i; j += blockDim.x)
      if (seqs[j] == s) bad = 1;
  __syncthreads();
  const int want = keep ? keep[i] : 0;
  if (bad || want < 0) {
    if (threadIdx.x == 0) report(c.status, KC_ERR_ARG | ((bad ? W_KV_SEQ : W_KV_ROWS) << 8));
    return;
  }
  const int len = kv_len(c, s), left = min(len, want);
  int32_t* row = c.table + (int64_t)s * c.max_pages;
  for (int p = held_pages(c, left) + threadIdx.x; p < held_pages(c, len); p += blockDim.x) {
    const int id = row[p];
    row[p] = -1;
    if (id >= 0 && id < c.n_pages) atomicSub(c.refs + id, 1);
    else report(c.status, KC_ERR_ARG | (W_KV_PAGE << 8));
  }
  __syncthreads();
  if (threadIdx.x == 0) c.len[s] = left;
}

void launch_kv_free(const KvView& c, const int32_t* seqs, const int32_t* keep, int n, cudaStream_t st) {
  launch_k(kv_free_kernel, n, 128, 0, st, c, seqs, keep, n);
}

// ---- extend ------------------------------------------------------------------
// One block. First every entry is looked over and the pages it needs are
// counted (marks find a sequence given twice); only if all of them are in
// order and there are pages enough does anything change. A sequence whose last
// page is partly full and held by others gets a page of its own for it (the
// copy runs in the next kernel); holders are served in the order of the call,
// and the one that is left alone with the page keeps it.
__global__ void __launch_bounds__(KV_BLOCK) kv_extend_kernel(KvView c, const int32_t* __restrict__ seqs,
                                                             const int32_t* __restrict__ n_new, int n) {
  pdl_enter();
  __shared__ int bad;
  const int tid = threadIdx.x;
  if (tid == 0) {
    bad = 0;
    *c.n_copy = 0;
  }
  __syncthreads();
  for (int i = tid; i < n; i += KV_BLOCK) {
    const int s = seqs ? seqs[i] : i, add = n_new[i];
    int last = -1, why = 0;
    if (s < 0 || s >= c.n_seq) {
      why = KC_ERR_ARG | (W_KV_SEQ << 8);
    } else {
      if (atomicCAS(c.mark + s, -1, i) != -1) why = KC_ERR_ARG | (W_KV_SEQ << 8);
      const int len = kv_len(c, s);
      if (add < 0) why = KC_ERR_ARG | (W_KV_ROWS << 8);
      else if ((int64_t)len + add > (int64_t)c.max_pages * c.page) why = KC_ERR_SHAPE | (W_KV_CAP << 8);
      else if (add > 0 && (len & (c.page - 1))) {
        last = c.table[(int64_t)s * c.max_pages + (len >> c.page_log2)];
        if (last < 0 || last >= c.n_pages) why = KC_ERR_ARG | (W_KV_PAGE << 8);
      }
    }
    if (why) {
      report(c.status, why);
      bad = 1;
    }
    c.last[i] = last;
  }
  __syncthreads();
  if (!bad) {
    // Pages needed (low half) and copies (high half), summed over the entries.
    long long run = 0;
    for (int base = 0; base < n; base += KV_BLOCK) {
      const int i = base + tid;
      long long v = 0;
      int last = -1;
      bool copy = false;
      if (i < n) {
        const int s = seqs ? seqs[i] : i;
        const int len = kv_len(c, s);
        last = c.last[i];
        if (last >= 0) {
          int holders = c.refs[last];
          if (holders > 1) {
            for (int j = 0; j < i && holders > 1; ++j) holders -= c.last[j] == last ? 1 : 0;
            copy = holders > 1;
          }
        }
        v = held_pages(c, len + n_new[i]) - held_pages(c, len) + (copy ? 1 + (1ll << 32) : 0);
      }
      long long total;
      const long long at = run + block_scan(v, total);
      if (i < n) {
        c.first[i] = (int)at;
        const int j = (int)(at >> 32);
        if (copy) {
          c.src[j] = last;
          c.dst[j] = (int)at;  // its place in `fresh` for now
          c.rows[j] = kv_len(c, seqs ? seqs[i] : i) & (c.page - 1);
        }
      }
      run += total;
    }
    const int need = (int)run, copies = (int)(run >> 32);
    // The `need` lowest free pages (n_seq * max_pages < 2^31, so `need` cannot
    // run into the copies' half).
    int found = 0;
    for (int base = 0; base < c.n_pages && found < need; base += KV_BLOCK * 8) {
      int ids[8], m = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = base + tid * 8 + u;
        if (p < c.n_pages && c.refs[p] == 0) ids[m++] = p;
      }
      long long total;
      const int at = found + (int)block_scan(m, total);
      for (int u = 0; u < m; ++u)
        if (at + u < need) c.fresh[at + u] = ids[u];
      found += (int)total;
    }
    __syncthreads();
    if (found < need) {
      if (tid == 0) report(c.status, KC_ERR_OOM | (W_KV_ROOM << 8));
    } else {
      for (int i = tid; i < copies; i += KV_BLOCK) {
        c.dst[i] = c.fresh[c.dst[i]];
        atomicSub(c.refs + c.src[i], 1);
      }
      if (tid == 0) *c.n_copy = copies;
      const int lane = tid & 31;
      for (int i = tid >> 5; i < n; i += KV_BLOCK / 32) {
        const int s = seqs ? seqs[i] : i, len = kv_len(c, s), add = n_new[i];
        const int first = c.first[i], count = (i + 1 < n ? c.first[i + 1] : need) - first;
        const int col = held_pages(c, len + add) - count;
        for (int t = lane; t < count; t += 32) {
          const int id = c.fresh[first + t];
          c.table[(int64_t)s * c.max_pages + col + t] = id;
          c.refs[id] = 1;
        }
        __syncwarp();
        if (lane == 0) c.len[s] = len + add;
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += KV_BLOCK) {
    const int s = seqs ? seqs[i] : i;
    if (s >= 0 && s < c.n_seq) c.mark[s] = -1;
  }
}

// ---- page copies -------------------------------------------------------------
// Rows 0 .. rows[i]-1 (null rows: all) of page src[i] to page dst[i], every
// layer and head, k and v. No dst is a src. A unit is one page of one layer of
// k or v; a block takes units in turn.
// Bound by the memory rate (each byte read and written once). Four 16-byte
// pieces of a thread under way and sixteen blocks per SM: a compaction that moves
// 1.72 GB of pages takes 297 us as a whole, 5.8 TB/s, 90% of a plain copy (one
// piece and eight blocks 311, four and eight 298, eight pieces and four blocks
// 317).
constexpr int COPY_THREADS = 256;
constexpr int COPY_AHEAD = 4;  // 16-byte pieces of a thread under way
__global__ void __launch_bounds__(COPY_THREADS) kv_copy_kernel(KvView c, bool whole, int32_t* table_remap,
                                                               const int* __restrict__ n_live) {
  pdl_enter();
  const int n = *c.n_copy;
  if (table_remap && n > 0) {
    // Compaction: table entries of moved pages follow them.
    const int64_t cells = (int64_t)c.n_seq * c.max_pages;
    const int live = *n_live;
    for (int64_t i = (int64_t)blockIdx.x * COPY_THREADS + threadIdx.x; i < cells;
         i += (int64_t)gridDim.x * COPY_THREADS) {
      const int p = table_remap[i];
      if (p >= live && p < c.n_pages) table_remap[i] = c.fresh[p];
    }
  }
  const int row_vec = c.hd / 8;               // 16-byte pieces of a row
  const int head_vec = c.page * row_vec;      // of a head's part of a page
  const int64_t page_vec = (int64_t)c.nkv * head_vec;
  const int64_t units = (int64_t)n * c.n_layer * 2;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int i = (int)(u / (2 * c.n_layer)), w = (int)(u % (2 * c.n_layer));
    uint4* pool = reinterpret_cast<uint4*>(w & 1 ? c.v : c.k) + (int64_t)(w >> 1) * c.n_pages * page_vec;
    const uint4* from = pool + c.src[i] * page_vec;
    uint4* to = pool + c.dst[i] * page_vec;
    // A head's rows lie together; whole pages altogether.
    const int per = whole ? (int)page_vec : c.rows[i] * row_vec, n_vec = whole ? (int)page_vec : per * c.nkv;
    for (int j0 = threadIdx.x; j0 < n_vec; j0 += COPY_AHEAD * COPY_THREADS) {
      uint4 v[COPY_AHEAD];
      int64_t at[COPY_AHEAD];
#pragma unroll
      for (int k = 0; k < COPY_AHEAD; ++k) {
        const int j = j0 + k * COPY_THREADS, h = j / per;
        at[k] = (int64_t)h * head_vec + (j - h * per);
        if (j < n_vec) v[k] = __ldcs(from + at[k]);
      }
#pragma unroll
      for (int k = 0; k < COPY_AHEAD; ++k)
        if (j0 + k * COPY_THREADS < n_vec) __stcs(to + at[k], v[k]);
    }
  }
}

static void launch_copies(const KvView& c, int most, bool whole, int32_t* remap, const int* n_live, cudaStream_t st) {
  const int64_t units = (int64_t)most * c.n_layer * 2;
  const int grid = (int)std::min<int64_t>(std::max<int64_t>(units, 1), 16 * (int64_t)num_sms());
  launch_k(kv_copy_kernel, grid, COPY_THREADS, 0, st, c, whole, remap, n_live);
}

void launch_kv_extend(const KvView& c, const int32_t* seqs, const int32_t* n_new, int n, cudaStream_t st) {
  launch_k(kv_extend_kernel, 1, KV_BLOCK, 0, st, c, seqs, n_new, n);
  launch_copies(c, n, false, nullptr, nullptr, st);
}

// ---- compact -----------------------------------------------------------------
// n_live = pages with holders. The i-th live page at or above n_live moves to
// the i-th free page below it (there are as many of one as of the other).
// fresh[src] = dst is the map that the tables follow.
__global__ void __launch_bounds__(KV_BLOCK) kv_compact_kernel(KvView c, int* live_out, int32_t* n_live) {
  pdl_enter();
  const int tid = threadIdx.x;
  long long live = 0;
  {
    long long mine = 0;
    for (int p = tid; p < c.n_pages; p += KV_BLOCK) mine += c.refs[p] > 0;
    block_scan(mine, live);
  }
  const int n = (int)live;
  long long run = 0;  // free pages below n (low half), live pages from n on (high half)
  for (int base = 0; base < c.n_pages; base += KV_BLOCK * 8) {
    long long v = 0;
    uint32_t pick = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int p = base + tid * 8 + u;
      if (p >= c.n_pages) break;
      if ((c.refs[p] > 0) == (p >= n)) {
        pick |= 1u << u;
        v += p < n ? 1 : 1ll << 32;
      }
    }
    long long total;
    const long long at = run + block_scan(v, total);
    int hole = (int)at, move = (int)(at >> 32);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (!(pick >> u & 1)) continue;
      const int p = base + tid * 8 + u;
      if (p < n) c.dst[hole++] = p;
      else c.src[move++] = p;
    }
    run += total;
  }
  __syncthreads();
  const int moves = (int)(run >> 32);
  for (int i = tid; i < moves; i += KV_BLOCK) {
    const int s = c.src[i], d = c.dst[i];
    c.fresh[s] = d;
    c.refs[d] = c.refs[s];
    c.refs[s] = 0;
  }
  if (tid == 0) {
    *c.n_copy = moves;
    *live_out = n;
    if (n_live) *n_live = n;
  }
}

void launch_kv_compact(const KvView& c, int32_t* n_live, cudaStream_t st) {
  int* live = c.first;  // one int of the workspace
  launch_k(kv_compact_kernel, 1, KV_BLOCK, 0, st, c, live, n_live);
  launch_copies(c, c.n_pages / 2, true, c.table, live, st);
}

// ---- copy --------------------------------------------------------------------
// Looks the whole list over; a page out of range, a destination given twice or
// one that is also a source leaves everything as it was.
__global__ void __launch_bounds__(KV_BLOCK) kv_copy_list_kernel(KvView c, const int32_t* __restrict__ src,
                                                                const int32_t* __restrict__ dst, int n) {
  pdl_enter();
  __shared__ int bad;
  const int tid = threadIdx.x;
  if (tid == 0) bad = 0;
  __syncthreads();
  for (int i = tid; i < n; i += KV_BLOCK) {
    const int s = src[i], d = dst[i];
    if (s < 0 || s >= c.n_pages || d < 0 || d >= c.n_pages || atomicCAS(c.mark + d, -1, i) != -1) bad = 1;
    c.src[i] = s;
    c.dst[i] = d;
  }
  __syncthreads();
  for (int i = tid; i < n; i += KV_BLOCK) {
    const int s = src[i];
    if (s >= 0 && s < c.n_pages && c.mark[s] != -1) bad = 1;
  }
  __syncthreads();
  for (int i = tid; i < n; i += KV_BLOCK) {
    const int d = dst[i];
    if (d >= 0 && d < c.n_pages) c.mark[d] = -1;
  }
  if (tid == 0) {
    if (bad) report(c.status, KC_ERR_ARG | (W_KV_COPY << 8));
    *c.n_copy = bad ? 0 : n;
  }
}

void launch_kv_copy_pages(const KvView& c, const int32_t* src, const int32_t* dst, int n, cudaStream_t st) {
  launch_k(kv_copy_list_kernel, 1, KV_BLOCK, 0, st, c, src, dst, n);
  launch_copies(c, n, true, nullptr, nullptr, st);
}

// ---- write -------------------------------------------------------------------
// Eight consecutive values of a row as cache values, in one 16-byte piece.
template <typename S, typename D>
__device__ __forceinline__ uint4 convert8(const S* p, bool aligned) {
  alignas(16) S in[8];
  if (aligned) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(S) / 2; ++i)
      reinterpret_cast<uint4*>(in)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) in[i] = p[i];
  }
  alignas(16) D o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (D)(float)in[i];
  return *reinterpret_cast<uint4*>(o);
}

constexpr int WRITE_THREADS = 128;
template <typename S, typename D>
__global__ void __launch_bounds__(WRITE_THREADS) kv_write_kernel(KvView c, int layer, const int32_t* __restrict__ seqs,
                                                                 const int32_t* __restrict__ row_start, int n,
                                                                 int n_rows, const S* __restrict__ k,
                                                                 const S* __restrict__ v, int64_t k_stride,
                                                                 int64_t v_stride, bool aligned, int blocks) {
  pdl_enter();
  if (blockIdx.x >= blocks) {
    // One block more where a list could name a sequence twice: it tells, beside
    // the others' writing (32 x 256 rows of 4 heads of 128 take 12.4 us as they did
    // without it, 1000 x 1 3.3 against 2.6, 4096 x 1 11.9 against 5.6; leaving the
    // second entry out would hold every write up: 14.5, 3.4 and 9.8). The marks
    // are -1 between calls.
    auto each = [&](auto&& fn) {  // eight entries of a thread under way
      for (int i0 = threadIdx.x; i0 < n; i0 += 8 * WRITE_THREADS) {
        int s[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) s[u] = i0 + u * WRITE_THREADS < n ? __ldg(seqs + i0 + u * WRITE_THREADS) : -1;
        fn(i0, s);
      }
      __syncthreads();
    };
    const auto real = [&](int s) { return s >= 0 && s < c.n_seq; };
    each([&](int i0, const int(&s)[8]) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (real(s[u])) atomicMax(c.mark + s[u], i0 + u * WRITE_THREADS);
    });
    each([&](int i0, const int(&s)[8]) {
      int last[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) last[u] = real(s[u]) ? __ldcg(c.mark + s[u]) : 0;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (real(s[u]) && last[u] != i0 + u * WRITE_THREADS) report(c.status, KC_ERR_ARG | (W_KV_SEQ << 8));
    });
    each([&](int, const int(&s)[8]) {
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (real(s[u])) c.mark[s[u]] = -1;
    });
    return;
  }
  const int row_vec = c.hd / 8, per = c.nkv * row_vec;  // 16-byte pieces of a head's row, of a row of k or v
  const int64_t pieces = (int64_t)n_rows * 2 * per;
  for (int64_t x = (int64_t)blockIdx.x * WRITE_THREADS + threadIdx.x; x < pieces;
       x += (int64_t)blocks * WRITE_THREADS) {
    const int r = (int)(x / (2 * per)), y = (int)(x - (int64_t)r * 2 * per);
    const bool is_v = y >= per;
    const int e = is_v ? y - per : y, h = e / row_vec, j = e - h * row_vec;
    int i = r, back = 1;  // the row is `back` positions from its sequence's end
    if (row_start) {
      i = kv_row_owner(row_start, n, r);
      if (i < 0) {
        if (y == 0) report(c.status, KC_ERR_ARG | (W_KV_ROWS << 8));
        continue;
      }
      back = row_start[i + 1] - r;
    }
    const int s = seqs ? seqs[i] : i;
    if (s < 0 || s >= c.n_seq) {
      if (y == 0) report(c.status, KC_ERR_ARG | (W_KV_SEQ << 8));
      continue;
    }
    const int pos = kv_len(c, s) - back;
    if (pos < 0) {
      if (y == 0) report(c.status, KC_ERR_ARG | (W_KV_ROWS << 8));
      continue;
    }
    const int id = c.table[(int64_t)s * c.max_pages + (pos >> c.page_log2)];
    if (id < 0 || id >= c.n_pages) {
      if (y == 0) report(c.status, KC_ERR_ARG | (W_KV_PAGE << 8));
      continue;
    }
    const S* from = (is_v ? v + r * v_stride : k + r * k_stride) + h * c.hd + j * 8;
    D* to = reinterpret_cast<D*>(is_v ? c.v : c.k) +
            ((((int64_t)layer * c.n_pages + id) * c.nkv + h) * c.page + (pos & (c.page - 1))) * c.hd + j * 8;
    *reinterpret_cast<uint4*>(to) = convert8<S, D>(from, aligned);
  }
}

template <typename S, typename D>
static void write_rows(const KvView& c, int layer, const int32_t* seqs, const int32_t* row_start, int n, int n_rows,
                       const void* k, const void* v, int64_t ks, int64_t vs, cudaStream_t st) {
  const int64_t pieces = (int64_t)n_rows * 2 * c.nkv * (c.hd / 8);
  const int grid = (int)std::min<int64_t>((pieces + WRITE_THREADS - 1) / WRITE_THREADS, 16 * (int64_t)num_sms());
  const int64_t el = 16 / sizeof(S);
  const bool aligned = !((uintptr_t)k & 15) && !((uintptr_t)v & 15) && ks % el == 0 && vs % el == 0;
  launch_k(kv_write_kernel<S, D>, grid + (seqs && n > 1), WRITE_THREADS, 0, st, c, layer, seqs, row_start, n, n_rows,
           static_cast<const S*>(k), static_cast<const S*>(v), ks, vs, aligned, grid);
}

void launch_kv_write(const KvView& c, int layer, const int32_t* seqs, const int32_t* row_start, int n, int n_rows,
                     int t, const void* k, const void* v, int64_t ks, int64_t vs, cudaStream_t st) {
  if (c.type == T_F16) {
    if (t == T_F32) write_rows<float, __half>(c, layer, seqs, row_start, n, n_rows, k, v, ks, vs, st);
    else write_rows<__half, __half>(c, layer, seqs, row_start, n, n_rows, k, v, ks, vs, st);
  } else {
    if (t == T_F32) write_rows<float, __nv_bfloat16>(c, layer, seqs, row_start, n, n_rows, k, v, ks, vs, st);
    else write_rows<__nv_bfloat16, __nv_bfloat16>(c, layer, seqs, row_start, n, n_rows, k, v, ks, vs, st);
  }
}

// ---- tensor maps -------------------------------------------------------------
static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encode() {
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    cudaDriverEntryPointQueryResult q;
    void* fn = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }();
  return encode;
}

static int encode_map(KvMap& map, int t, int rank, const void* base, const cuuint64_t* dims,
                        const cuuint64_t* strides, const cuuint32_t* box) {
  const auto encode = tensor_map_encode();
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUtensorMapDataType el = t == T_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : t == T_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                              : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (!encode || encode(reinterpret_cast<CUtensorMap*>(map.b), el, rank, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return KC_ERR_CUDA;
  return KC_OK;
}

int make_kv_maps(const KvView& c, int box_rows, KvMaps& maps) {
  const cuuint64_t row = (cuuint64_t)c.hd * 2;
  const cuuint64_t dims[4] = {(cuuint64_t)c.hd, (cuuint64_t)c.page, (cuuint64_t)c.nkv,
                              (cuuint64_t)c.n_layer * c.n_pages};
  const cuuint64_t strides[3] = {row, row * c.page, row * c.page * c.nkv};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
  const int rc = encode_map(maps.k, c.type, 4, c.k, dims, strides, box);
  return rc == KC_OK ? encode_map(maps.v, c.type, 4, c.v, dims, strides, box) : rc;
}

int make_q_map(const AttnArgs& a, KvMap& map) {
  const int group = a.nh / a.c.nkv;
  const cuuint64_t dims[3] = {(cuuint64_t)a.c.hd, (cuuint64_t)a.nh, (cuuint64_t)a.n_rows};
  const int el = a.t_q == T_F32 ? 4 : 2;
  const cuuint64_t strides[2] = {(cuuint64_t)a.c.hd * el, (cuuint64_t)a.q_stride * el};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / el), (cuuint32_t)group, (cuuint32_t)(128 / group)};
  return encode_map(map, a.t_q, 3, a.q, dims, strides, box);
}

// ---- workspace ---------------------------------------------------------------
int64_t kv_workspace_ints(const KvView& c) {
  const int64_t m = std::max(c.n_seq, c.n_pages);
  return 4 * m + 2 * (int64_t)c.n_seq + c.n_pages + 4;
}

cudaError_t kv_workspace_init(KvView& c, int* work, cudaStream_t st) {
  const int64_t m = std::max(c.n_seq, c.n_pages);
  c.mark = work;
  c.src = c.mark + m;
  c.dst = c.src + m;
  c.rows = c.dst + m;
  c.last = c.rows + m;
  c.first = c.last + c.n_seq;
  c.fresh = c.first + c.n_seq;
  c.n_copy = c.fresh + c.n_pages;
  cudaError_t e = cudaMemsetAsync(c.mark, 0xff, m * sizeof(int), st);
  if (e == cudaSuccess) e = cudaMemsetAsync(c.n_copy, 0, 4 * sizeof(int), st);
  return e;
}

}  // namespace kc
