// Device helpers of the paged cache shared by its kernels (kv.cu, attn_*.cu).
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "kv.h"

namespace kc {

// Positions sequence s holds, within what its table can hold.
__device__ __forceinline__ int kv_len(const KvView& c, int s) {
  const int64_t cap = (int64_t)c.max_pages * c.page;
  const int len = c.len[s];
  return len < 0 ? 0 : (int)(len < cap ? len : cap);
}

// The entry i whose rows row_start[i] .. row_start[i+1]-1 hold row r, or -1.
__device__ __forceinline__ int kv_row_owner(const int32_t* __restrict__ row_start, int n, int r) {
  int lo = 0, hi = n;  // row_start[lo] <= r < row_start[hi], if the rows ascend
  if (r < row_start[0] || r >= row_start[n]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (row_start[mid] <= r) lo = mid;
    else hi = mid;
  }
  return row_start[lo] <= r && r < row_start[hi] ? lo : -1;
}

// For a block of T threads of a call that writes to the sequences it lists: one
// block more where a list could name a sequence twice tells, beside the others'
// writing (32 x 256 rows of 4 heads of 128 take 12.4 us as they did without it,
// 1000 x 1 3.3 against 2.6, 4096 x 1 11.9 against 5.6; leaving the second entry out
// would hold every write up: 14.5, 3.4 and 9.8). The marks are -1 between calls.
template <int T>
__device__ __forceinline__ void kv_report_repeats(const KvView& c, const int32_t* seqs, int n) {
  auto each = [&](auto&& fn) {  // eight entries of a thread under way
    for (int i0 = threadIdx.x; i0 < n; i0 += 8 * T) {
      int s[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) s[u] = i0 + u * T < n ? __ldg(seqs + i0 + u * T) : -1;
      fn(i0, s);
    }
    __syncthreads();
  };
  const auto real = [&](int s) { return s >= 0 && s < c.n_seq; };
  each([&](int i0, const int(&s)[8]) {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (real(s[u])) atomicMax(c.mark + s[u], i0 + u * T);
  });
  each([&](int i0, const int(&s)[8]) {
    int last[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) last[u] = real(s[u]) ? __ldcg(c.mark + s[u]) : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (real(s[u]) && last[u] != i0 + u * T) report(c.status, KC_ERR_ARG | (W_KV_SEQ << 8));
  });
  each([&](int, const int(&s)[8]) {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (real(s[u])) c.mark[s[u]] = -1;
  });
}

}  // namespace kc
