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

}  // namespace kc
