// Rotary positions (rope.cu): the host-side launchers.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "kv.h"
#include "rope_turns.h"

namespace kc {

// Rows of n_head heads of hd, strides in elements; out may be x.
void launch_rope(const RopeParams& r, const int32_t* positions, int n_rows, int n_head, int hd, int t, const void* x,
                 int64_t x_stride, void* out, int64_t out_stride, cudaStream_t st);

struct AppendArgs {
  KvView c;
  int layer;
  const int32_t* seqs;       // null: 0 .. n-1
  const int32_t* row_start;  // [n + 1]; null: one row each
  int n, n_rows, nh;         // nh 0: no queries
  const void *q, *k, *v;
  void* q_out;
  int64_t q_stride, k_stride, v_stride, out_stride;
};
void launch_kv_append(const AppendArgs& a, const RopeParams& r, int t, cudaStream_t st);

}  // namespace kc
