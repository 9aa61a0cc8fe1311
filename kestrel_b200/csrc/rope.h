// Rotary positions (rope.cu): the rotation of a rope id as the kernels take it,
// and the host-side launchers.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "kv.h"

namespace kc {

constexpr int ROPE_MAX_DIM = 256;

// The pairs' frequencies as 64-bit fractions of a turn per position: the phase
// position * turn[i], modulo 2^64, is exact however far the position. Passed to
// the kernels by value (1 KB), so a rope id holds no device memory.
struct RopeParams {
  int dim;           // values of a head that turn, the first ones
  int interleaved;   // pairs (2i, 2i + 1); otherwise (i, i + dim / 2)
  float gain;        // cos and sin are multiplied by it
  uint64_t turn[ROPE_MAX_DIM / 2];
};

enum : int { ROPE_NONE = 0, ROPE_LINEAR = 1, ROPE_YARN = 2, ROPE_BANDS = 3 };

// The formulas of kc_rope, in the host's widest type. False: a frequency above
// ROPE_MAX_FREQUENCY, past which the far positions' phases would not be exact.
constexpr double ROPE_MAX_FREQUENCY = 4.0;
bool make_rope(RopeParams& r, int dim, bool interleaved, float base, int scaling, float factor, int original, float low,
               float high, float gain, const float* freq_factors);

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
