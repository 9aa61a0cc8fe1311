// Sampling of tokens from logits (sample.cu): the host-side launcher.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace kc {

constexpr int SAMPLE_MAX_VOCAB = 393216;  // eight blocks' shared memory

struct SampleArgs {
  const void* logits;  // [n] rows of n_vocab, `stride` elements apart
  int64_t stride;
  int n, n_vocab;
  const float* u;            // [n]
  const float* temperature;  // [n] or null: 1
  const int32_t* top_k;      // [n] or null: 0
  const float* top_p;        // [n] or null: 1
  const float* min_p;        // [n] or null: 0
  int32_t* tokens;           // [n]
  float* probs;              // [n] or null
  const int* at;             // null: 0; else u and probs are those from *at on
};
int launch_sample(const SampleArgs& a, int t, cudaStream_t st);

}  // namespace kc
