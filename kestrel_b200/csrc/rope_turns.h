// The rotation of a rope id as the kernels take it, and how it is made of kc_rope's
// arguments: host code without CUDA.
#pragma once

#include <math.h>
#include <stdint.h>

#include <algorithm>

#ifdef __CUDACC__
#pragma nv_diag_suppress 20208  // (long double: on the host only)
#endif

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

// The formulas of kc_rope, in the host's widest type (64-bit mantissas): a turn is off
// by 10 roundings of 2^-64 of itself at most, and 2^-65, so the phase at position 2^31
// by 2^-31 of a turn where the frequency is 1 at most, and 2^-30 up to
// ROPE_MAX_FREQUENCY. False: one above that, whose far phases would be worse.
constexpr double ROPE_MAX_FREQUENCY = 4.0;
inline bool make_rope(RopeParams& r, int dim, bool interleaved, float base, int scaling, float factor, int original, float low,
               float high, float gain, const float* freq_factors) {
  const long double two_pi = 2 * acosl(-1.0L), s = factor, len = original;
  r = RopeParams{};
  r.dim = dim;
  r.interleaved = interleaved;
  r.gain = gain != 0.f ? gain : scaling == ROPE_YARN && s > 1 ? (float)(1 + 0.1L * logl(s)) : 1.f;
  long double from = 0, to = 0;
  if (scaling == ROPE_YARN) {
    const auto pair_of = [&](long double turns) { return dim * logl(len / (two_pi * turns)) / (2 * logl(base)); };
    from = std::max(0.0L, floorl(pair_of(high)));
    to = std::min((long double)dim - 1, ceill(pair_of(low)));
  }
  for (int i = 0; i < dim / 2; ++i) {
    // (The exponent's rounding, which a large base would multiply, put right.)
    const long double e = -2.0L * i / dim;
    long double w = powl(base, e);
    w += w * logl(base) * (fmal(-e, dim, -2.0L * i) / dim);
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
    if (!(w <= ROPE_MAX_FREQUENCY)) return false;
    long double turn = w / two_pi;
    turn -= floorl(turn);  // whole turns a position change nothing
    r.turn[i] = (uint64_t)(int64_t)llrintl(ldexpl(turn - (turn >= 0.5L ? 1 : 0), 64));
  }
  return true;
}

}  // namespace kc
