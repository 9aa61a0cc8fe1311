// Device helpers of the attention kernels: TMA loads from the pools, 16-bit
// conversions, warp-level matrix products.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "kv.h"

namespace kc {

// Box of a pool: `x` the first of 64 columns of a head's rows, `row` within the
// page, head, and layer * n_pages + page. Columns past head_dim and pages past
// the pool read as zeros.
__device__ __forceinline__ void kv_load(void* dst, const KvMap* map, int x, int row, int head, int page,
                                        uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const KvMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const KvMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two f32 values as a pair of T, and what the pair leaves of them.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __half>) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t rest2(float lo, float hi, uint32_t pair) {
  float a, b;
  if constexpr (std::is_same_v<T, __half>) {
    a = __half2float(__ushort_as_half((unsigned short)(pair & 0xFFFF)));
    b = __half2float(__ushort_as_half((unsigned short)(pair >> 16)));
  } else {
    a = __uint_as_float(pair << 16);
    b = __uint_as_float(pair & 0xFFFF0000u);
  }
  return pack2<T>(lo - a, hi - b);
}

// Two weights (not negative) as a pair of T. One that f16 would round to zero
// becomes its smallest value instead, 2^-24, so that an infinite value still
// makes the result infinite, not NaN (0 times it); the rest takes what is too
// much off again, and without a rest 2^-24 against weights of up to 2^15 is
// below what the type of the result holds.
template <typename T>
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  uint32_t r = pack2<T>(lo, hi);
  if constexpr (std::is_same_v<T, __half>) {
    const uint32_t least = min(__float_as_uint(lo), 1u) | min(__float_as_uint(hi), 1u) << 16;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(least));
  }
  return r;
}

// A sum carried by values and rests. Of an infinite or NaN one the values' sum is
// right by itself: it meets the rests as 0 times it, or with the other sign.
// (Values are zero only where what they carry is, or is below 2^-39 of its
// row's largest.)
__device__ __forceinline__ float with_rest(float value, float rest) {
  const float s = value + rest;
  return fabsf(value) < INFINITY ? s : value;
}

// The power of two that puts a row's largest magnitude in [2^14, 2^15), within
// f16's range (1 for a row of zeros or one that is not finite).
__device__ __forceinline__ float pow2_factor(float amax) {
  const int ex = (int)(__float_as_uint(amax) >> 23);
  return ex > 0 && ex < 255 ? __uint_as_float((uint32_t)min(254, 127 + 14 + 127 - ex) << 23) : 1.f;
}

// Two f32 lanes at once (sm_100's packed instructions).
__device__ __forceinline__ uint64_t f2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 f2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// Eight consecutive values, aligned to 16 bytes.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  alignas(16) T x[8];
  *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
}

// The first n of 16 values (n a multiple of 8) to p, whose row starts and
// lengths are multiples of the lowest set bit of `grain` bytes. 32 bytes a
// store where they are aligned: a whole sector.
__device__ __forceinline__ void store32(void* p, const uint32_t (&u)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]),
               "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const float* v, int n, uint32_t grain) {
  if constexpr (sizeof(T) == 4) {
    uint32_t u[2][8];
#pragma unroll
    for (int i = 0; i < 16; ++i) u[i / 8][i % 8] = __float_as_uint(v[i]);
    if (!(grain & 31)) {
      store32(p, u[0]);
      if (n > 8) store32(p + 8, u[1]);
      return;
    }
  } else {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    if (!(grain & 31) && n > 8) return store32(p, u);
    if (!(grain & 15)) {
      reinterpret_cast<uint4*>(p)[0] = make_uint4(u[0], u[1], u[2], u[3]);
      if (n > 8) reinterpret_cast<uint4*>(p)[1] = make_uint4(u[4], u[5], u[6], u[7]);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < n) p[i] = (T)v[i];
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// D = A B (nothing is added: for sums that are rounded to nearest outside).
template <typename T>
__device__ __forceinline__ void mma16816_only(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, "
        "%10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, "
        "%10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

}  // namespace kc
