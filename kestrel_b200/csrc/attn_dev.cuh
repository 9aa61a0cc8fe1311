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
__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// 2^x of two lanes on the FMA pipes, beside the special-function unit, for
// weights that are rounded to 16 bits: x = n + f with f in [-1/2, 1/2] (the
// rounding that adding 1.5 * 2^23 does), 2^f by the cubic whose largest
// relative error there is least (7.5e-5, a sixth of f16's half unit; computed
// by Lawson's reweighted least squares), n into the exponent. x <= 120; below
// -126 the result is 0 but for 2^-126; a NaN comes out as a value past the
// 16-bit types' range.
__device__ __forceinline__ float2 exp2_cubic(float2 v) {
  const uint64_t x = f2(max_nan(v.x, -126.f), max_nan(v.y, -126.f));
  const uint64_t t = add2(x, f2(12582912.f, 12582912.f));
  const uint64_t f = fma2(add2(t, f2(-12582912.f, -12582912.f)), f2(-1.f, -1.f), x);
  uint64_t p = fma2(f, f2(0.05517137654f, 0.05517137654f), f2(0.24261121067f, 0.24261121067f));
  p = fma2(p, f, f2(0.69326103069f, 0.69326103069f));
  p = fma2(p, f, f2(0.99992806957f, 0.99992806957f));
  const float2 a = f2(p), n = f2(t);
  return make_float2(__uint_as_float(__float_as_uint(a.x) + (__float_as_uint(n.x) << 23)),
                     __uint_as_float(__float_as_uint(a.y) + (__float_as_uint(n.y) << 23)));
}

__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
}

// Four consecutive values, aligned to four.
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 x = *reinterpret_cast<const float4*>(p);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  alignas(8) T x[4];
  *reinterpret_cast<uint2*>(x) = *reinterpret_cast<const uint2*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)x[i];
}
// 16 bytes of values of T.
__device__ __forceinline__ void store_piece(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const float* v) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
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

}  // namespace kc
