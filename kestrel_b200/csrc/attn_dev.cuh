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

// Two f32 lanes at once: v * m + a, v + w.
__device__ __forceinline__ float2 fma2(float2 v, float m, float a) {
  uint64_t r, x, y, z;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(v.x), "f"(v.y));
  asm("mov.b64 %0, {%1, %1};" : "=l"(y) : "f"(m));
  asm("mov.b64 %0, {%1, %1};" : "=l"(z) : "f"(a));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}
__device__ __forceinline__ float2 add2(float2 v, float2 w) {
  uint64_t r, x, y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(v.x), "f"(v.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(w.x), "f"(w.y));
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
  return v;
}

// Four consecutive values, aligned to four; eight, aligned to 16 bytes.
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
__device__ __forceinline__ void store8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
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
