// Helpers shared by the model operators that take several element types: eight-element vector access,
// pairs of 16-bit values, and the per-device opt-in of a kernel's shared memory.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "noise_b200.h"

namespace noise {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename E>
__device__ __forceinline__ E from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Two values as one 32-bit word, the first in the lower half.
template <typename E>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename E>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Eight consecutive elements of a 16-bit type, 16-byte aligned.
template <typename E>
struct Vec8 {
  uint4 w;
  __device__ __forceinline__ void load(const E* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<E>(u[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
};

// n / d for n < 2^31 by a multiplication: with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1, the quotient is
// (mulhi(m, n) + n) >> s (Granlund and Montgomery, division by invariant integers).
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(uint32_t divisor) : d(divisor), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

// Four consecutive elements, aligned to their size: one 8-byte access of a 16-bit type, one 16-byte access of fp32.
template <typename E>
struct Vec4 {
  uint2 w;
  __device__ __forceinline__ void load(const E* p) { w = __ldcs(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void store(E* p) const { __stcs(reinterpret_cast<uint2*>(p), w); }
  __device__ __forceinline__ void get(float2 (&v)[2]) const { v[0] = unpack2<E>(w.x), v[1] = unpack2<E>(w.y); }
  __device__ __forceinline__ void set(const float2 (&v)[2]) { w = make_uint2(pack2<E>(v[0].x, v[0].y), pack2<E>(v[1].x, v[1].y)); }
};
template <>
struct Vec4<float> {
  float4 a;
  __device__ __forceinline__ void load(const float* p) { a = __ldcs(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void store(float* p) const { __stcs(reinterpret_cast<float4*>(p), a); }
  __device__ __forceinline__ void get(float2 (&v)[2]) const { v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w); }
  __device__ __forceinline__ void set(const float2 (&v)[2]) { a = make_float4(v[0].x, v[0].y, v[1].x, v[1].y); }
};

// 16 bytes of global memory into shared memory without a register; `have` false fills zeros and reads nothing.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool have = true) {
  const int n = have ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A kernel's opt-in to `bytes` of dynamic shared memory (and to clusters of more than 8 CTAs), made once
// per device: the attribute belongs to the device that is current when it is set.
struct KernelOptIn {
  std::atomic<uint64_t> done{0};
  template <typename K>
  bool operator()(K kernel, int bytes, bool wide_cluster = false) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    if (wide_cluster &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return false;
    done.fetch_or(bit, std::memory_order_release);
    return true;
  }
};

inline bool is_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace noise
