// Shared by the policy-training kernels (learn_*.cu): element types, warp and CTA
// reductions in a fixed order, launch status.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/swarp_b200.h"

namespace swarp {
namespace learn {

constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// max that hands a NaN on (fmaxf drops it), so that a NaN logit reaches the result
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x to 2 ulp; what is below 2^-126 becomes 0
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename V> __device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = max_nan(v, __shfl_xor_sync(kAll, v, d));
  return v;
}

inline int launch_status() {
  return cudaGetLastError() == cudaSuccess ? SWARP_OK : SWARP_ERR_CUDA;
}

inline size_t align256(size_t b) { return (b + 255) / 256 * 256; }

}  // namespace learn
}  // namespace swarp
