// Device helpers shared by the kernels on rows of logits (logits.cu, distill.cu).
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"

namespace sq {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// 2^x by the hardware instruction; exp2f gives the same bits for x in [-64, 0] (compared over
// 2^30 arguments), so the integer weights of a draw can be computed outside this library.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

// A logit as the draw and the record see it: NaN counts as masked (-inf), -0 as +0.
__device__ __forceinline__ float plain_logit(float v) { return v != v ? -INFINITY : v + 0.0f; }

// Order-preserving key of a plain logit.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;     // order_key(-inf)

}  // namespace sq
