// Arithmetic shared by the experts' products and the row kernels of their backward pass.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "moe_ops.h"

namespace b200 {

__device__ __forceinline__ void unpackBf16x8(uint4 q, float* f) {
  const __nv_bfloat162* p = (const __nv_bfloat162*)&q;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __bfloat1622float2(p[i]);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ uint4 packBf16x8(const float* f) {
  uint4 q;
  __nv_bfloat162* p = (__nv_bfloat162*)&q;
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return q;
}

// 1 / (1 + exp(-v)). The short exponential and division are off by a few units of 2^-22 where the result is rounded to bf16 (2^-9 at
// most): the epilogue computes one per element. For v below -87 the divisor is huge and the result 0, as it should be.
__device__ __forceinline__ float sigmoidOf(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// Activation of an ungated layer, or of the gate: relu, gelu (v times the normal distribution function, by erf) or silu (v * sigmoid).
__device__ __forceinline__ float activation(int act, float v) {
  if (act == ACT_SILU) return v * sigmoidOf(v);
  if (act == ACT_GELU) return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
  return act == ACT_RELU && v < 0.0f ? 0.0f : v;   // (a NaN stays one)
}

// Value and derivative. silu' = s (1 + v (1 - s)); gelu' = cdf + v * density; relu' is 0 at 0.
template <int ACT>
__device__ __forceinline__ void activationAndSlope(float v, float* value, float* slope) {
  if (ACT == ACT_SILU) {
    const float s = sigmoidOf(v);
    *value = v * s;
    *slope = s * (1.0f + v * (1.0f - s));
  } else if (ACT == ACT_GELU) {
    const float cdf = 0.5f * (1.0f + erff(v * 0.70710678118654752f));
    *value = v * cdf;
    *slope = cdf + v * 0.39894228040143268f * __expf(-0.5f * v * v);
  } else if (ACT == ACT_RELU) {
    *value = v < 0.0f ? 0.0f : v;
    *slope = v > 0.0f ? 1.0f : 0.0f;
  } else {
    *value = v;
    *slope = 1.0f;
  }
}

}  // namespace b200
