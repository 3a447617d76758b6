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

// 1 / (1 + exp(-v)). The short exponential and division are off by a few units of 2^-22 where the result is rounded to bf16 (2^-8 at
// most): the epilogue computes one per element. Where the divisor passes 2^126, for v below -87.3, the short division gives 0: silu, less than 1.1e-36 there, is flushed.
__device__ __forceinline__ float sigmoidOf(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }

// The normal distribution function at v, 0.5 erfc(-v / sqrt 2), from a Chebyshev fit of erfc with a relative error of 1.2e-7 everywhere (W. H. Press et al.,
// Numerical Recipes, erfcc): no branches, half the instructions of erff, and no cancellation on the left. The short exponential adds 2^-21 there and
// (2 + 0.6 v^2) 2^-23 of it further out.
__device__ __forceinline__ float normalCdf(float v) {
  const float z = fabsf(v) * 0.70710678118654752f, t = __fdividef(1.0f, fmaf(0.5f, z, 1.0f));
  float p = fmaf(t, 0.17087277f, -0.82215223f);
  p = fmaf(t, p, 1.48851587f);
  p = fmaf(t, p, -1.13520398f);
  p = fmaf(t, p, 0.27886807f);
  p = fmaf(t, p, -0.18628806f);
  p = fmaf(t, p, 0.09678418f);
  p = fmaf(t, p, 0.37409196f);
  p = fmaf(t, p, 1.00002368f);
  p = fmaf(t, p, -1.26551223f);
  const float half = 0.5f * t * __expf(fmaf(-z, z, p));
  return v < 0.0f ? half : 1.0f - half;
}

// Activation of an ungated layer, or of the gate: relu, gelu (v times the normal distribution function) or silu (v * sigmoid).
template <int ACT>
__device__ __forceinline__ float activation(float v) {
  if (ACT == ACT_SILU) return v * sigmoidOf(v);
  if (ACT == ACT_GELU) return v * normalCdf(v);
  return ACT == ACT_RELU && v < 0.0f ? 0.0f : v;   // (a NaN stays one)
}
// Of N values, times `up` of a gated layer (u): decided once, not for every value.
template <int N>
__device__ __forceinline__ void activateAll(int act, float (&v)[N], const float (&u)[N]) {
  switch (act) {
    case ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activation<ACT_RELU>(v[i]);
      break;
    case ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activation<ACT_GELU>(v[i]);
      break;
    case ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activation<ACT_SILU>(v[i]);
      break;
    case ACT_SWIGLU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activation<ACT_SILU>(v[i]) * u[i];
      break;
    case ACT_GEGLU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activation<ACT_GELU>(v[i]) * u[i];
      break;
    default: break;
  }
}

// Value and derivative. silu' = s (1 + v (1 - s)); gelu' = cdf + v * density; relu' is 0 at 0.
template <int ACT>
__device__ __forceinline__ void activationAndSlope(float v, float* value, float* slope) {
  if (ACT == ACT_SILU) {
    const float s = sigmoidOf(v);
    *value = v * s;
    *slope = s * (1.0f + v * (1.0f - s));
  } else if (ACT == ACT_GELU) {
    const float cdf = normalCdf(v);
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

// dbias[i] = bf16(sum of partial[k][i] over the slices, in order): thread `at` of `threads`, four neighbouring sums at a time (n is a multiple of 8).
__device__ __forceinline__ void biasFromSlices(const float* partial, __nv_bfloat16* dbias, size_t n, int slices, size_t at, size_t threads) {
  for (size_t i = at * 4; i < n; i += threads * 4) {
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int k = 0; k < slices; ++k) {
      const float4 v = *(const float4*)(partial + k * n + i);
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    __nv_bfloat162 out[2] = {__floats2bfloat162_rn(s.x, s.y), __floats2bfloat162_rn(s.z, s.w)};
    *(uint2*)(dbias + i) = *(uint2*)out;
  }
}

}  // namespace b200
