// Rotary positions: pairs of channels (a, b) of the first 2 * half channels of every head become amplitude * (a cos - b sin, b cos + a sin), the angle of pair i at
// position p being 2 pi p turns[i]; `inverse` turns back, which is also the gradient's way. Pairs are (i, i + half), or neighbours (2 i, 2 i + 1).
// An angle of a far position is many turns: the product is made in 64 bits and only what is left of the last turn is rounded to fp32. Each is computed once for a
// token and serves its heads, of queries and keys alike.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../kernels/common.cuh"
#include "cp.h"

namespace b200 {

namespace {

constexpr int kMaxHalf = 512;

template <typename T> __device__ __forceinline__ float toFloat(T v);
template <> __device__ __forceinline__ float toFloat(float v) { return v; }
template <> __device__ __forceinline__ float toFloat(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float toFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T fromFloat(float v);
template <> __device__ __forceinline__ float fromFloat(float v) { return v; }
template <> __device__ __forceinline__ __half fromFloat(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat(float v) { return __float2bfloat16_rn(v); }

template <typename T, int E> struct alignas(E * sizeof(T)) Channels { T v[E]; };

// E channels at a time: 16 bytes, or one where sizes, strides or addresses do not allow more.
template <typename T, int E>
__device__ __forceinline__ void turnHeads(const RotaryArgs& a, int b, int tok, const float2* table) {
  const int paired = a.interleaved && E > 1 ? 2 * a.half / E : a.half / E;   // items of a head that turn: a pack of neighbours, or one of a and one of b
  const int items = paired + (a.dim - 2 * a.half) / E, heads = a.heads[0] + a.heads[1];
  const int stride = gridDim.y * blockDim.x;
  for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < heads * items; i += stride) {
    int head = i / items;
    const int p = i - head * items, which = head >= a.heads[0];
    if (which) head -= a.heads[0];
    const T* x = (const T*)a.x[which] + (b * a.inStride[which][0] + tok * a.inStride[which][1] + head * a.inStride[which][2]);
    T* y = (T*)a.y[which] + (b * a.outStride[which][0] + tok * a.outStride[which][1] + head * a.outStride[which][2]);
    using C = Channels<T, E>;
    if (p >= paired) {
      const int at = 2 * a.half + (p - paired) * E;
      *(C*)(y + at) = *(const C*)(x + at);
    } else if (E > 1 && a.interleaved) {
      C v = *(const C*)(x + p * E);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 t = table[(p * E + e) / 2];
        const float lo = toFloat(v.v[e]), hi = toFloat(v.v[(e + 1) % E]);
        v.v[e] = fromFloat<T>(lo * t.x - hi * t.y);
        v.v[(e + 1) % E] = fromFloat<T>(hi * t.x + lo * t.y);
      }
      *(C*)(y + p * E) = v;
    } else {
      const int first = a.interleaved ? 2 * p : p * E, second = a.interleaved ? first + 1 : a.half + p * E;   // (neighbours: one channel at a time)
      C u = *(const C*)(x + first), v = *(const C*)(x + second);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float2 t = table[p * E + e];
        const float lo = toFloat(u.v[e]), hi = toFloat(v.v[e]);
        u.v[e] = fromFloat<T>(lo * t.x - hi * t.y);
        v.v[e] = fromFloat<T>(hi * t.x + lo * t.y);
      }
      *(C*)(y + first) = u;
      *(C*)(y + second) = v;
    }
  }
}

// A CTA (of gridDim.y, where tokens are few) has a token.
template <typename T>
__global__ void __launch_bounds__(256) rotaryKernel(const __grid_constant__ RotaryArgs a) {
  __shared__ float2 table[kMaxHalf];
  pdlEnter();
  for (int token = blockIdx.x; token < a.batch * a.tokens; token += gridDim.x) {
    const int b = token / a.tokens, tok = token - b * a.tokens;
    long long at = a.offset + tok;
    if (a.positions) {
      const long long i = b * a.positionStride[0] + tok * a.positionStride[1];
      at = a.positions64 ? ((const long long*)a.positions)[i] : (long long)((const int*)a.positions)[i];
    }
    for (int i = threadIdx.x; i < a.half; i += blockDim.x) {
      double t = (double)at * a.turns[i];
      t -= rint(t);
      float s, c;
      sincospif((float)(2.0 * t), &s, &c);
      table[i] = make_float2(a.amplitude * c, a.inverse ? -a.amplitude * s : a.amplitude * s);
    }
    __syncthreads();
    if (a.wide) turnHeads<T, 16 / sizeof(T)>(a, b, tok, table);
    else turnHeads<T, 1>(a, b, tok, table);
    __syncthreads();
  }
}

}  // namespace

const void* rotaryKernelFn(int type) {
  return type == ATTN_F16 ? (const void*)rotaryKernel<__half> : type == ATTN_BF16 ? (const void*)rotaryKernel<__nv_bfloat16> : (const void*)rotaryKernel<float>;
}

}  // namespace b200
