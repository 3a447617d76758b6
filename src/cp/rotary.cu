// Rotary positions: pairs of channels (a, b) of the first 2 * half channels of every head become amplitude * (a cos - b sin, b cos + a sin), the angle of pair i at
// position p being 2 pi p turns[i]; `inverse` turns back, which is also the gradient's way. Pairs are (i, i + half), or neighbours (2 i, 2 i + 1).
// An angle of a far position is many turns: the product is made in 64 bits and only what is left of the last turn is rounded to fp32. Each is computed once for a
// token and serves its heads, of queries and keys alike.
// Bound by memory: 16384 tokens of 40 heads of 128 channels in bf16 (336 MB there and back) 59 to 64 us from box to box, 5.3 to 5.6 TB/s where a copy reaches 6.5; a token alone takes its launch.
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

// E channels at a time: 16 bytes, or one where sizes, strides or addresses do not allow more. An item is a pack of each half of the pairs, a pack of neighbours, or one that is
// only copied; a thread steps from item to item without a division.
template <typename T, int E>
__device__ __forceinline__ void turnHeads(const RotaryArgs& a, int token0, int tokens, const float2* table) {
  using C = Channels<T, E>;
  const bool neighbours = a.interleaved && E > 1;
  const int paired = neighbours ? 2 * a.half / E : a.half / E, heads = a.heads[0] + a.heads[1];
  const int stride = gridDim.y * blockDim.x, first = blockIdx.y * blockDim.x + threadIdx.x;
  const int stepRows = stride / a.items, stepP = stride % a.items, stepTokens = stepRows / heads, stepHeads = stepRows % heads;
  int p = first % a.items, row = first / a.items, local = row / heads, head = row % heads;
  const unsigned each = a.tokens, token = (unsigned)token0 + local;   // (one behind the last may be 2^31 or more)
  unsigned tok = token % each;
  int b = token / each;
  while (local < tokens) {
    const int which = head >= a.heads[0];
    const long long h = which ? head - a.heads[0] : head;
    const T* x = (const T*)a.x[which] + (b * a.inStride[which][0] + tok * a.inStride[which][1] + h * a.inStride[which][2]);
    T* y = (T*)a.y[which] + (b * a.outStride[which][0] + tok * a.outStride[which][1] + h * a.outStride[which][2]);
    const float2* angles = table + local * a.half;
    if (p >= paired) {
      const int at = 2 * a.half + (p - paired) * E;
      *(C*)(y + at) = *(const C*)(x + at);
    } else if (neighbours) {
      C v = *(const C*)(x + p * E);
#pragma unroll
      for (int e = 0; e + 1 < E; e += 2) {
        const float2 r = angles[(p * E + e) / 2];
        const float lo = toFloat(v.v[e]), hi = toFloat(v.v[(e + 1) % E]);
        v.v[e] = fromFloat<T>(lo * r.x - hi * r.y);
        v.v[(e + 1) % E] = fromFloat<T>(hi * r.x + lo * r.y);
      }
      *(C*)(y + p * E) = v;
    } else {
      const int one = a.interleaved ? 2 * p : p * E, two = a.interleaved ? one + 1 : a.half + one;
      C u = *(const C*)(x + one), v = *(const C*)(x + two);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float2 r = angles[p * E + e];
        const float lo = toFloat(u.v[e]), hi = toFloat(v.v[e]);
        u.v[e] = fromFloat<T>(lo * r.x - hi * r.y);
        v.v[e] = fromFloat<T>(hi * r.x + lo * r.y);
      }
      *(C*)(y + one) = u;
      *(C*)(y + two) = v;
    }
    p += stepP;
    int more = stepTokens;
    head += stepHeads;
    if (p >= a.items) {
      p -= a.items;
      ++head;
    }
    if (head >= heads) {
      head -= heads;
      ++more;
    }
    local += more;
    for (tok += more; tok >= each; tok -= each) ++b;
  }
}

// A CTA has `tokensAtOnce` tokens; where tokens are few, gridDim.y CTAs share the heads of the same ones.
template <typename T>
__global__ void __launch_bounds__(256, 6) rotaryKernel(const __grid_constant__ RotaryArgs a) {
  __shared__ float2 table[kMaxHalf];
  const int token0 = blockIdx.x * a.tokensAtOnce, tokens = min(a.tokensAtOnce, a.batch * a.tokens - token0);
  pdlEnter();
  for (int i = threadIdx.x; i < tokens * a.half; i += blockDim.x) {
    const int local = i / a.half, pair = i - local * a.half, b = (token0 + local) / a.tokens, tok = token0 + local - b * a.tokens;
    long long at = a.offset + tok;
    if (a.positions) {
      const long long n = b * a.positionStride[0] + tok * a.positionStride[1];
      at = a.positions64 ? ((const long long*)a.positions)[n] : (long long)((const int*)a.positions)[n];
    }
    double t = (double)at * a.turns[pair];
    t -= rint(t);
    float s, c;
    sincospif((float)(2.0 * t), &s, &c);
    table[i] = make_float2(a.amplitude * c, a.inverse ? -a.amplitude * s : a.amplitude * s);
  }
  __syncthreads();
  if (a.wide) turnHeads<T, 16 / sizeof(T)>(a, token0, tokens, table);
  else turnHeads<T, 1>(a, token0, tokens, table);
}

}  // namespace

const void* rotaryKernelFn(int type) {
  return type == ATTN_F16 ? (const void*)rotaryKernel<__half> : type == ATTN_BF16 ? (const void*)rotaryKernel<__nv_bfloat16> : (const void*)rotaryKernel<float>;
}

}  // namespace b200
