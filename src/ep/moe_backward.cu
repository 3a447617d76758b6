// Row kernels of a mixture-of-experts layer's backward pass: the derivative of the experts' activation with the sums of the bias gradient,
// and the gradients of combine and dispatch over the rows of one GPU. All are bound by memory: each operand is read once, each
// result written once, bf16 (weights and their gradients fp32) in memory and fp32 in between.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../kernels/common.cuh"
#include "moe_math.cuh"
#include "moe_ops.h"

namespace b200 {

namespace {

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* f) { unpackBf16x8(*(const uint4*)p, f); }
__device__ __forceinline__ void load8(const float* p, float* f) {
  *(float4*)f = *(const float4*)p;
  *(float4*)(f + 4) = *(const float4*)(p + 4);
}
__device__ __forceinline__ int rowsInUse(const int* counts, int e, int cap) { return counts ? min(max(counts[e], 0), cap) : cap; }

}  // namespace

// dz = dout * act'(z) for the rows in use of every expert; gated: d(gate) = dout * up * act'(gate) and d(up) = dout * act(gate). CTA (c, e, s) takes
// columns [c * kActCols, ...) of expert e, a thread 8 neighbouring ones, and of each gridDim.z * 8 rows the 8 of slice s. The sums over a slice's rows stay
// in registers and are joined in a fixed order: the bias gradient has the same bits every time. Memory bounds it: 8 x 512 rows, 28672 columns, swiglu, 97 us
// (6.0 TB/s), with z in fp32 121 us, where four CTAs fit an SM (with the three that the compiler chose, 154).
// dz is rounded to bf16: the products that follow take it as a bf16 operand. z comes as the forward call kept it (Z), in fp32, or rounded to bf16 where the caller prefers half
// the memory in the largest tensor that a layer keeps. With the rounding of their results the gradients are off by 0.00235 of their norm with z in fp32, by 0.0024 (gelu, silu) and 0.003 (gated) with it in
// bf16, without either by 0.0017; the bias gradient adds dz before its rounding where there is an activation.
template <int ACT, typename Z>
__global__ void __launch_bounds__(kActThreads, 4) expertActKernel(const __grid_constant__ ExpertActArgs a) {
  pdlEnter();
  constexpr bool kGated = ACT == ACT_SWIGLU || ACT == ACT_GEGLU;
  constexpr int kParts = kGated ? 2 : 1, kRows = kActThreads * 8 / kActCols;   // rows of a CTA at a time
  constexpr int kBase = ACT == ACT_SWIGLU ? ACT_SILU : ACT == ACT_GEGLU ? ACT_GELU : ACT;
  __shared__ float sums[kRows][kParts][kActCols];
  const int e = blockIdx.y, slice = blockIdx.z;
  const int pack = threadIdx.x % (kActCols / 8), ty = threadIdx.x / (kActCols / 8);
  const int col = blockIdx.x * kActCols + pack * 8;
  const int rows = rowsInUse(a.counts, e, a.cap);
  const bool inside = col < a.cols;
  const __nv_bfloat16* dout = (const __nv_bfloat16*)a.dout + (size_t)e * a.cap * a.cols + col;
  const size_t ld = (size_t)kParts * a.cols, base = (size_t)e * a.cap * ld + col;
  float acc[kParts][8];
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[p][i] = 0.0f;
  if (inside) {
#pragma unroll 2
    for (int row = slice * kRows + ty; row < rows; row += a.slices * kRows) {
      float g[8], z[kParts][8];
      unpackBf16x8(*(const uint4*)(dout + (size_t)row * a.cols), g);
      if (ACT != ACT_NONE) {
        const Z* pre = (const Z*)a.pre + base + (size_t)row * ld;
        __nv_bfloat16* dz = (__nv_bfloat16*)a.dz + base + (size_t)row * ld;
#pragma unroll
        for (int p = 0; p < kParts; ++p) load8(pre + p * a.cols, z[p]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float value, slope;
          activationAndSlope<kBase>(z[0][i], &value, &slope);
          if (kGated) {
            const float up = z[kParts - 1][i];
            z[kParts - 1][i] = g[i] * value;
            z[0][i] = g[i] * up * slope;
          } else {
            z[0][i] = g[i] * slope;
          }
        }
#pragma unroll
        for (int p = 0; p < kParts; ++p) *(uint4*)(dz + p * a.cols) = packBf16x8(z[p]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[0][i] = g[i];
      }
#pragma unroll
      for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[p][i] += z[p][i];
    }
  }
  if (!a.partial) return;
#pragma unroll
  for (int p = 0; p < kParts; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[ty][p][pack * 8 + i] = acc[p][i];
  __syncthreads();
  for (int i = threadIdx.x; i < kParts * kActCols; i += kActThreads) {
    const int p = i / kActCols, c = i % kActCols;
    if (blockIdx.x * kActCols + c >= a.cols) continue;
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) s += sums[r][p][c];
    a.partial[((size_t)slice * a.experts + e) * ld + (size_t)p * a.cols + blockIdx.x * kActCols + c] = s;
  }
}

// dbias = bf16(the slices' sums, in order), where no product on CTA pairs follows that would do it on the side. Short: 5 experts of 2200 columns 6 us
// under a profiler, most of them a launch's.
__global__ void __launch_bounds__(kActThreads) expertBiasKernel(const __grid_constant__ ExpertActArgs a) {
  pdlEnter();
  const size_t n = (size_t)a.experts * a.cols * (a.act == ACT_SWIGLU || a.act == ACT_GEGLU ? 2 : 1);
  biasFromSlices(a.partial, (__nv_bfloat16*)a.dbias, n, a.slices, (size_t)blockIdx.x * kActThreads + threadIdx.x, (size_t)gridDim.x * kActThreads);
}

template <typename Z>
static const void* actKernelFn(int act) {
  switch (act) {
    case ACT_RELU: return (const void*)expertActKernel<ACT_RELU, Z>;
    case ACT_GELU: return (const void*)expertActKernel<ACT_GELU, Z>;
    case ACT_SILU: return (const void*)expertActKernel<ACT_SILU, Z>;
    case ACT_SWIGLU: return (const void*)expertActKernel<ACT_SWIGLU, Z>;
    case ACT_GEGLU: return (const void*)expertActKernel<ACT_GEGLU, Z>;
    default: return nullptr;
  }
}
const void* expertActKernelFn(int act, bool preFp32) {
  if (act == ACT_NONE) return (const void*)expertActKernel<ACT_NONE, __nv_bfloat16>;   // (reads no z)
  return preFp32 ? actKernelFn<float>(act) : actKernelFn<__nv_bfloat16>(act);
}
const void* expertBiasKernelFn() { return (const void*)expertBiasKernel; }

// ---------------------------------------------------------------------------------------------- combine's gradient
// combine is out[t] = sum_k w[t,k] * y[row(t,k)], so dy[row] = w * dout[t] and dw[t,k] = <dout[t], y[row]>. One CTA per token: its
// gradient is read once for up to KR of the token's rows (eight at most), which are on their way together. The products' sums are joined lane by lane and warp by
// warp, in the same order every time. Memory bounds it: 4096 tokens of 8 rows of 7168, 168 us (5.9 TB/s).
template <int KR>
__global__ void __launch_bounds__(kMoeRowThreads) combineBackwardKernel(const __grid_constant__ MoeRowsArgs a) {
  pdlEnter();
  constexpr int kWarps = kMoeRowThreads / 32;
  __shared__ float sums[kWarps][KR];
  const int packs = a.hidden / 8, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (unsigned t = blockIdx.x; t < (unsigned)a.tokens; t += gridDim.x) {   // (signed, the last step may pass 2^31)
    const uint4* g4 = (const uint4*)a.dout + (size_t)t * packs;
    for (int k0 = 0; k0 < a.topk; k0 += KR) {
      int row[KR];
      float w[KR], dot[KR];
#pragma unroll
      for (int r = 0; r < KR; ++r) {
        row[r] = -1;
        w[r] = dot[r] = 0.0f;
        if (k0 + r < a.topk) {
          const size_t o = (size_t)t * a.topk + k0 + r;
          const int at = a.rows[o];
          if (at >= 0 && at < a.numRows) {
            row[r] = at;
            w[r] = a.weights[o];
          }
        }
      }
      for (int p = threadIdx.x; p < packs; p += kMoeRowThreads) {
        uint4 y[KR];
        const uint4 gq = g4[p];
#pragma unroll
        for (int r = 0; r < KR; ++r) y[r] = row[r] >= 0 ? __ldcs((const uint4*)a.y + (size_t)row[r] * packs + p) : make_uint4(0, 0, 0, 0);
        float g[8];
        unpackBf16x8(gq, g);
#pragma unroll
        for (int r = 0; r < KR; ++r) {
          if (row[r] < 0) continue;
          float f[8];
          unpackBf16x8(y[r], f);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dot[r] += g[i] * f[i];
            f[i] = w[r] * g[i];
          }
          __stcs((uint4*)a.dy + (size_t)row[r] * packs + p, packBf16x8(f));
        }
      }
#pragma unroll
      for (int r = 0; r < KR; ++r) {
#pragma unroll
        for (int o = 16; o; o >>= 1) dot[r] += __shfl_xor_sync(~0u, dot[r], o);
        if (lane == 0) sums[warp][r] = dot[r];
      }
      __syncthreads();
      if ((int)threadIdx.x < KR && k0 + (int)threadIdx.x < a.topk) {
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) s += sums[v][threadIdx.x];
        a.dweights[(size_t)t * a.topk + k0 + threadIdx.x] = s;
      }
      __syncthreads();
    }
  }
}

const void* combineBackwardKernelFn(int topk) {
  return topk <= 1 ? (const void*)combineBackwardKernel<1> : topk <= 2 ? (const void*)combineBackwardKernel<2>
         : topk <= 4 ? (const void*)combineBackwardKernel<4> : (const void*)combineBackwardKernel<8>;
}

// ---------------------------------------------------------------------------------------------- dispatch's gradient
// dispatch copies a token to a row of each of its experts, so dx[t] = sum_k dtoks[row(t,k)], in fp32 and in the order of the entries. Memory bounds it: 4096
// tokens of 8 rows of 7168, 89 us (5.9 TB/s).
__global__ void __launch_bounds__(kMoeRowThreads) dispatchBackwardKernel(const __grid_constant__ MoeRowsArgs a) {
  pdlEnter();
  constexpr int KR = 8;
  const int packs = a.hidden / 8;
  for (unsigned t = blockIdx.x; t < (unsigned)a.tokens; t += gridDim.x) {   // (signed, the last step may pass 2^31)
    for (int p = threadIdx.x; p < packs; p += kMoeRowThreads) {
      float acc[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
      for (int k0 = 0; k0 < a.topk; k0 += KR) {
        uint4 v[KR];
#pragma unroll
        for (int r = 0; r < KR; ++r) {
          v[r] = make_uint4(0, 0, 0, 0);
          if (k0 + r < a.topk) {
            const int row = a.rows[(size_t)t * a.topk + k0 + r];
            if (row >= 0 && row < a.numRows) v[r] = __ldcs((const uint4*)a.y + (size_t)row * packs + p);
          }
        }
#pragma unroll
        for (int r = 0; r < KR; ++r) {
          float f[8];
          unpackBf16x8(v[r], f);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] += f[i];
        }
      }
      ((uint4*)a.dx)[(size_t)t * packs + p] = packBf16x8(acc);
    }
  }
}
const void* dispatchBackwardKernelFn() { return (const void*)dispatchBackwardKernel; }

// ---------------------------------------------------------------------------------------------- rows of the last dispatch
// rows[t,k] = row of the dispatched tensor that holds the entry, -1 where there is none. rowOf keeps older words where the last dispatch
// wrote none (unused entries, rows beyond the capacity): a word counts when its row is in use and names this entry as its source.
__global__ void __launch_bounds__(kMoeRowThreads) dispatchRowsKernel(const __grid_constant__ DispatchRowsArgs a) {
  pdlEnter();
  for (size_t i = (size_t)blockIdx.x * kMoeRowThreads + threadIdx.x; i < a.entries; i += (size_t)gridDim.x * kMoeRowThreads) {
    const int64_t e = a.idx[i];
    const int row = a.rowOf[i];
    int got = -1;
    if (e >= 0 && e < a.experts && row / a.cap == (int)e && row - (int)e * a.cap < a.counts[e]) {
      const int2 from = a.srcInfo[row];
      if (from.x == a.rank && from.y == (int)i) got = row;
    }
    a.rows[i] = got;
  }
}
const void* dispatchRowsKernelFn() { return (const void*)dispatchRowsKernel; }

}  // namespace b200
