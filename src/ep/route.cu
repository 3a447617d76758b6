// Routing of tokens to experts: scores, an additive bias, groups, top-k and weights, forward and backward.
//
// For a token with logits l[0..E): s = softmax(l) or sigmoid(l); experts are ranked by s + bias. With groups (equal runs of neighbouring
// experts) a group's score is its best expert's rank value, or the sum of its two best; only the experts of the `keep` best groups
// remain. The topk best experts are taken, best first, equal ones (and equal groups) by index. Weights are scale * s of the taken
// experts, divided by their sum (sigmoid: plus 1e-20) when renormalised. The bias only chooses. A logit of -inf or NaN (or a rank value that is) takes its
// expert out; entries that find no expert are -1 with weight 0.
//
// One warp per token; a lane holds V neighbouring experts in registers, so that the lowest lane of equal ones has the lowest index.
// A pass of the selection is a maximum over the lane's values, one redux over the warp's and a ballot.
//
// What is chosen is what the formulas say in exact arithmetic, not what fp32 makes of them: without a bias experts are ranked by their
// logits, which order them as the scores do; where rounded values decide (bias, sums of two scores) and two that matter are nearer
// to each other than their rounding errors may be, the token is ranked again in 64 bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include "../kernels/common.cuh"
#include "moe_ops.h"

namespace b200 {

namespace {

constexpr int kRouteWarps = 4;
constexpr unsigned kAll = 0xffffffffu;

template <typename T> __device__ __forceinline__ float toFloat(T v);
template <> __device__ __forceinline__ float toFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ float toFloat<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float toFloat<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T fromFloat(float v);
template <> __device__ __forceinline__ float fromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half fromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 fromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A logit as the ranking sees it: -inf for experts that are out, the largest number for +inf (so that differences stay defined), no -0.
__device__ __forceinline__ float cleanLogit(float v) { return v > -INFINITY ? fminf(v, FLT_MAX) + 0.0f : -INFINITY; }

// The lane's V logits, experts lane * V ...; -inf behind the last.
template <typename T, int V>
__device__ __forceinline__ void loadLogits(const T* row, int experts, int e0, bool wide, float (&l)[V]) {
  constexpr int kPer = 16 / (int)sizeof(T) < V ? 16 / (int)sizeof(T) : V;   // of a pack
  if (wide && e0 + V <= experts) {
    struct alignas(kPer * sizeof(T)) Pack { T v[kPer]; };
#pragma unroll
    for (int p = 0; p < V / kPer; ++p) {
      const Pack q = *(const Pack*)(row + e0 + p * kPer);
#pragma unroll
      for (int i = 0; i < kPer; ++i) l[p * kPer + i] = cleanLogit(toFloat<T>(q.v[i]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) l[j] = e0 + j < experts ? cleanLogit(toFloat<T>(row[e0 + j])) : -INFINITY;
  }
}

__device__ __forceinline__ float warpSum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ double warpSum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// Orders floats (no NaN, no -0) as unsigned words.
__device__ __forceinline__ uint32_t orderedBits(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float fromOrdered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The largest value of the warp.
__device__ __forceinline__ float warpMax(float v) { return fromOrdered(__reduce_max_sync(kAll, orderedBits(v))); }
__device__ __forceinline__ double warpMax(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

__device__ __forceinline__ float expOf(float v) { return expf(v); }
__device__ __forceinline__ double expOf(double v) { return exp(v); }

__device__ __forceinline__ int groupOf(const RouteArgs& a, int e) { return a.groupMagic ? (int)__umulhi((uint32_t)e, a.groupMagic) : e; }

// Whether the order of two rank values (or sums of two) may be another one than that of the exact values: a score is off by a few
// units of 2^-24 of itself (exp, the sum, a division), and of 2^-24 in a softmax whose exponents are rounded differences; the sum with the bias by half a unit of itself.
__device__ __forceinline__ bool near(float above, float below) { return above - below <= 0x1p-20f + 0x1p-21f * fabsf(above); }

// Takes the token's experts into e (entry k in lane k, -1 = none). R = float: returns false when rounding may have decided.
template <typename R, int V>
__device__ __forceinline__ bool chooseExperts(const RouteArgs& a, const float (&l)[V], int lane, int* taken) {
  constexpr bool kExact = sizeof(R) == 8;
  const int e0 = lane * V;
  const bool byLogit = a.bias == nullptr, sums = a.groups > 1 && a.top2;
  bool sure = true;
  R v[V];
  if (byLogit && !sums) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (R)l[j];
  } else {
    if (a.sigmoid) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = (R)1 / ((R)1 + expOf((R)-l[j]));
    } else {
      R top = (R)l[0];
#pragma unroll
      for (int j = 1; j < V; ++j) top = (R)l[j] > top ? (R)l[j] : top;
      top = warpMax(top);
      R sum = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[j] = l[j] > -INFINITY ? expOf((R)l[j] - top) : (R)0;
        sum += v[j];
      }
      sum = warpSum(sum);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = v[j] / sum;   // (a token without experts: taken out below)
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (a.bias && e0 + j < a.experts) v[j] += (R)a.bias[e0 + j];
      if (!(l[j] > -INFINITY) || !(v[j] > (R)-INFINITY)) v[j] = (R)-INFINITY;
      v[j] += (R)0;
    }
  }

  if (a.groups > 1) {
    R score = (R)-INFINITY;   // of group `lane`
    for (int g = 0; g < a.groups; ++g) {
      R one = (R)-INFINITY, two = (R)-INFINITY;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (groupOf(a, e0 + j) == g && e0 + j < a.experts) {
          two = v[j] > one ? one : v[j] > two ? v[j] : two;
          one = v[j] > one ? v[j] : one;
        }
      }
      const R best = warpMax(one);
      R sum = best;
      if (sums) {
        const unsigned who = __ballot_sync(kAll, one == best);
        const R next = warpMax(lane == __ffs(who) - 1 ? two : one);
        if (next > (R)-INFINITY) sum += next;
      }
      if (lane == g) score = sum;
    }
    int ahead = 0;   // groups that are better than this lane's
    for (int g = 0; g < a.groups; ++g) {
      const R other = __shfl_sync(kAll, score, g);
      ahead += other > score || (other == score && g < lane);
    }
    const bool mine = lane < a.groups;
    const unsigned kept = __ballot_sync(kAll, mine && ahead < a.keep);
    if (!kExact && a.keep < a.groups && (!byLogit || sums)) {
      const float last = (float)__shfl_sync(kAll, score, __ffs(__ballot_sync(kAll, mine && ahead == a.keep - 1)) - 1);
      const float next = (float)__shfl_sync(kAll, score, __ffs(__ballot_sync(kAll, mine && ahead == a.keep)) - 1);
      if (near(last, next)) sure = false;
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e0 + j < a.experts && !(kept >> groupOf(a, e0 + j) & 1)) v[j] = (R)-INFINITY;
    if (byLogit && sums) {   // inside the groups the logits are the order
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = v[j] > (R)-INFINITY ? (R)l[j] : (R)-INFINITY;
    }
  }

  *taken = -1;
  R before = (R)INFINITY;
  int beforeAt = -1;
  const bool rounded = !kExact && !byLogit;
  for (int k = 0; k < a.topk + (rounded ? 1 : 0); ++k) {
    R best = v[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < V; ++j) {
      at = v[j] > best ? j : at;
      best = v[j] > best ? v[j] : best;
    }
    const R top = warpMax(best);
    if (!(top > (R)-INFINITY)) break;
    const int winner = __ffs(__ballot_sync(kAll, best == top)) - 1;
    const int e = winner * V + __shfl_sync(kAll, at, winner);
    if (rounded) {
      if (k > 0 && near((float)before, (float)top)) {
        // equal logits and biases have equal values in exact arithmetic too, and the lower index came first
        float mineA = 0.0f, mineB = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (e0 + j == beforeAt) mineA = l[j];
          if (e0 + j == e) mineB = l[j];
        }
        const bool same = __shfl_sync(kAll, mineA, beforeAt / V) == __shfl_sync(kAll, mineB, e / V) && a.bias[beforeAt] == a.bias[e];
        if (!same) sure = false;
      }
      before = top;
      beforeAt = e;
    }
    if (k < a.topk && lane == k) *taken = e;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e0 + j == e) v[j] = (R)-INFINITY;
  }
  return sure;
}

// The same in 64 bits, for the few tokens that need it.
template <typename T, int V>
__device__ __noinline__ int chooseExactly(const RouteArgs& a, const T* row, int lane) {
  float l[V];
  loadLogits<T, V>(row, a.experts, lane * V, false, l);
  int taken;
  chooseExperts<double, V>(a, l, lane, &taken);
  return taken;
}

// Largest value and sum of exp(l - largest) over the token's experts (sum 0 where there is none).
template <int V>
__device__ __forceinline__ void softmaxOf(const float (&l)[V], float* top, float* sum) {
  float m = l[0];
#pragma unroll
  for (int j = 1; j < V; ++j) m = fmaxf(m, l[j]);
  m = warpMax(m);
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) s += l[j] > -INFINITY ? expf(l[j] - m) : 0.0f;
  *top = m;
  *sum = warpSum(s);
}

// Each lane's share s / (sum of s + 1e-20) of sigmoid scores, 0 for l = -inf. All of it is held relative to exp(the largest logit, if negative), so that
// scores that fp32 has no numbers for keep their shares.
__device__ __forceinline__ float sigmoidShare(float l) {
  const float top = fminf(warpMax(l), 0.0f);
  if (!(top > -INFINITY)) return 0.0f;   // the same in all lanes
  const float t = l > -INFINITY ? (l > 0.0f ? 1.0f / (1.0f + expf(-l)) : expf(l - top) / (1.0f + expf(l))) : 0.0f;
  return t / (warpSum(t) + expf(-46.0517019f - top));   // 1e-20 = exp(-46.05...)
}

}  // namespace

template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32) routeKernel(const __grid_constant__ RouteArgs a) {
  pdlEnter();
  const int lane = threadIdx.x & 31, t = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = (const T*)a.logits + (size_t)t * a.experts;
  float l[V];
  loadLogits<T, V>(row, a.experts, lane * V, a.wide, l);
  int e;
  if (!chooseExperts<float, V>(a, l, lane, &e)) e = chooseExactly<T, V>(a, row, lane);
  const float le = e >= 0 ? cleanLogit(toFloat<T>(row[e])) : -INFINITY;
  float w;
  if (a.sigmoid) {
    w = a.renormalize ? sigmoidShare(le) : e >= 0 ? 1.0f / (1.0f + expf(-le)) : 0.0f;
  } else if (a.renormalize) {
    // the softmax over the taken experts alone
    const float top = warpMax(le);
    w = e >= 0 ? expf(le - top) : 0.0f;
    const float sum = warpSum(w);
    w = sum > 0.0f ? w / sum : 0.0f;
  } else {
    float top, sum;
    softmaxOf<V>(l, &top, &sum);
    w = e >= 0 ? expf(le - top) / sum : 0.0f;
  }
  if (lane < a.topk) {
    a.idx[(size_t)t * a.topk + lane] = e;
    a.weights[(size_t)t * a.topk + lane] = a.scale * w;
  }
}

// dlogits of sum_k dweights[k] * weights[k]. With u = weights / scale and g = scale * dweights:
//   softmax, renormalised: u is the softmax over the taken logits: d_k = u_k (g_k - sum_j g_j u_j);
//   softmax: d_e = [e taken] g_e s_e - s_e sum_j g_j s_j for every expert; sigmoid: d_k = g_k s_k (1 - s_k);
//   sigmoid, renormalised: u_k = s_k / (sum_j s_j + 1e-20) and d_k = (g_k - sum_j g_j u_j) u_k (1 - s_k).
// The selection is piecewise constant: it and the bias have no gradient. Entries of -1 (or outside) add nothing; an expert that is named
// twice gets both shares.
template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32) routeBackwardKernel(const __grid_constant__ RouteArgs a) {
  pdlEnter();
  const int lane = threadIdx.x & 31, t = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  const T* row = (const T*)a.logits + (size_t)t * a.experts;
  T* out = (T*)a.dlogits + (size_t)t * a.experts;
  const int e0 = lane * V;
  int e = -1;
  float g = 0.0f, le = -INFINITY;
  if (lane < a.topk) {
    const int64_t i = a.idx[(size_t)t * a.topk + lane];
    if (i >= 0 && i < a.experts) {
      le = cleanLogit(toFloat<T>(row[i]));
      if (le > -INFINITY) {
        e = (int)i;
        g = a.scale * a.dweights[(size_t)t * a.topk + lane];
      }
    }
  }
  float d[V];
#pragma unroll
  for (int j = 0; j < V; ++j) d[j] = 0.0f;
  float share;   // of expert e in its entry
  if (a.sigmoid) {
    const float u = a.renormalize ? sigmoidShare(le) : e >= 0 ? 1.0f / (1.0f + expf(-le)) : 0.0f;
    if (a.renormalize) g -= warpSum(g * u);
    // 1 - s without cancellation: exp(-l) / (1 + exp(-l)) = 1 / (1 + exp(l))
    share = e >= 0 ? g * u * (1.0f / (1.0f + expf(le))) : 0.0f;
  } else if (a.renormalize) {
    const float top = warpMax(le), x = e >= 0 ? expf(le - top) : 0.0f, total = warpSum(x);
    const float u = total > 0.0f ? x / total : 0.0f;
    share = u * (g - warpSum(g * u));
  } else {
    float l[V], top, sum;
    loadLogits<T, V>(row, a.experts, e0, a.wide, l);
    softmaxOf<V>(l, &top, &sum);
    share = e >= 0 ? g * (expf(le - top) / sum) : 0.0f;
    const float mean = warpSum(share);
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = l[j] > -INFINITY ? -mean * (expf(l[j] - top) / sum) : 0.0f;
  }
  for (int k = 0; k < a.topk; ++k) {
    const int ek = __shfl_sync(kAll, e, k);
    const float dk = __shfl_sync(kAll, share, k);
    if (ek < e0 || ek >= e0 + V) continue;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e0 + j == ek) d[j] += dk;
  }
  constexpr int kPer = 16 / (int)sizeof(T) < V ? 16 / (int)sizeof(T) : V;
  if (a.wide && e0 + V <= a.experts) {
    struct alignas(kPer * sizeof(T)) Pack { T v[kPer]; };
#pragma unroll
    for (int p = 0; p < V / kPer; ++p) {
      Pack q;
#pragma unroll
      for (int i = 0; i < kPer; ++i) q.v[i] = fromFloat<T>(d[p * kPer + i]);
      *(Pack*)(out + e0 + p * kPer) = q;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e0 + j < a.experts) out[e0 + j] = fromFloat<T>(d[j]);
  }
}

template <typename T>
static const void* routeFn(int experts, bool backward) {
#define B200_ROUTE(V) \
  if (experts <= 32 * V) return backward ? (const void*)routeBackwardKernel<T, V> : (const void*)routeKernel<T, V>
  B200_ROUTE(1);
  B200_ROUTE(2);
  B200_ROUTE(4);
  B200_ROUTE(8);
  B200_ROUTE(16);
  B200_ROUTE(32);
#undef B200_ROUTE
  return nullptr;
}
static const void* routeFnOf(int type, int experts, bool backward) {
  return type == ROUTE_F32 ? routeFn<float>(experts, backward) : type == ROUTE_F16 ? routeFn<__half>(experts, backward) : routeFn<__nv_bfloat16>(experts, backward);
}
const void* routeKernelFn(int type, int experts) { return routeFnOf(type, experts, false); }
const void* routeBackwardKernelFn(int type, int experts) { return routeFnOf(type, experts, true); }
int routeWarps() { return kRouteWarps; }

}  // namespace b200
