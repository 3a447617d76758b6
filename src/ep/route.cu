// Routing of tokens to experts: scores, an additive bias, groups, top-k and weights, forward and backward.
//
// For a token with logits l[0..E): s = softmax(l) or sigmoid(l); experts are ranked by s + bias. With groups (equal runs of neighbouring
// experts) a group's score is its best expert's rank value, or the sum of its two best; only the experts of the `keep` best groups
// remain. The topk best experts are taken, best first, equal ones (and equal groups) by index. Weights are scale * s of the taken
// experts, divided by their sum (sigmoid: plus 1e-20) when renormalised. The bias only chooses. A logit of -inf or NaN (or a rank value that is) takes its
// expert out; entries that find no expert are -1 with weight 0.
//
// One warp per token. Its lanes are dealt out to the groups (as many to each, a power of two), and a lane holds up to V neighbouring experts of its group in
// registers: the lowest lane of equal ones has the lowest index, and a group's score is a butterfly over its lanes. A pass of the selection is a
// maximum over the lane's values as ordered words, one redux over the warp's and a ballot. 8192 tokens of 256 experts: 6.6 us by
// bf16 logits alone, 12.4 with a bias, 14.6 in 8 groups too, where the bytes would take 0.8. Instructions are most of that, 1109 of a warp for each token: under a profiler (18.5 us, caches
// cold) the SMs are busy for 11.4 us and issue in 69 % of their cycles, the integer units take 61 %; the rest of the time is the start, the logits' way from memory, and a second wave that is
// not full (1.7 of 8 CTAs per SM). Occupancies from 24 to 64 warps per SM made no difference.
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

// Which experts a lane holds: `n` from e0 on.
struct Share {
  int e0, n;
};
__device__ __forceinline__ Share shareOf(const RouteArgs& a, int lane) {
  const int group = lane / a.lanes, in = lane % a.lanes * a.perLane;   // lanes is a power of two
  return {group * a.perGroup + in, group < a.groups ? max(0, min(a.perLane, a.perGroup - in)) : 0};
}

// The lane's logits; -inf behind the last.
template <typename T, int V>
__device__ __forceinline__ void loadLogits(const T* row, const Share& my, bool wide, float (&l)[V]) {
  constexpr int kPer = 16 / (int)sizeof(T) < V ? 16 / (int)sizeof(T) : V;   // of a pack
  if (wide && my.n == V) {
    struct alignas(kPer * sizeof(T)) Pack { T v[kPer]; };
#pragma unroll
    for (int p = 0; p < V / kPer; ++p) {
      const Pack q = *(const Pack*)(row + my.e0 + p * kPer);
#pragma unroll
      for (int i = 0; i < kPer; ++i) l[p * kPer + i] = cleanLogit(toFloat<T>(q.v[i]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) l[j] = j < my.n ? cleanLogit(toFloat<T>(row[my.e0 + j])) : -INFINITY;
  }
}

// The sum of a lane's values as a tree: six additions in a row for 64 of them, where one after the other would round 63 times.
template <int FROM, int N, typename R, int V>
__device__ __forceinline__ R treeSum(const R (&v)[V]) {
  if constexpr (N == 1) return v[FROM];
  else return treeSum<FROM, N / 2>(v) + treeSum<FROM + N / 2, N / 2>(v);
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

// Numbers (no NaN, no -0) as unsigned words in their order; 0 is below all of them.
__device__ __forceinline__ uint32_t orderedBits(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t orderedBits(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return b ^ ((uint64_t)((long long)b >> 63) | 0x8000000000000000ull);
}
template <typename T> __device__ __forceinline__ uint32_t orderedBits16(T v) {
  const uint32_t b = *(const uint16_t*)&v;
  return b ^ (b & 0x8000u ? 0xffffu : 0x8000u);
}
__device__ __forceinline__ float fromOrdered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// The largest of the warp.
__device__ __forceinline__ uint32_t warpMax(uint32_t v) { return __reduce_max_sync(kAll, v); }
__device__ __forceinline__ uint64_t warpMax(uint64_t v) {
  const uint32_t high = __reduce_max_sync(kAll, (uint32_t)(v >> 32));
  return (uint64_t)high << 32 | __reduce_max_sync(kAll, (uint32_t)(v >> 32) == high ? (uint32_t)v : 0u);
}
__device__ __forceinline__ float warpMax(float v) { return fromOrdered(warpMax(orderedBits(v))); }
__device__ __forceinline__ double warpMax(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// For the ranking: in fp32 the short forms, whose errors `near` allows for.
__device__ __forceinline__ float rankExp(float v) { return __expf(v); }
__device__ __forceinline__ double rankExp(double v) { return exp(v); }
__device__ __forceinline__ float rankDivide(float a, float b) { return __fdividef(a, b); }
__device__ __forceinline__ double rankDivide(double a, double b) { return a / b; }

// A lane's words, best first. Up to 8 are sorted once (by neighbours, so that equal ones keep their order) with their places in the
// nibbles of a register: taking one off moves the others up. Searching all of them in every pass took twice the instructions. UNIQUE: no two
// are equal, and nobody asks for places.
template <typename Key, int V, bool UNIQUE, bool SORTED = V <= 8>
struct Heads {
  Key key[V];
  uint32_t places = 0;
  __device__ __forceinline__ explicit Heads(const Key (&k)[V]) {
    int place[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      key[j] = k[j];
      place[j] = j;
    }
#pragma unroll
    for (int round = 0; round < V; ++round)
#pragma unroll
      for (int j = round & 1; j + 1 < V; j += 2) {
        const bool swap = key[j + 1] > key[j];
        const Key high = max(key[j], key[j + 1]);
        key[j + 1] = min(key[j], key[j + 1]);
        key[j] = high;
        if (UNIQUE) continue;
        const int p = swap ? place[j + 1] : place[j];
        place[j + 1] = swap ? place[j] : place[j + 1];
        place[j] = p;
      }
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (!UNIQUE) places |= (uint32_t)place[j] << 4 * j;
  }
  __device__ __forceinline__ Key best() const { return key[0]; }
  __device__ __forceinline__ int at(Key) const { return places & 15; }
  __device__ __forceinline__ void drop(Key) {
#pragma unroll
    for (int j = 0; j + 1 < V; ++j) key[j] = key[j + 1];
    key[V - 1] = 0;
    places >>= 4;
  }
  __device__ __forceinline__ void dropIf(Key top) {
    if (key[0] == top) drop(top);
  }
};
template <typename Key, int V, bool UNIQUE>
struct Heads<Key, V, UNIQUE, false> {
  Key key[V];
  __device__ __forceinline__ explicit Heads(const Key (&k)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = k[j];
  }
  __device__ __forceinline__ Key best() const {
    Key b = key[0];
#pragma unroll
    for (int j = 1; j < V; ++j) b = max(b, key[j]);
    return b;
  }
  __device__ __forceinline__ int at(Key top) const {
    int e = 0;
#pragma unroll
    for (int j = V - 1; j >= 0; --j) e = key[j] == top ? j : e;
    return e;
  }
  __device__ __forceinline__ void drop(Key top) {
    const int e = at(top);
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = j == e ? (Key)0 : key[j];
  }
  __device__ __forceinline__ void dropIf(Key top) {   // (unique)
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = key[j] == top ? (Key)0 : key[j];
  }
};

// Whether the order of two rank values (or sums of two) may be another one than that of the exact values. In units of u = 2^-23 the short exponential of x is off by
// 2 + 1.2 |x| of itself, its argument's rounding adds 0.5 |x|, the division 2. Of a sigmoid that is s (1 - s) (2 + 1.2 |l|) + 2 s < 4. Of softmax shares p = e^x / sum, of
// which up to four are compared: sum of p (2 + 1.7 |x|) < 3 for themselves, as much and the same over all other experts (at most 1.7 * 1.9, where those have half of the sum) for the
// denominator's terms, 5.5 for adding it up (trees of six additions in a lane and five over the warp) and 2 for the division, less than 14 in all. So differences of two values, or of sums
// of two, are off by less than 16 u = 2^-19. Adding the bias and the second
// value rounds by half a unit each: 2^-21 of `size`, the largest sum of magnitudes on either side, holds all of it. (Not of the value itself: two that cancel leave little of it, and all of their
// rounding.) Infinite values, as sums beyond fp32 are, and a size beyond fp32 are near to everything.
__device__ __forceinline__ bool near(float above, float below, float size) { return !(above - below > 0x1p-19f + 0x1p-21f * size); }

// The token's experts (entry k in lane k, -1 = none). R = float: *sure says whether rounding may have decided.
template <typename R, typename T, int V>
__device__ __forceinline__ int chooseExperts(const RouteArgs& a, const T* row, const Share& my, const float (&l)[V], int lane, bool* sure) {
  constexpr bool kExact = sizeof(R) == 8;
  using Key = decltype(orderedBits((R)0));
  const bool byLogit = a.bias == nullptr, sums = a.groups > 1 && a.top2, scores = !byLogit || sums;
  *sure = true;
  R v[V];   // rank values, -inf for experts that are out
  if (!scores) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (R)l[j];
  } else {
    if (a.sigmoid) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = rankDivide((R)1, (R)1 + rankExp((R)-l[j]));
    } else {
      R top = (R)l[0];
#pragma unroll
      for (int j = 1; j < V; ++j) top = (R)l[j] > top ? (R)l[j] : top;
      top = warpMax(top);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = l[j] > -INFINITY ? rankExp((R)l[j] - top) : (R)0;
      const R sum = warpSum(treeSum<0, V>(v));
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = rankDivide(v[j], sum);   // (a token without experts: taken out below)
    }
    if (!byLogit) {
      if (V % 4 == 0 && a.wideBias && my.n == V) {
#pragma unroll
        for (int p = 0; p < V / 4; ++p) {
          const float4 q = *(const float4*)(a.bias + my.e0 + p * 4);
          v[p * 4] += (R)q.x;
          v[p * 4 + 1 < V ? p * 4 + 1 : 0] += (R)q.y;
          v[p * 4 + 2 < V ? p * 4 + 2 : 0] += (R)q.z;
          v[p * 4 + 3 < V ? p * 4 + 3 : 0] += (R)q.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < my.n) v[j] += (R)a.bias[my.e0 + j];
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      v[j] = l[j] > -INFINITY && v[j] > (R)-INFINITY ? v[j] + (R)0 : (R)-INFINITY;
    }
  }

  bool mine = true;   // whether this lane's group stays
  if (a.groups > 1) {
    R one = v[0], two = (R)-INFINITY;
#pragma unroll
    for (int j = 1; j < V; ++j) {
      two = v[j] > one ? one : v[j] > two ? v[j] : two;
      one = v[j] > one ? v[j] : one;
    }
    for (int o = 1; o < a.lanes; o <<= 1) {
      const R other = __shfl_xor_sync(kAll, one, o), next = __shfl_xor_sync(kAll, two, o);
      const R low = other > one ? one : other;
      one = other > one ? other : one;
      two = next > two ? next : two;
      two = low > two ? low : two;
    }
    const R score = sums && two > (R)-INFINITY ? one + two : one;
    const int group = lane / a.lanes;
    int ahead = 0;   // groups that are better
    for (int g = 0; g < a.groups; ++g) {
      const R other = __shfl_sync(kAll, score, g * a.lanes);
      ahead += other > score || (other == score && g < group);
    }
    mine = group < a.groups && ahead < a.keep;
    if (!kExact && scores) {
      const bool real = group < a.groups;
      const int lastLane = __ffs(__ballot_sync(kAll, real && ahead == a.keep - 1)) - 1, nextLane = __ffs(__ballot_sync(kAll, real && ahead == a.keep)) - 1;
      const float last = (float)__shfl_sync(kAll, score, lastLane), next = (float)__shfl_sync(kAll, score, nextLane);
      const float size = !(one > (R)-INFINITY) ? 0.0f : fabsf((float)one) + (sums && two > (R)-INFINITY ? fabsf((float)two) : 0.0f);   // (0: no expert)
      const float larger = fmaxf(__shfl_sync(kAll, size, lastLane), __shfl_sync(kAll, size, nextLane));
      if (near(last, next, larger) && (last > -INFINITY || larger > 0.0f)) *sure = false;   // (of groups without experts the lower ones stay)
    }
  }
  if constexpr (sizeof(T) == 2 && !kExact) {
    if (byLogit) {
      // The logit's 16 bits and the expert's number make a word that no other expert has: the largest says which one it is
      uint32_t word[V];
#pragma unroll
      for (int j = 0; j < V; ++j) word[j] = mine && v[j] > (R)-INFINITY ? orderedBits16(fromFloat<T>(l[j])) << 16 | (uint32_t)(0xffff - (my.e0 + j)) : 0u;
      Heads<uint32_t, V, true> heads(word);
      int taken = -1;
      for (int k = 0; k < a.topk; ++k) {
        const uint32_t top = warpMax(heads.best());
        if (top == 0) break;
        heads.dropIf(top);
        if (lane == k) taken = 0xffff - (int)(top & 0xffff);
      }
      return taken;
    }
  }
  Key key[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const R rank = byLogit && sums ? (R)l[j] : v[j];   // inside the groups the logits are the order
    key[j] = mine && v[j] > (R)-INFINITY ? orderedBits(rank) : (Key)0;
  }

  Heads<Key, V, false> heads(key);
  int taken = -1;
  Key value = 0;   // of this lane's entry
  const bool rounded = !kExact && !byLogit;
  const int passes = a.topk + (rounded ? 1 : 0);   // with the best of those that are left
  for (int k = 0; k < passes; ++k) {
    const Key best = heads.best(), top = warpMax(best);
    if (top == 0) break;
    const int winner = __ffs(__ballot_sync(kAll, best == top)) - 1;
    const int e = __shfl_sync(kAll, my.e0 + heads.at(top), winner);
    if (lane == winner) heads.drop(top);
    if (lane == k) {
      taken = e;
      value = top;
    }
  }
  if (rounded) {
    // two next to each other that are too near; equal logits and biases have equal values in exact arithmetic too, and the lower index came first
    const float own = fromOrdered((uint32_t)value), above = __shfl_up_sync(kAll, own, 1);
    const int other = __shfl_up_sync(kAll, taken, 1);
    const bool doubt = lane > 0 && taken >= 0 && near(above, own, fabsf(above)) && !(cleanLogit(toFloat<T>(row[taken])) == cleanLogit(toFloat<T>(row[other])) && a.bias[taken] == a.bias[other]);
    if (__any_sync(kAll, doubt)) *sure = false;
    if (lane >= a.topk) taken = -1;
  }
  return taken;
}

// The same in 64 bits, for the few tokens that need it.
template <typename T, int V>
__device__ __noinline__ int chooseExactly(const RouteArgs& a, const T* row, int lane) {
  const Share my = shareOf(a, lane);
  float l[V];
  loadLogits<T, V>(row, my, false, l);
  bool sure;
  return chooseExperts<double, T, V>(a, row, my, l, lane, &sure);
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
  const Share my = shareOf(a, lane);
  float l[V];
  loadLogits<T, V>(row, my, a.wide, l);
  bool sure;
  int e = chooseExperts<float, T, V>(a, row, my, l, lane, &sure);
  if (!sure) e = chooseExactly<T, V>(a, row, lane);
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
  const Share my = shareOf(a, lane);
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
    loadLogits<T, V>(row, my, a.wide, l);
    softmaxOf<V>(l, &top, &sum);
    share = e >= 0 ? g * (expf(le - top) / sum) : 0.0f;
    const float mean = warpSum(share);
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = l[j] > -INFINITY ? -mean * (expf(l[j] - top) / sum) : 0.0f;
  }
  for (int k = 0; k < a.topk; ++k) {
    const int ek = __shfl_sync(kAll, e, k);
    const float dk = __shfl_sync(kAll, share, k);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (my.e0 + j == ek) d[j] += dk;
  }
  constexpr int kPer = 16 / (int)sizeof(T) < V ? 16 / (int)sizeof(T) : V;
  if (a.wide && my.n == V) {
    struct alignas(kPer * sizeof(T)) Pack { T v[kPer]; };
#pragma unroll
    for (int p = 0; p < V / kPer; ++p) {
      Pack q;
#pragma unroll
      for (int i = 0; i < kPer; ++i) q.v[i] = fromFloat<T>(d[p * kPer + i]);
      *(Pack*)(out + my.e0 + p * kPer) = q;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < my.n) out[my.e0 + j] = fromFloat<T>(d[j]);
  }
}

template <typename T>
static const void* routeFn(int perLane, bool backward) {
#define B200_ROUTE(V) \
  if (perLane <= V) return backward ? (const void*)routeBackwardKernel<T, V> : (const void*)routeKernel<T, V>
  B200_ROUTE(1);
  B200_ROUTE(2);
  B200_ROUTE(4);
  B200_ROUTE(8);
  B200_ROUTE(16);
  B200_ROUTE(32);
#undef B200_ROUTE
  return backward ? nullptr : (const void*)routeKernel<T, kRouteMaxPerLane>;   // backwards there are no groups that leave lanes idle
}
static const void* routeFnOf(int type, int perLane, bool backward) {
  return type == ROUTE_F32 ? routeFn<float>(perLane, backward) : type == ROUTE_F16 ? routeFn<__half>(perLane, backward) : routeFn<__nv_bfloat16>(perLane, backward);
}
const void* routeKernelFn(int type, int perLane) { return routeFnOf(type, perLane, false); }
const void* routeBackwardKernelFn(int type, int perLane) { return routeFnOf(type, perLane, true); }
int routeWarps() { return kRouteWarps; }

}  // namespace b200
