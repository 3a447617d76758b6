// Attention for sm_100a, the forward pass: o_i = sum_j p_ij v_j / l_i over the keys j that query i sees, p_ij = exp(scale q_i.k_j - m_i), l_i their sum, and
// lse_i = m_i + ln l_i. One pass over the keys with a running maximum: probabilities never reach memory.
//
// One CTA per SM, in roles:
//   warps 0-7   two groups of four; a thread holds a row of 128 scores: maximum, exponentials, their sum, and the probabilities in 16 bits back into
//               tensor memory, over the scores. The maximum is only raised (and the sums so far multiplied) where a score passes it by 2^8: the largest
//               probability is then 2^8 instead of 1, which costs nothing in a floating-point type.
//   warp 8      TMA producer: tiles of queries once, keys and values through a ring in shared memory
//   warp 9      MMA issuer: S = Q K^T from shared memory, O += P V with P from tensor memory
// While one group works on its scores the tensor cores work for the other. In the form for many rows ("pairs") the groups have a tile of 128 rows of
// queries each; in the form for less than that ("single") they share one and take the tiles of keys in turn, and their results are joined at the end. There the keys may also be cut into
// parts for several CTAs, whose results a second kernel joins; so they may in the form for a decoder's few rows, below.
//
// What bounds it: at 128 channels a tile of 128 x 128 scores is 1024 cycles for the tensor cores and as many for its exponentials (16 a cycle), and takes 1800: a group's products, maximum
// and exponentials depend on one another, and two groups hide that in part. 8192 x 8192 of 32 heads over 8, everything seen, 822 to 850 us after a rest (1.3 PFLOP/s), causal 441 to 453; the
// products alone 635, all but the products 709. Pass after pass the power limit has the clock down, and it is 999 and 515 to 531 us. Single queries are bound by memory: 64 on 8192 keys each, 32 heads over 8, 2.1 GB, 316 to 327 us.
//
// Rows behind a tile's last are whatever shared memory held: they reach only results that nobody stores. Values behind a sequence's last key may be
// anything (0 * NaN is NaN): zeros are written over them in shared memory.
// Every wait is bounded; on expiry the kernel records a status, waits for its copies and products in flight, frees its tensor memory and returns.
#include "attention.cuh"

namespace b200 {

using namespace attn;

namespace {

constexpr uint32_t kTmemCols = 512;
constexpr float kLag = 8.0f;   // by how many powers of two a score may pass the running maximum

template <int DP, bool PAIRS> struct ForwardShape {
  static constexpr uint32_t kTileBytes = DP / 64 * kHalfTile;
  static constexpr int kQTiles = PAIRS ? 2 : 1;
  static constexpr int kStages = (PAIRS ? 4 : 6) * (DP == 64 ? 2 : 1) - (!PAIRS && DP == 64 ? 1 : 0);
  static constexpr uint32_t kRing = kQTiles * kTileBytes, kCtrl = kRing + kStages * kTileBytes;
  static_assert((2 * kStages + 10) * 8 + 8 <= 512, "control block");
  static constexpr uint32_t kExchange = kCtrl + 512;       // maxima and sums of the second group's rows, where it has the first one's
  static constexpr size_t kBytes = kExchange + (PAIRS ? 0 : 1024);   // (dynamic shared memory, all that this kernel has, begins on a multiple of 1024 bytes)
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

// The order in which tiles of keys and values go through the ring: K0 V0 K1 V1 ... where one tile serves both groups, K0 K1 V0 K2 V1 K3 ... where the groups take turns.
template <bool PAIRS> __device__ __forceinline__ int placeOfK(int i) { return PAIRS ? 2 * i : i < 2 ? i : 2 * i - 1; }
template <bool PAIRS> __device__ __forceinline__ int placeOfV(int i, int n) { return PAIRS ? 2 * i + 1 : min(i + 2, n) + i; }

// The largest of 64 scores.
__device__ __forceinline__ float maxOf(const uint32_t (&x)[32], const uint32_t (&y)[32]) {
  float a = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])), b = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
#pragma unroll
  for (int k = 2; k < 32; k += 2) {
    a = max3(a, __uint_as_float(x[k]), __uint_as_float(x[k + 1]));
    b = max3(b, __uint_as_float(y[k]), __uint_as_float(y[k + 1]));
  }
  return fmaxf(a, b);
}

// A row's 128 scores become probabilities in 16 bits, in their place; m and l are its maximum and sum so far, of the keys from k0 on those in front of `limit` count. Where the
// maximum is raised the sums of `sums` (if there are any yet) are multiplied.
template <typename T, int DP>
__device__ __forceinline__ void softmaxTile(uint32_t tS, uint32_t tO, bool sums, int limit, int k0, float c, uint64_t c2, float& m, float& l, uint32_t probBar, int lane) {
  uint32_t s[4][32];
  tmemLd32(tS, s[0]);
  tmemLd32(tS + 32, s[1]);
  tmemLdWait32(s[0]);
  tmemLdWait32(s[1]);
  tmemLd32(tS + 64, s[2]);
  tmemLd32(tS + 96, s[3]);
  // the first half's maximum while the second half is on its way, unless some of it is hidden
  const bool hide = __any_sync(~0u, limit < k0 + 128);
  float mx = hide ? 0.0f : maxOf(s[0], s[1]);
  tmemLdWait32(s[2]);
  tmemLdWait32(s[3]);
  if (hide) {
#pragma unroll
    for (int k = 0; k < 128; ++k)
      if (k0 + k >= limit) s[k / 32][k % 32] = __float_as_uint(-INFINITY);
    mx = maxOf(s[0], s[1]);
  }
  mx = fmaxf(mx, maxOf(s[2], s[3]));
  const bool raise = (mx - m) * c > kLag;   // (nothing seen so far and nothing now: NaN, no)
  if (__any_sync(~0u, raise)) {
    const float to = raise ? mx : m, factor = raise ? exp2Fast((m - to) * c) : 1.0f;
    m = to;
    l *= factor;
    if (sums) {
      // the products that wrote these sums were issued, and finished, in front of the scores
#pragma unroll
      for (int k = 0; k < DP / 32; ++k) {
        uint32_t o[32];
        tmemLd32(tO + k * 32, o);
        tmemLdWait32(o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
        tmemSt32(tO + k * 32, o);
      }
    }
  }
  const float shift = Pack<T>::kForwardBias - (m == -INFINITY ? 0.0f : m * c);
  const uint64_t shift2 = pair(shift, shift);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t p[32];
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      uint32_t &lo = s[half * 2 + k / 16][k % 16 * 2], &hi = s[half * 2 + k / 16][k % 16 * 2 + 1];
      const uint64_t x = fma2(packF32x2(lo, hi), c2, shift2);
      lo = __float_as_uint(exp2Fast(lowOf(x)));
      hi = __float_as_uint(exp2Fast(highOf(x)));
      p[k] = Pack<T>::two(__uint_as_float(lo), __uint_as_float(hi));
    }
    tmemSt32(tS + half * 64, p);
  }
  tmemStWait();
  tcFenceBefore();
  __syncwarp();
  if (lane == 0) mbarArrive(probBar);
  // the sum is added up while the tensor cores work on the probabilities
  uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 64; ++k) sum[k % 4] = add2(sum[k % 4], packF32x2(s[k / 16][k % 16 * 2], s[k / 16][k % 16 * 2 + 1]));
  sum[0] = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
  l += lowOf(sum[0]) + highOf(sum[0]);
}

// What a row's log-sum-exp and the reciprocal of its sum say of its result: what the sums are multiplied by (`share`), and, where other keys' results are joined, those and their
// share.
__device__ __forceinline__ void closeRow(const AttnArgs& a, float lse, float inv, size_t at, size_t atLse, int part, bool valid, bool exists, float& share, float& joined,
                                         const float*& from) {
  share = inv;
  joined = 0.0f;
  from = nullptr;
  if (a.splits > 1) {
    if (exists) a.partLse[(size_t)part * a.batch * a.q * a.heads + at] = lse;
  } else {
    if (a.joinOut && valid) {
      const float other = a.joinLse[atLse], top = fmaxf(lse, other);
      if (top != -INFINITY) {
        const float x = expf(lse - top), y = expf(other - top), both = x + y;
        lse = top + logf(both);
        share = inv * x / both;
        joined = y / both;
        from = a.joinOut + at * a.dim;
      }
    }
    if (exists) a.lse[atLse] = lse;
  }
}

// 32 channels of a row's result, or of a part's.
template <typename T>
__device__ __forceinline__ void storeChannels(const AttnArgs& a, float (&f)[32], int channel, size_t at, int part, const float* from, float joined) {
  if (from) {
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      if (channel + e >= a.dim) break;
      const float4 v = *(const float4*)(from + channel + e);
      f[e] += joined * v.x; f[e + 1] += joined * v.y; f[e + 2] += joined * v.z; f[e + 3] += joined * v.w;
    }
  }
  if (a.splits > 1 || a.outFp32) {
    float* to = a.splits > 1 ? a.partOut + ((size_t)part * a.batch * a.q * a.heads + at) * a.dim : (float*)a.out + at * a.dim;
#pragma unroll
    for (int e = 0; e < 32; e += 4)
      if (channel + e < a.dim) *(float4*)(to + channel + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
  } else {
    uint16_t* to = (uint16_t*)a.out + at * a.dim;
#pragma unroll
    for (int e = 0; e < 32; e += 8)
      if (channel + e < a.dim)
        *(uint4*)(to + channel + e) = make_uint4(Pack<T>::two(f[e], f[e + 1]), Pack<T>::two(f[e + 2], f[e + 3]), Pack<T>::two(f[e + 4], f[e + 5]), Pack<T>::two(f[e + 6], f[e + 7]));
  }
}

template <typename T, int DP, bool PAIRS>
__global__ void __launch_bounds__(ForwardWarps::kThreads, 1)
attnForwardKernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ AttnArgs a) {
  using Shape = ForwardShape<DP, PAIRS>;
  using W = ForwardWarps;
  constexpr int kStages = Shape::kStages;
  constexpr uint32_t kTileBytes = Shape::kTileBytes;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* fullBar = (uint64_t*)(smem + Shape::kCtrl);   // [kStages]
  uint64_t* emptyBar = fullBar + kStages;                 // [kStages]
  uint64_t* qBar = emptyBar + kStages;                    // [2]
  uint64_t* scoreBar = qBar + 2;                          // [2] scores of a group are there
  uint64_t* probBar = scoreBar + 2;                       // [2] its probabilities are
  uint64_t* outBar = probBar + 2;                         // [2] its sums are complete
  uint64_t* fixBar = outBar + 2;                          // the last values have zeros behind them
  uint64_t* drainBar = fixBar + 1;
  uint32_t* tmemSlot = (uint32_t*)(drainBar + 1);
  volatile uint32_t* abortFlag = tmemSlot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbarInit(smemAddr(&fullBar[s]), 1); mbarInit(smemAddr(&emptyBar[s]), 1); }
    for (int t = 0; t < 2; ++t) { mbarInit(smemAddr(&qBar[t]), 1); mbarInit(smemAddr(&scoreBar[t]), 1); mbarInit(smemAddr(&probBar[t]), 4); mbarInit(smemAddr(&outBar[t]), 1); }
    mbarInit(smemAddr(fixBar), 1);
    mbarInit(smemAddr(drainBar), 1);
    *abortFlag = 0;
    mbarInitFence();
    prefetchTensorMap(&tmQ);
    prefetchTensorMap(&tmK);
    prefetchTensorMap(&tmV);
  }
  if (warp == W::kMma) {
    tmemAlloc(smemAddr(tmemSlot), kTmemCols);
    tmemRelinquish();
  }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmem = *tmemSlot;
  pdlEnter();   // the set-up above overlaps the end of the kernel before

  // ---- this CTA's share: the tiles of queries with the most visible keys come first
  const unsigned owners = a.batch * a.kvHeads, owner = blockIdx.x % owners, share = blockIdx.x / owners;
  const int kvHead = owner % a.kvHeads, b = owner / a.kvHeads, part = PAIRS ? 0 : share % a.splits;
  const int tile0 = (int)(gridDim.x / owners - 1 - share) / (PAIRS ? 1 : a.splits) * Shape::kQTiles;
  const Sequence seq = sequenceOf(a, b);
  int begin = 0, n = 0, count[2];   // tiles of keys: the first of this part, how many for both groups, and for each
  int tok0[2];
  if (PAIRS) {
    for (int t = 0; t < 2; ++t) {
      tok0[t] = (tile0 + t) * a.tileTokens;
      const int last = min(tok0[t] + a.tileTokens, seq.q) - 1;
      count[t] = last < tok0[t] ? 0 : (visibleOf(a, seq, last) + 127) / 128;
      n = max(n, count[t]);
    }
  } else {
    tok0[0] = tok0[1] = tile0 * a.tileTokens;
    const int last = min(tok0[0] + a.tileTokens, seq.q) - 1;
    const int all = last < tok0[0] ? 0 : (visibleOf(a, seq, last) + 127) / 128;
    const int each = (all + a.splits - 1) / a.splits;
    begin = min(all, part * each);
    n = min(all, begin + each) - begin;
    count[0] = (n + 1) / 2;
    count[1] = n / 2;
  }
  // values behind the sequence's last: the tensor map gives zeros behind the tensor's last
  const int fixTile = seq.kv < a.kv && seq.kv % 128 ? seq.kv / 128 - begin : -1;
  const uint32_t smem0 = smemAddr(smem);
  auto fail = [&](uint32_t what) {
    *abortFlag = 1;
    reportTimeout(a.status, what);
  };

  if (warp >= W::kCompute) regsGive<W::kFewRegs>();
  if (warp == W::kProducer) {
    uint32_t armed = 0, qArmed = 0;   // bits: stages and tiles of queries on their way
    int place = 0;
    bool ok = true;
    auto next = [&](const CUtensorMap* map, int tile) {
      const int s = place % kStages;
      const uint32_t ph = (place / kStages) & 1;
      ok = ok && warpWaitOr(smemAddr(&emptyBar[s]), ph ^ 1, abortFlag);
      if (!ok) {
        if (lane == 0) fail(1000 + s);
        return;
      }
      if (lane == 0) {
        const uint32_t bar = smemAddr(&fullBar[s]);
        mbarExpectTx(bar, kTileBytes);
        loadTile<DP>(smem0 + Shape::kRing + s * kTileBytes, map, (begin + tile) * 128, kvHead, b, bar);
      }
      armed |= 1u << s;
      ++place;
    };
    if (n > 0) {
      if (lane == 0)
        for (int t = 0; t < Shape::kQTiles; ++t) {
          if (!count[t]) continue;
          mbarExpectTx(smemAddr(&qBar[t]), DP / 64 * a.tileTokens * a.group * 128);
          loadTile<DP>(smem0 + t * kTileBytes, &tmQ, tok0[t], kvHead * a.group, b, smemAddr(&qBar[t]));
        }
      for (int t = 0; t < Shape::kQTiles; ++t) qArmed |= count[t] ? 1u << t : 0u;
      if (PAIRS) {
        for (int i = 0; i < n && ok; ++i) {
          next(&tmK, i);
          if (ok) next(&tmV, i);
        }
      } else {
        for (int i = 0; i < min(n, 2) && ok; ++i) next(&tmK, i);
        for (int i = 0; i < n && ok; ++i) {
          next(&tmV, i);
          if (ok && i + 2 < n) next(&tmK, i + 2);
        }
      }
      if (ok && fixTile >= 0 && fixTile < n) {
        const int at = placeOfV<PAIRS>(fixTile, n), s = at % kStages;   // the last tile: its stage is not used again
        ok = warpWaitOr(smemAddr(&fullBar[s]), (at / kStages) & 1, abortFlag);
        if (ok) {
          clearRows<DP>(smem + Shape::kRing + s * kTileBytes, seq.kv % 128, lane);
          if (lane == 0) mbarArrive(smemAddr(fixBar));
        } else if (lane == 0) {
          fail(1100);
        }
      }
      if (__any_sync(~0u, *abortFlag)) {
        // copies already issued still write into this CTA's shared memory: wait for them (bounded)
        for (int s = 0; s < kStages; ++s)
          if (armed >> s & 1) mbarWait(smemAddr(&fullBar[s]), (uint32_t)((place - 1 - (place - 1 - s + kStages) % kStages) / kStages) & 1, 1u << 20);
        for (int t = 0; t < 2; ++t)
          if (qArmed >> t & 1) mbarWait(smemAddr(&qBar[t]), 0, 1u << 20);
      }
    }
  } else if (warp == W::kMma) {
    if (n > 0 && electOne()) {
      bool ok = true;
      auto need = [&](bool got, uint32_t what) {
        if (ok && !got) fail(what);
        ok = ok && got;
        return ok;
      };
      auto full = [&](int place) { return need(waitOr(smemAddr(&fullBar[place % kStages]), (place / kStages) & 1, abortFlag), 2000 + place % kStages); };
      auto tileAt = [&](int place) { return smem0 + Shape::kRing + (place % kStages) * kTileBytes; };
      auto scores = [&](int t, int tile) {   // S of group t
        const int at = placeOfK<PAIRS>(tile);
        if (!full(at)) return;
        tcFenceAfter();
        productOfTiles<T, DP>(tmem + t * 128, descAlong(smem0 + (PAIRS ? t : 0) * kTileBytes), descAlong(tileAt(at)));
        ummaCommit(smemAddr(&scoreBar[t]));
        if (!PAIRS) ummaCommit(smemAddr(&emptyBar[at % kStages]));
      };
      for (int t = 0; t < 2 && ok; ++t) {
        if (!count[t]) continue;
        if ((PAIRS || t == 0) && !need(waitOr(smemAddr(&qBar[t]), 0, abortFlag), 2100)) break;
        scores(t, PAIRS ? 0 : t);
      }
      if (PAIRS && ok) ummaCommit(smemAddr(&emptyBar[0]));
      for (int i = 0; i < (PAIRS ? n : count[0]) && ok; ++i) {
        for (int t = 0; t < 2 && ok; ++t) {
          if (i >= count[t]) continue;
          const int tile = PAIRS ? i : 2 * i + t, at = placeOfV<PAIRS>(tile, n);
          if (!full(at)) break;
          if (tile == fixTile && !need(waitOr(smemAddr(fixBar), 0, abortFlag), 2200)) break;
          if (!need(waitOr(smemAddr(&probBar[t]), i & 1, abortFlag), 2300 + t)) break;
          tcFenceAfter();
          productWithTmem<T, DP>(tmem + 256 + t * 128, tmem + t * 128, descAcross(tileAt(at)), i != 0);
          if (!PAIRS) ummaCommit(smemAddr(&emptyBar[at % kStages]));
          if (i + 1 == count[t]) ummaCommit(smemAddr(&outBar[t]));
          else scores(t, PAIRS ? i + 1 : tile + 2);   // over the probabilities: products are carried out in order
        }
        if (PAIRS && ok) {
          ummaCommit(smemAddr(&emptyBar[placeOfV<true>(i, n) % kStages]));
          if (i + 1 < n) ummaCommit(smemAddr(&emptyBar[placeOfK<true>(i + 1) % kStages]));
        }
      }
      if (!ok) {   // products in flight still read shared memory and write tensor memory
        ummaCommit(smemAddr(drainBar));
        mbarWait(smemAddr(drainBar), 0, 1u << 20);
      }
    }
  } else if (warp < W::kCompute) {
    regsTake<W::kManyRegs>();
    const int t = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tS = tmem + lanes + t * 128, tO = tmem + lanes + 256 + t * 128;
    const int rows = a.tileTokens * a.group;
    const bool working = quarter * 32 < rows;   // a warp without rows only keeps step
    const int tok = tok0[t] + row / a.group, head = kvHead * a.group + row % a.group;
    const bool valid = row < rows && tok < seq.q, exists = row < rows && tok < a.q;
    const int limit = valid ? visibleOf(a, seq, tok) : 0x7fffffff;   // (rows that nobody stores are not masked)
    const float c = a.scale * kLog2e;
    const uint64_t c2 = pair(c, c);
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int i = 0; i < count[t]; ++i) {
      ok = warpWaitOr(smemAddr(&scoreBar[t]), i & 1, abortFlag);
      if (!ok) {
        if (lane == 0) fail(3000 + t);
        break;
      }
      tcFenceAfter();
      if (working) {
        softmaxTile<T, DP>(tS, tO, i > 0, limit, (begin + (PAIRS ? i : 2 * i + t)) * 128, c, c2, m, l, smemAddr(&probBar[t]), lane);
      } else {
        tcFenceBefore();
        __syncwarp();
        if (lane == 0) mbarArrive(smemAddr(&probBar[t]));
      }
    }
    if (ok && count[t]) {
      ok = warpWaitOr(smemAddr(&outBar[t]), 0, abortFlag);
      if (ok && !PAIRS && t == 0 && count[1]) ok = warpWaitOr(smemAddr(&outBar[1]), 0, abortFlag);
      if (!ok && lane == 0) fail(3100 + t);
      tcFenceAfter();
    }
    float* const ml = (float*)(smem + Shape::kExchange) + row;
    if (!PAIRS) {
      // both groups have the same rows, and the first one stores them: it can read the second's sums, not what they are to be multiplied by
      if (t == 1 && count[1] && ok) {
        ml[0] = m;
        ml[128] = l;
      }
      ok = allWell<W::kCompute * 32>(1, ok);
    }
    if ((PAIRS || t == 0) && ok && working) {
      float weight = 1.0f, theirs = 0.0f;   // of this group's sums, and of the second's
      if (!PAIRS && count[1]) {
        const float m1 = ml[0], to = fmaxf(m, m1);
        weight = m == to ? 1.0f : exp2Fast((m - to) * c);
        theirs = m1 == to ? 1.0f : exp2Fast((m1 - to) * c);
        l = l * weight + ml[128] * theirs;
        m = to;
      }
      const bool empty = !valid || l == 0.0f;
      const float inv = empty ? 0.0f : 1.0f / l;
      const size_t at = ((size_t)b * a.q + tok) * a.heads + head;   // row of out
      const size_t atLse = ((size_t)b * a.heads + head) * a.q + tok;
      const float lse = empty ? -INFINITY : fmaf(m, a.scale, logf(l) - Pack<T>::kForwardBias * kLn2);
      float share, joined;
      const float* from;
      closeRow(a, lse, inv, at, atLse, part, valid, exists, share, joined, from);
#pragma unroll
      for (int k = 0; k < DP / 32; ++k) {
        uint32_t o[32], u[32];
        float f[32];
        if (count[t]) {
          tmemLd32(tO + k * 32, o);
          if (!PAIRS && count[1]) {
            tmemLd32(tO + 128 + k * 32, u);
            tmemLdWait32(u);
          }
          tmemLdWait32(o);
        }
        if (!exists) continue;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          f[e] = count[t] ? __uint_as_float(o[e]) * weight : 0.0f;
          if (!PAIRS && count[1]) f[e] += __uint_as_float(u[e]) * theirs;
          f[e] = empty || !count[t] ? 0.0f : f[e] * share;
        }
        storeChannels<T>(a, f, k * 32, at, part, from, joined);
      }
    }
  }

  // ---- teardown
  tcFenceBefore();
  __syncthreads();
  if (warp == W::kMma) {
    tcFenceAfter();
    tmemDealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------- few rows
// The form for calls with at most 32 rows to a key head (a token of a decoder: the heads that share it): a warp has all rows, and the tensor memory, registers and shared memory of a CTA are such
// that two are on an SM. There a CTA works on few keys, and what it waits for at its beginning (lengths, the first copies) and at its end is as long as the work: the other CTA
// fills it. Of one tile a CTA takes 10000 to 13000 cycles: 500 to set up, 1400 for the lengths, 2400 for the first scores, 2700 for softmax, 800 for the product, 2000 for the
// result. The single form, one CTA to an SM, took 92 us for 128 queries on up to 1024 keys each (46 by their bytes), this one 68.
struct FewWarps {
  static constexpr int kCompute = 0, kProducer = 1, kMma = 2, kThreads = 96;
};
template <int DP> struct FewShape {
  static constexpr uint32_t kQHalf = kFewRows * 128;                   // queries: 32 rows of 64 channels; the product reads 128, of which the others are whatever follows
  static constexpr uint32_t kTileBytes = DP / 64 * kHalfTile;
  static constexpr int kStages = DP == 64 ? 6 : 3;
  static constexpr uint32_t kRing = DP / 64 * kQHalf, kCtrl = kRing + kStages * kTileBytes;
  static_assert((2 * kStages + 6) * 8 + 8 <= 512, "control block");
  static constexpr size_t kBytes = kCtrl + 512;
  static_assert(2 * (kBytes + 1024) <= 228 * 1024 && 3 * (kBytes + 1024) > 228 * 1024, "two on an SM, as in tensor memory");
};

template <typename T, int DP>
__global__ void __launch_bounds__(FewWarps::kThreads, 2)
attnFewKernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ AttnArgs a) {
  using Shape = FewShape<DP>;
  using W = FewWarps;
  constexpr int kStages = Shape::kStages;
  constexpr uint32_t kTileBytes = Shape::kTileBytes, kSums = 128;   // tensor memory: scores (then probabilities) at 0, sums behind them
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* fullBar = (uint64_t*)(smem + Shape::kCtrl);   // [kStages]
  uint64_t* emptyBar = fullBar + kStages;                 // [kStages]
  uint64_t* qBar = emptyBar + kStages;
  uint64_t* scoreBar = qBar + 1;                          // scores are there
  uint64_t* probBar = scoreBar + 1;                       // probabilities are
  uint64_t* outBar = probBar + 1;                         // sums are complete
  uint64_t* fixBar = outBar + 1;                          // the last values have zeros behind them
  uint64_t* drainBar = fixBar + 1;
  uint32_t* tmemSlot = (uint32_t*)(drainBar + 1);
  volatile uint32_t* abortFlag = tmemSlot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbarInit(smemAddr(&fullBar[s]), 1); mbarInit(smemAddr(&emptyBar[s]), 1); }
    for (uint64_t* bar : {qBar, scoreBar, probBar, outBar, fixBar, drainBar}) mbarInit(smemAddr(bar), 1);
    *abortFlag = 0;
    mbarInitFence();
    prefetchTensorMap(&tmQ);
    prefetchTensorMap(&tmK);
    prefetchTensorMap(&tmV);
  }
  if (warp == W::kMma) {
    tmemAlloc(smemAddr(tmemSlot), 256);
    tmemRelinquish();
  }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmem = *tmemSlot;
  pdlEnter();   // the set-up above overlaps the end of the kernel before

  const unsigned owners = a.batch * a.kvHeads, owner = blockIdx.x % owners;
  const int kvHead = owner % a.kvHeads, b = owner / a.kvHeads, part = blockIdx.x / owners;
  const Sequence seq = sequenceOf(a, b);
  const int all = seq.q ? (visibleOf(a, seq, seq.q - 1) + 127) / 128 : 0, each = (all + a.splits - 1) / a.splits;
  const int begin = min(all, part * each), n = min(all, begin + each) - begin;   // tiles of keys: the first of this part, how many
  // values behind the sequence's last: the tensor map gives zeros behind the tensor's last
  const int fixTile = seq.kv < a.kv && seq.kv % 128 ? seq.kv / 128 - begin : -1;
  const uint32_t smem0 = smemAddr(smem);
  auto fail = [&](uint32_t what) {
    *abortFlag = 1;
    reportTimeout(a.status, what);
  };
  auto tileAt = [&](int place) { return smem0 + Shape::kRing + place % kStages * kTileBytes; };   // K0 V0 K1 V1 ...

  if (warp == W::kProducer) {
    int place = 0;
    bool ok = true;
    auto next = [&](const CUtensorMap* map, int tile) {
      const int s = place % kStages;
      ok = ok && warpWaitOr(smemAddr(&emptyBar[s]), ((place / kStages) & 1) ^ 1, abortFlag);
      if (!ok) {
        if (lane == 0) fail(1000 + s);
        return;
      }
      if (lane == 0) {
        const uint32_t bar = smemAddr(&fullBar[s]);
        mbarExpectTx(bar, kTileBytes);
        loadTile<DP>(tileAt(place), map, (begin + tile) * 128, kvHead, b, bar);
      }
      ++place;
    };
    if (n > 0) {
      if (lane == 0) {
        mbarExpectTx(smemAddr(qBar), DP / 64 * a.tileTokens * a.group * 128);
#pragma unroll
        for (int h = 0; h < DP / 64; ++h) tmaLoad4d(smem0 + h * Shape::kQHalf, &tmQ, h * 64, kvHead * a.group, 0, b, smemAddr(qBar));
      }
      for (int i = 0; i < n && ok; ++i) {
        next(&tmK, i);
        if (ok) next(&tmV, i);
      }
      if (ok && fixTile >= 0 && fixTile < n) {
        const int at = 2 * fixTile + 1, s = at % kStages;   // the last tile: its stage is not used again
        ok = warpWaitOr(smemAddr(&fullBar[s]), (at / kStages) & 1, abortFlag);
        if (ok) {
          clearRows<DP>(smem + Shape::kRing + s * kTileBytes, seq.kv % 128, lane);
          if (lane == 0) mbarArrive(smemAddr(fixBar));
        } else if (lane == 0) {
          fail(1100);
        }
      }
      if (__any_sync(~0u, *abortFlag)) {
        // copies already issued still write into this CTA's shared memory: wait for them (bounded)
        for (int at = max(0, place - kStages); at < place; ++at) mbarWait(smemAddr(&fullBar[at % kStages]), (at / kStages) & 1, 1u << 20);
        mbarWait(smemAddr(qBar), 0, 1u << 20);
      }
    }
  } else if (warp == W::kMma) {
    if (n > 0 && electOne()) {
      bool ok = true;
      auto need = [&](bool got, uint32_t what) {
        if (ok && !got) fail(what);
        ok = ok && got;
        return ok;
      };
      auto full = [&](int place) { return need(waitOr(smemAddr(&fullBar[place % kStages]), (place / kStages) & 1, abortFlag), 2000 + place % kStages); };
      auto scores = [&](int i) {
        if (!full(2 * i)) return;
        tcFenceAfter();
        productOfTiles<T, DP, 128, Shape::kQHalf>(tmem, descAlong(smem0), descAlong(tileAt(2 * i)));
        ummaCommit(smemAddr(scoreBar));
        ummaCommit(smemAddr(&emptyBar[2 * i % kStages]));
      };
      if (need(waitOr(smemAddr(qBar), 0, abortFlag), 2100)) scores(0);
      for (int i = 0; i < n && ok; ++i) {
        if (!full(2 * i + 1)) break;
        if (i == fixTile && !need(waitOr(smemAddr(fixBar), 0, abortFlag), 2200)) break;
        if (!need(waitOr(smemAddr(probBar), i & 1, abortFlag), 2300)) break;
        tcFenceAfter();
        productWithTmem<T, DP>(tmem + kSums, tmem, descAcross(tileAt(2 * i + 1)), i != 0);
        ummaCommit(smemAddr(&emptyBar[(2 * i + 1) % kStages]));
        if (i + 1 == n) ummaCommit(smemAddr(outBar));
        else scores(i + 1);   // over the probabilities: products are carried out in order
      }
      if (!ok) {   // products in flight still read shared memory and write tensor memory
        ummaCommit(smemAddr(drainBar));
        mbarWait(smemAddr(drainBar), 0, 1u << 20);
      }
    }
  } else {
    const int tok = lane / a.group, head = kvHead * a.group + lane % a.group;
    const bool exists = tok < a.q, valid = tok < seq.q;   // (one tile: rows behind its last are tokens behind the last)
    const int limit = valid ? visibleOf(a, seq, tok) : 0x7fffffff;   // (rows that nobody stores are not masked)
    const float c = a.scale * kLog2e;
    const uint64_t c2 = pair(c, c);
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      ok = warpWaitOr(smemAddr(scoreBar), i & 1, abortFlag);
      if (!ok) break;
      tcFenceAfter();
      softmaxTile<T, DP>(tmem, tmem + kSums, i > 0, limit, (begin + i) * 128, c, c2, m, l, smemAddr(probBar), lane);
    }
    if (n > 0 && ok) ok = warpWaitOr(smemAddr(outBar), 0, abortFlag);
    if (!ok && lane == 0) fail(3000);
    tcFenceAfter();
    if (ok) {
      const bool empty = !valid || l == 0.0f;
      const float inv = empty ? 0.0f : 1.0f / l;
      const size_t at = ((size_t)b * a.q + tok) * a.heads + head, atLse = ((size_t)b * a.heads + head) * a.q + tok;
      const float lse = empty ? -INFINITY : fmaf(m, a.scale, logf(l) - Pack<T>::kForwardBias * kLn2);
      float share, joined;
      const float* from;
      closeRow(a, lse, inv, at, atLse, part, valid, exists, share, joined, from);
#pragma unroll
      for (int k = 0; k < DP / 32; ++k) {
        uint32_t o[32];
        float f[32];
        if (n > 0) {
          tmemLd32(tmem + kSums + k * 32, o);
          tmemLdWait32(o);
        }
        if (!exists) continue;
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = empty || n <= 0 ? 0.0f : __uint_as_float(o[e]) * share;
        storeChannels<T>(a, f, k * 32, at, part, from, joined);
      }
    }
  }

  // ---- teardown
  tcFenceBefore();
  __syncthreads();
  if (warp == W::kMma) {
    tcFenceAfter();
    tmemDealloc(tmem, 256);
  }
}

// Joins the parts of the keys: out = sum_s exp(lse_s - L) out_s with L = ln sum_s exp(lse_s); what `join` names is one more part. quads * a.joinShares threads take a row: four
// channels of every joinShares-th part each, all of them on their way at once, and the first of those with the same channels joins the others'. Its time is that of a launch and a
// load: 16 parts of 32 rows 3.3 us (a thread for four channels that walked the parts one after the other took 8.6).
constexpr int kJoinTurns = kAttnJoinTurns;
static_assert(kAttnMaxSplits <= kJoinTurns * (256 / (kAttnMaxDim / 4)), "parts of a thread");   // (256 / ... is a power of two)
template <typename T>
__global__ void __launch_bounds__(256) attnJoinKernel(const __grid_constant__ AttnArgs a) {
  __shared__ float4 sums[256];
  __shared__ float2 heads[256];   // maximum and sum of the weights
  const int quads = a.dim / 4, each = quads * a.joinShares, perCta = 256 / each;
  const int slot = threadIdx.x / each, share = threadIdx.x % each / quads, d = threadIdx.x % quads * 4;
  const size_t rows = (size_t)a.batch * a.q * a.heads, row = (size_t)blockIdx.x * perCta + slot;
  const bool some = slot < perCta && row < rows;
  pdlEnter();
  float lse[kJoinTurns], top = -INFINITY, total = 0.0f;
  float4 v[kJoinTurns], f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < kJoinTurns; ++i) {
    const int s = share + i * a.joinShares;
    const bool mine = some && s < a.splits;
    lse[i] = mine ? a.partLse[s * rows + row] : -INFINITY;
    v[i] = mine ? *(const float4*)(a.partOut + (s * rows + row) * a.dim + d) : f;   // (zeros in a part that saw no key)
  }
  const int head = (int)(row % a.heads);
  const size_t token = row / a.heads;   // of the batch
  const int b = (int)(token / a.q), tok = (int)(token % a.q);
  const size_t atLse = ((size_t)b * a.heads + head) * a.q + tok;
  const bool join = some && share == 0 && a.joinOut && tok < (a.qLengths ? a.qLengths[b] : a.q);
  const float otherLse = join ? a.joinLse[atLse] : -INFINITY;
  const float4 other = join ? *(const float4*)(a.joinOut + row * a.dim + d) : f;
  // joins (to, sum, x) to what this thread has
  auto add = [&](float to, float weight, float4 x) {
    if (to == -INFINITY) return;
    const float m = fmaxf(top, to), old = expf(top - m), now = expf(to - m);
    total = total * old + weight * now;
    f.x = f.x * old + x.x * now; f.y = f.y * old + x.y * now; f.z = f.z * old + x.z * now; f.w = f.w * old + x.w * now;
    top = m;
  };
#pragma unroll
  for (int i = 0; i < kJoinTurns; ++i) top = fmaxf(top, lse[i]);
  const float shift = top == -INFINITY ? 0.0f : top;
#pragma unroll
  for (int i = 0; i < kJoinTurns; ++i) {
    const float weight = expf(lse[i] - shift);
    total += weight;
    f.x += v[i].x * weight; f.y += v[i].y * weight; f.z += v[i].z * weight; f.w += v[i].w * weight;
  }
  if (share) {
    sums[threadIdx.x] = f;
    heads[threadIdx.x] = make_float2(top, total);
  }
  __syncthreads();
  if (share || !some) return;
  for (int i = 1; i < a.joinShares; ++i) add(heads[threadIdx.x + i * quads].x, heads[threadIdx.x + i * quads].y, sums[threadIdx.x + i * quads]);
  add(otherLse, 1.0f, other);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  f.x *= inv; f.y *= inv; f.z *= inv; f.w *= inv;
  if (d == 0) a.lse[atLse] = total == 0.0f ? -INFINITY : top + logf(total);
  if (a.outFp32) *(float4*)((float*)a.out + row * a.dim + d) = f;
  else *(uint2*)((uint16_t*)a.out + row * a.dim + d) = make_uint2(Pack<T>::two(f.x, f.y), Pack<T>::two(f.z, f.w));
}

}  // namespace

template <typename T> static const void* forwardFn(int dim, AttnForm form) {
  if (form == ATTN_FEW) return dim <= 64 ? (const void*)attnFewKernel<T, 64> : (const void*)attnFewKernel<T, 128>;
  const bool pairs = form == ATTN_PAIRS;
  if (dim <= 64) return pairs ? (const void*)attnForwardKernel<T, 64, true> : (const void*)attnForwardKernel<T, 64, false>;
  return pairs ? (const void*)attnForwardKernel<T, 128, true> : (const void*)attnForwardKernel<T, 128, false>;
}
const void* attnForwardKernelFn(int type, int dim, AttnForm form) { return type == ATTN_F16 ? forwardFn<__half>(dim, form) : forwardFn<__nv_bfloat16>(dim, form); }
size_t attnForwardSmemBytes(int dim, AttnForm form) {
  if (form == ATTN_FEW) return dim <= 64 ? FewShape<64>::kBytes : FewShape<128>::kBytes;
  const bool pairs = form == ATTN_PAIRS;
  if (dim <= 64) return pairs ? ForwardShape<64, true>::kBytes : ForwardShape<64, false>::kBytes;
  return pairs ? ForwardShape<128, true>::kBytes : ForwardShape<128, false>::kBytes;
}
const void* attnJoinKernelFn(int type) { return type == ATTN_F16 ? (const void*)attnJoinKernel<__half> : (const void*)attnJoinKernel<__nv_bfloat16>; }
int attnForwardThreads(AttnForm form) { return form == ATTN_FEW ? FewWarps::kThreads : ForwardWarps::kThreads; }
int attnForwardRegs(AttnForm form) { return form == ATTN_FEW ? 1 : ForwardWarps::kLaunchRegs; }

}  // namespace b200
