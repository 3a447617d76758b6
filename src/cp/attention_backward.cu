// Attention for sm_100a, the backward pass, which computes the probabilities again: with p_ij = exp(s_ij - lse_i), s_ij = scale q_i.k_j,
//   dv_j = sum_i p_ij do_i      ds_ij = p_ij (do_i.v_j - <do_i, o_i>)      dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i
// over the pairs that see each other; the sums for dk and dv run over the heads that share them as well.
//
// Where tiles are few, several CTAs share one's partners, and another kernel adds up what they have, part by part.
//
// Two kinds of CTAs in one launch, each with the sums of its tile in tensor memory from the first product to the last: one owns a tile of keys and walks the queries (dk, dv),
// the other owns a tile of queries and walks the keys (dq). Together they make seven products of a tile where five would do, if the tiles of dq were added up
// in memory by whoever has a part of them: then the order of the additions, and the result, would change from run to run, or CTAs would have to wait for one another.
//
// Roles as in the forward pass: warps 0-7 have a row of the tile each and, in two groups, a half of its columns; warp 8 feeds the ring, warp 9 issues products. Probabilities
// and ds go back into tensor memory in 16 bits, each over the half it was computed from, and are the first operand of the next products from there.
// "Fine" products, for calls that they cost little: what the rounding of probabilities and ds to 16 bits left is multiplied too. It lies over the scores, whose next tile then waits.
//
// What bounds it: products and elements of a tile alternate in part; a tile takes about 2900 cycles (keys) and 2450 (queries), of which the tensor cores work 2048 and 1536 at 128 channels. 8192 causal tokens of
// 32 heads over 8 take 1372 us after a rest and 1546 to 1631 pass after pass, 4096 383 under a profiler, tensor cores busy 69 % of it; five products of what is seen would be 837 and 209.
//
// fp16: probabilities are held times 2^15, ds times a power of two that brings the largest that it could be (by the longest rows of do and v, and the largest delta) to 2^15; the sums
// are in fp32 and are multiplied back.
#include "attention.cuh"

namespace b200 {

using namespace attn;

namespace {

constexpr uint32_t kTmemCols = 512;

template <int DP> struct BackwardShape {
  static constexpr uint32_t kTileBytes = DP / 64 * kHalfTile;
  static constexpr int kStages = DP == 64 ? 8 : 5;
  static constexpr uint32_t kRing = 2 * kTileBytes, kStats = kRing + kStages * kTileBytes, kCtrl = kStats + 2048;
  static constexpr size_t kBytes = kCtrl + 1024;   // (dynamic shared memory, all that these kernels have, begins on a multiple of 1024 bytes)
  static_assert(kBytes <= 227 * 1024 && (2 * kStages + 13) * 8 + 8 <= 1024, "shared memory");
};

// The power of two that ds is multiplied by, in fp16: |ds| <= p (|do.v| + |delta|) <= |do| |v| + |delta|, by the longest rows and the largest delta of all tiles. delta is not bounded by
// |do| |v|: o is a mean of values of all of a row's keys, of which a call may have a block, and a gradient of the log-sum-exp may be in it. (The bits of floats that are not negative
// are ordered as they are, NaN on top.)
template <typename T>
__device__ __forceinline__ float gradScale(const AttnArgs& a, int b, int kvHead) {
  if (Pack<T>::kBackwardBias == 0.0f) return 1.0f;
  const uint32_t* at = a.bounds + ((size_t)b * a.kvHeads + kvHead) * (2 * a.tiles + a.vTiles);
  uint32_t largest[3] = {0, 0, 0};   // |do|^2, |delta|, |v|^2
#pragma unroll 4
  for (int i = threadIdx.x & 31; i < a.tiles; i += 32) {
    largest[0] = max(largest[0], at[2 * i]);
    largest[1] = max(largest[1], at[2 * i + 1]);
  }
#pragma unroll 4
  for (int i = threadIdx.x & 31; i < a.vTiles; i += 32) largest[2] = max(largest[2], at[2 * a.tiles + i]);
#pragma unroll
  for (uint32_t& x : largest) x = __reduce_max_sync(~0u, x);
  const float most = fmaf(sqrtf(__uint_as_float(largest[0])), sqrtf(__uint_as_float(largest[2])), __uint_as_float(largest[1]));
  if (!(most > 0.0f) || most > 3.0e38f) return 1.0f;   // nothing to do, or nothing to save
  int e;
  frexpf(most, &e);                                     // most < 2^e
  return exp2f((float)max(-113, min(100, 15 - e)));
}

struct BackwardBars {
  uint64_t *full, *empty, *own, *first, *second, *firstDone, *secondDone, *outBar, *probDone, *fix, *drain;
  uint32_t* tmemSlot;
  volatile uint32_t* abortFlag;
};

template <int DP>
__device__ __forceinline__ BackwardBars backwardSetUp(uint8_t* smem, int warp) {
  BackwardBars s;
  s.full = (uint64_t*)(smem + BackwardShape<DP>::kCtrl);
  s.empty = s.full + BackwardShape<DP>::kStages;
  s.own = s.empty + BackwardShape<DP>::kStages;
  s.first = s.own + 1;           // scores are there
  s.second = s.first + 1;        // [2] do.v is, in each of its places
  s.firstDone = s.second + 2;    // scores are used up
  s.secondDone = s.firstDone + 1;   // [2] ds is in tensor memory, in each of its places
  s.outBar = s.secondDone + 2;
  s.probDone = s.outBar + 1;     // probabilities are in tensor memory
  s.fix = s.probDone + 1;        // [2]
  s.drain = s.fix + 2;
  s.tmemSlot = (uint32_t*)(s.drain + 1);
  s.abortFlag = s.tmemSlot + 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * BackwardShape<DP>::kStages; ++i) mbarInit(smemAddr(&s.full[i]), 1);
    mbarInit(smemAddr(s.own), 1);
    mbarInit(smemAddr(s.first), 1);
    mbarInit(smemAddr(s.firstDone), BackwardWarps::kCompute);
    for (int i = 0; i < 2; ++i) {
      mbarInit(smemAddr(&s.second[i]), 1);
      mbarInit(smemAddr(&s.secondDone[i]), BackwardWarps::kCompute);
    }
    mbarInit(smemAddr(s.outBar), 1);
    mbarInit(smemAddr(s.probDone), BackwardWarps::kCompute);
    mbarInit(smemAddr(&s.fix[0]), 1);
    mbarInit(smemAddr(&s.fix[1]), 1);
    mbarInit(smemAddr(s.drain), 1);
    *s.abortFlag = 0;
    mbarInitFence();
  }
  if (warp == BackwardWarps::kMma) {
    tmemAlloc(smemAddr(s.tmemSlot), kTmemCols);
    tmemRelinquish();
  }
  return s;
}

// Rows of sums [128][DP] in tensor memory, times `factor` (and plus what is there already), become a gradient's rows.
template <typename T, int DP>
__device__ __forceinline__ void storeGradient(const AttnArgs& a, uint32_t tmem, bool some, float factor, bool exists, bool valid, size_t row, void* grad, bool fp32, const float* add) {
#pragma unroll
  for (int k = 0; k < DP / 32; ++k) {
    uint32_t o[32];
    float f[32];
    if (some) {
      tmemLd32(tmem + k * 32, o);
      tmemLdWait32(o);
    }
    if (!exists) continue;
#pragma unroll
    for (int e = 0; e < 32; ++e) f[e] = some && valid ? __uint_as_float(o[e]) * factor : 0.0f;
    if (add && valid) {
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        if (k * 32 + e >= a.dim) break;
        const float4 v = *(const float4*)(add + row * a.dim + k * 32 + e);
        f[e] += v.x; f[e + 1] += v.y; f[e + 2] += v.z; f[e + 3] += v.w;
      }
    }
    if (fp32) {
      float* to = (float*)grad + row * a.dim;
#pragma unroll
      for (int e = 0; e < 32; e += 4)
        if (k * 32 + e < a.dim) *(float4*)(to + k * 32 + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    } else {
      uint16_t* to = (uint16_t*)grad + row * a.dim;
#pragma unroll
      for (int e = 0; e < 32; e += 8)
        if (k * 32 + e < a.dim)
          *(uint4*)(to + k * 32 + e) = make_uint4(Pack<T>::two(f[e], f[e + 1]), Pack<T>::two(f[e + 2], f[e + 3]), Pack<T>::two(f[e + 4], f[e + 5]), Pack<T>::two(f[e + 6], f[e + 7]));
    }
  }
}

// ---------------------------------------------------------------------------------------------- dk and dv
// Tensor memory: scores [keys x queries] at 0, do.v at 128 (then, over the half of a warp's columns, probabilities and ds), dv at 256, dk at 384. Scores are taken into registers
// at once, and the next tile's are made meanwhile: its exponentials are computed while the tensor cores add this tile's to dv and dk and make the next do.v. With the
// probabilities over the scores, the next scores waited for their product: a third of the tensor cores' time.
template <typename T, int DP, bool FINE>
__device__ __forceinline__ void backwardKv(const CUtensorMap& tmQ, const CUtensorMap& tmDo, const CUtensorMap& tmK, const CUtensorMap& tmV, const AttnArgs& a, uint8_t* smem,
                                           const BackwardBars& s, uint32_t tmem, unsigned block) {
  using Shape = BackwardShape<DP>;
  // Queries stay until their product with ds, two steps behind their scores; do for one step less: a ring for each.
  constexpr int kStages = Shape::kStages, kQStages = (kStages + 1) / 2, kDoStages = kStages - kQStages;
  constexpr uint32_t kTileBytes = Shape::kTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = a.tileTokens * a.group;
  volatile uint32_t* abortFlag = s.abortFlag;
  const unsigned owners = a.batch * a.kvHeads, owner = block % owners, share = block / owners;
  const int kvHead = owner % a.kvHeads, b = owner / a.kvHeads, key0 = share / a.kvParts * 128, part = share % a.kvParts;   // (the first keys are seen most)
  const Sequence seq = sequenceOf(a, b);
  // tiles of queries: from the first that sees a key of this tile to the last, or this part of them
  const int all = (seq.q + a.tileTokens - 1) / a.tileTokens;
  const long long firstTok = a.causal ? max(0ll, (long long)key0 - seq.offset) : 0;
  const int first = (int)min((long long)all, firstTok / a.tileTokens), partners = key0 < seq.kv ? all - first : 0, each = (partners + a.kvParts - 1) / a.kvParts;
  const int begin = first + min(partners, part * each), n = min(partners, (part + 1) * each) - min(partners, part * each);
  const int fixRows = seq.q < a.q && begin + n == all ? seq.q % a.tileTokens * a.group : 0;   // of the last tile, behind which rows may hold anything
  const uint32_t smem0 = smemAddr(smem);
  auto fail = [&](uint32_t what) {
    *abortFlag = 1;
    reportTimeout(a.status, what);
  };

  auto stageOf = [](int isDo, int tile) { return isDo ? kQStages + tile % kDoStages : tile % kQStages; };
  auto phaseOf = [](int isDo, int tile) { return (uint32_t)(tile / (isDo ? kDoStages : kQStages)) & 1; };

  if (warp >= BackwardWarps::kCompute) regsGive<BackwardWarps::kFewRegs>();
  if (warp == BackwardWarps::kProducer) {
    int loaded[2] = {};   // queries, do
    bool ok = !*abortFlag, ownArmed = false;
    auto next = [&](const CUtensorMap* map, int isDo, const float* stats) {
      const int tile = loaded[isDo], at = stageOf(isDo, tile);
      ok = ok && warpWaitOr(smemAddr(&s.empty[at]), phaseOf(isDo, tile) ^ 1, abortFlag);
      if (!ok) {
        if (lane == 0) fail(1000 + at);
        return;
      }
      if (lane == 0) {
        const uint32_t bar = smemAddr(&s.full[at]);
        mbarExpectTx(bar, DP / 64 * rows * 128 + (stats ? 1024 : 0));
        loadTile<DP>(smem0 + Shape::kRing + at * kTileBytes, map, (begin + tile) * a.tileTokens, kvHead * a.group, b, bar);
        if (stats) bulkLoad(smem0 + Shape::kStats + (tile & 1) * 1024, stats, 1024, bar);
      }
      ++loaded[isDo];
    };
    if (n > 0) {
      if (ok && lane == 0) {
        mbarExpectTx(smemAddr(s.own), 2 * kTileBytes);
        loadTile<DP>(smem0, &tmK, key0, kvHead, b, smemAddr(s.own));
        loadTile<DP>(smem0 + kTileBytes, &tmV, key0, kvHead, b, smemAddr(s.own));
      }
      ownArmed = ok;
      // A tile's numbers per row arrive with its do. The buffer was last read for the tile before the last, whose do has left the ring by then if the ring has room for two; else
      // its stage is waited for.
      const float* stats = a.stats + (((size_t)b * a.kvHeads + kvHead) * a.tiles + begin) * 256;
      for (int i = 0; i < n && ok; ++i) {
        next(&tmQ, 0, nullptr);
        if (ok && kDoStages > 2 && i >= 2) {
          ok = warpWaitOr(smemAddr(&s.empty[stageOf(1, i - 2)]), phaseOf(1, i - 2), abortFlag);
          if (!ok && lane == 0) fail(1050);
        }
        if (ok) next(&tmDo, 1, stats + (size_t)i * 256);
      }
      if (ok && fixRows) {
        for (int k = 0; k < 2 && ok; ++k) {
          const int at = stageOf(k, n - 1);
          ok = warpWaitOr(smemAddr(&s.full[at]), phaseOf(k, n - 1), abortFlag);
          if (ok) {
            clearRows<DP>(smem + Shape::kRing + at * kTileBytes, fixRows, lane);
            if (lane == 0) mbarArrive(smemAddr(&s.fix[k]));
          } else if (lane == 0) {
            fail(1100);
          }
        }
      }
      if (__any_sync(~0u, *abortFlag)) {
        // copies already issued still write into this CTA's shared memory: wait for them (bounded)
        for (int isDo = 0; isDo < 2; ++isDo)
          for (int tile = max(0, loaded[isDo] - (isDo ? kDoStages : kQStages)); tile < loaded[isDo]; ++tile)
            mbarWait(smemAddr(&s.full[stageOf(isDo, tile)]), phaseOf(isDo, tile), 1u << 20);
        if (ownArmed) mbarWait(smemAddr(s.own), 0, 1u << 20);
      }
    }
  } else if (warp == BackwardWarps::kMma) {
    if (n > 0 && electOne()) {
      bool ok = true;
      auto need = [&](bool got, uint32_t what) {
        if (ok && !got) fail(what);
        ok = ok && got;
        return ok;
      };
      auto full = [&](int isDo, int tile) { return need(waitOr(smemAddr(&s.full[stageOf(isDo, tile)]), phaseOf(isDo, tile), abortFlag), 2000 + stageOf(isDo, tile)); };
      auto tileAt = [&](int isDo, int tile) { return smem0 + Shape::kRing + stageOf(isDo, tile) * kTileBytes; };
      auto scores = [&](int i) {
        if (!full(0, i)) return;
        if (fixRows && i == n - 1 && !need(waitOr(smemAddr(&s.fix[0]), 0, abortFlag), 2200)) return;
        tcFenceAfter();
        productOfTiles<T, DP>(tmem, descAlong(smem0), descAlong(tileAt(0, i)));
        ummaCommit(smemAddr(s.first));
      };
      auto doV = [&](int i) {
        if (!full(1, i)) return;
        if (fixRows && i == n - 1 && !need(waitOr(smemAddr(&s.fix[1]), 0, abortFlag), 2201)) return;
        tcFenceAfter();
        productOfTiles<T, DP>(tmem + 128, descAlong(smem0 + kTileBytes), descAlong(tileAt(1, i)));
        ummaCommit(smemAddr(s.second));
      };
      if (need(waitOr(smemAddr(s.own), 0, abortFlag), 2100)) scores(0);
      if (ok) doV(0);
      for (int i = 0; i < n && ok; ++i) {
        if (!FINE && i + 1 < n) {
          if (!need(waitOr(smemAddr(s.firstDone), i & 1, abortFlag), 2300)) break;   // scores are in registers
          scores(i + 1);
        }
        if (!ok || !need(waitOr(smemAddr(s.probDone), i & 1, abortFlag), 2400)) break;
        tcFenceAfter();
        productWithTmem<T, DP>(tmem + 256, tmem + 128, descAcross(tileAt(1, i)), i != 0);
        if (FINE) productWithTmem<T, DP>(tmem + 256, tmem, descAcross(tileAt(1, i)), true);
        if (!need(waitOr(smemAddr(s.secondDone), i & 1, abortFlag), 2500)) break;
        tcFenceAfter();
        ummaCommit(smemAddr(&s.empty[stageOf(1, i)]));   // (its do.v was issued in front of this; the row's numbers that came with it are used up)
        productWithTmem<T, DP>(tmem + 384, tmem + 160, descAcross(tileAt(0, i)), i != 0);
        if (FINE) productWithTmem<T, DP>(tmem + 384, tmem + 32, descAcross(tileAt(0, i)), true);
        ummaCommit(smemAddr(&s.empty[stageOf(0, i)]));
        if (FINE && i + 1 < n) scores(i + 1);
        if (!ok) break;
        if (i + 1 < n) doV(i + 1);   // over probabilities and ds: products are carried out in order
        else ummaCommit(smemAddr(s.outBar));
      }
      if (!ok) {
        ummaCommit(smemAddr(s.drain));
        mbarWait(smemAddr(s.drain), 0, 1u << 20);
      }
    }
  } else if (warp < BackwardWarps::kCompute) {
    regsTake<BackwardWarps::kManyRegs>();
    const int half = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane, key = key0 + row;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tS = tmem + lanes + half * 64, tDp = tS + 128;
    const float c = a.scale * kLog2e, up = n > 0 ? gradScale<T>(a, b, kvHead) : 1.0f, down = up * exp2f(-Pack<T>::kBackwardBias);
    const uint64_t c2 = pair(c, c), down2 = pair(down, down);
    const bool valid = key < seq.kv;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const float* stats = (const float*)(smem + Shape::kStats + (i & 1) * 1024);   // of the tile's rows: minus the log-sum-exp [128], minus <do, o> [128]
      ok = warpWaitOr(smemAddr(&s.full[stageOf(1, i)]), phaseOf(1, i), abortFlag) && warpWaitOr(smemAddr(s.first), i & 1, abortFlag);
      if (!ok) {
        if (lane == 0) fail(3000);
        break;
      }
      tcFenceAfter();
      const int tok0 = (begin + i) * a.tileTokens;
      const bool hide = a.causal && tok0 + seq.offset < key0 + 127;
      const int seen = key - seq.offset - tok0;   // the first token of the tile that sees this key
      const int from = !hide || seen <= 0 ? 0 : min(seen, 128) * a.group;
      uint32_t x[2][32], packed[32];
      uint64_t p[32];
      tmemLd32(tS, x[0]);
      tmemLd32(tS + 32, x[1]);
      tmemLdWait32(x[0]);
      tmemLdWait32(x[1]);
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) mbarArrive(smemAddr(s.firstDone));
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 lse = *(const float4*)(stats + half * 64 + q * 32 + k);
          const uint64_t lo = fma2(packF32x2(x[q][k], x[q][k + 1]), c2, pair(lse.x, lse.y)), hi = fma2(packF32x2(x[q][k + 2], x[q][k + 3]), c2, pair(lse.z, lse.w));
          p[q * 16 + k / 2] = pair(exp2Fast(lowOf(lo)), exp2Fast(highOf(lo)));
          p[q * 16 + k / 2 + 1] = pair(exp2Fast(lowOf(hi)), exp2Fast(highOf(hi)));
        }
      }
      if (hide) {
#pragma unroll
        for (int k = 0; k < 32; ++k) p[k] = pair(half * 64 + 2 * k < from ? 0.0f : lowOf(p[k]), half * 64 + 2 * k + 1 < from ? 0.0f : highOf(p[k]));
      }
#pragma unroll
      for (int k = 0; k < 32; ++k) packed[k] = Pack<T>::two(lowOf(p[k]), highOf(p[k]));
      ok = warpWaitOr(smemAddr(s.second), i & 1, abortFlag);
      if (!ok) {
        if (lane == 0) fail(3001);
        break;
      }
      tcFenceAfter();
      tmemLd32(tDp, x[0]);
      tmemLd32(tDp + 32, x[1]);
      tmemLdWait32(x[0]);
      tmemLdWait32(x[1]);
      // what is added to dv does not wait for ds
      tmemSt32(tDp, packed);
      if (FINE) {
#pragma unroll
        for (int k = 0; k < 32; ++k) packed[k] = remainderOf<T>(packed[k], lowOf(p[k]), highOf(p[k]));
        tmemSt32(tS, packed);
      }
      tmemStWait();
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) mbarArrive(smemAddr(s.probDone));
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 delta = *(const float4*)(stats + 128 + half * 64 + q * 32 + k);
          uint64_t lo = add2(packF32x2(x[q][k], x[q][k + 1]), pair(delta.x, delta.y)), hi = add2(packF32x2(x[q][k + 2], x[q][k + 3]), pair(delta.z, delta.w));
          if (Pack<T>::kBackwardBias != 0.0f) {
            lo = mul2(lo, down2);
            hi = mul2(hi, down2);
          }
          lo = mul2(p[q * 16 + k / 2], lo);
          hi = mul2(p[q * 16 + k / 2 + 1], hi);
          packed[q * 16 + k / 2] = Pack<T>::two(lowOf(lo), highOf(lo));
          packed[q * 16 + k / 2 + 1] = Pack<T>::two(lowOf(hi), highOf(hi));
          if (FINE) {
            p[q * 16 + k / 2] = lo;
            p[q * 16 + k / 2 + 1] = hi;
          }
        }
      }
      tmemSt32(tDp + 32, packed);
      if (FINE) {
#pragma unroll
        for (int k = 0; k < 32; ++k) packed[k] = remainderOf<T>(packed[k], lowOf(p[k]), highOf(p[k]));
        tmemSt32(tS + 32, packed);
      }
      tmemStWait();
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) mbarArrive(smemAddr(s.secondDone));
    }
    if (ok && n > 0) {
      ok = warpWaitOr(smemAddr(s.outBar), 0, abortFlag);
      if (!ok && lane == 0) fail(3100);
      tcFenceAfter();
    }
    if (!__any_sync(~0u, *abortFlag)) {
      const bool whole = a.kvParts == 1;
      const size_t at = ((size_t)b * a.kv + key) * a.kvHeads + kvHead, atPart = whole ? at : (size_t)part * a.batch * a.kv * a.kvHeads + at;
      const float factor = half ? a.scale / up : exp2f(-Pack<T>::kBackwardBias);   // of dk, of dv
      storeGradient<T, DP>(a, tmem + lanes + 256 + half * 128, n > 0, factor, key < a.kv, valid, atPart, whole ? (half ? a.dk : a.dv) : (half ? a.partDk : a.partDv), !whole || a.gradFp32,
                           whole ? (half ? a.addDk : a.addDv) : nullptr);
    }
  }
}

// ---------------------------------------------------------------------------------------------- dq
// Tensor memory: scores [queries x keys] at 0, do.v (then ds) of two tiles at 128 and 256, dq at 384. Scores are taken into registers at once, and the next tile's are made
// while exponentials are computed; so is its do.v, in the other place. So products and elements of a tile do not wait for one another.
template <typename T, int DP, bool FINE>
__device__ __forceinline__ void backwardQ(const CUtensorMap& tmQ, const CUtensorMap& tmDo, const CUtensorMap& tmK, const CUtensorMap& tmV, const AttnArgs& a, uint8_t* smem,
                                          const BackwardBars& s, uint32_t tmem, unsigned block) {
  using Shape = BackwardShape<DP>;
  // Keys stay until their product with ds, values only until do.v: a ring for each, so that values come in early (in one ring of five stages the next do.v waited half of the
  // time for values that could not be asked for before the last ds was used).
  constexpr int kStages = Shape::kStages, kKeyStages = (kStages + 1) / 2, kValueStages = kStages - kKeyStages;
  constexpr uint32_t kTileBytes = Shape::kTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = a.tileTokens * a.group;
  volatile uint32_t* abortFlag = s.abortFlag;
  const unsigned owners = a.batch * a.kvHeads, owner = block % owners;
  const int share = block / owners, part = share % a.qParts;
  const int kvHead = owner % a.kvHeads, b = owner / a.kvHeads, qTile = a.tiles - 1 - share / a.qParts, tok0 = qTile * a.tileTokens;
  const Sequence seq = sequenceOf(a, b);
  const int last = min(tok0 + a.tileTokens, seq.q) - 1;
  const int partners = last < tok0 ? 0 : (visibleOf(a, seq, last) + 127) / 128, each = (partners + a.qParts - 1) / a.qParts;
  const int begin = min(partners, part * each), n = min(partners, begin + each) - begin;   // tiles of keys: all that the last query sees, or this part of them
  const int fixRows = seq.kv < a.kv ? seq.kv % 128 : 0, fixTile = fixRows ? seq.kv / 128 - begin : -1;   // keys and values behind the last may be anything
  const uint32_t smem0 = smemAddr(smem);
  auto fail = [&](uint32_t what) {
    *abortFlag = 1;
    reportTimeout(a.status, what);
  };

  auto stageOf = [](int values, int tile) { return values ? kKeyStages + tile % kValueStages : tile % kKeyStages; };
  auto phaseOf = [](int values, int tile) { return (uint32_t)(tile / (values ? kValueStages : kKeyStages)) & 1; };

  if (warp >= BackwardWarps::kCompute) regsGive<BackwardWarps::kFewRegs>();
  if (warp == BackwardWarps::kProducer) {
    int loaded[2] = {};   // keys, values
    bool ok = !*abortFlag, ownArmed = false;
    auto next = [&](const CUtensorMap* map, int values) {
      const int tile = loaded[values], at = stageOf(values, tile);
      ok = ok && warpWaitOr(smemAddr(&s.empty[at]), phaseOf(values, tile) ^ 1, abortFlag);
      if (!ok) {
        if (lane == 0) fail(1000 + at);
        return;
      }
      if (lane == 0) {
        const uint32_t bar = smemAddr(&s.full[at]);
        mbarExpectTx(bar, kTileBytes);
        loadTile<DP>(smem0 + Shape::kRing + at * kTileBytes, map, (begin + tile) * 128, kvHead, b, bar);
      }
      ++loaded[values];
    };
    if (n > 0) {
      if (ok && lane == 0) {
        mbarExpectTx(smemAddr(s.own), 2 * (DP / 64) * rows * 128);
        loadTile<DP>(smem0, &tmQ, tok0, kvHead * a.group, b, smemAddr(s.own));
        loadTile<DP>(smem0 + kTileBytes, &tmDo, tok0, kvHead * a.group, b, smemAddr(s.own));
      }
      ownArmed = ok;
      for (int i = 0; i < n && ok; ++i) {
        next(&tmK, 0);
        if (ok) next(&tmV, 1);
      }
      if (ok && fixTile >= 0 && fixTile == n - 1) {
        for (int k = 0; k < 2 && ok; ++k) {
          const int at = stageOf(k, n - 1);
          ok = warpWaitOr(smemAddr(&s.full[at]), phaseOf(k, n - 1), abortFlag);
          if (ok) {
            clearRows<DP>(smem + Shape::kRing + at * kTileBytes, fixRows, lane);
            if (lane == 0) mbarArrive(smemAddr(&s.fix[k]));
          } else if (lane == 0) {
            fail(1100);
          }
        }
      }
      if (__any_sync(~0u, *abortFlag)) {
        for (int values = 0; values < 2; ++values)
          for (int tile = max(0, loaded[values] - (values ? kValueStages : kKeyStages)); tile < loaded[values]; ++tile)
            mbarWait(smemAddr(&s.full[stageOf(values, tile)]), phaseOf(values, tile), 1u << 20);
        if (ownArmed) mbarWait(smemAddr(s.own), 0, 1u << 20);
      }
    }
  } else if (warp == BackwardWarps::kMma) {
    if (n > 0 && electOne()) {
      bool ok = true;
      auto need = [&](bool got, uint32_t what) {
        if (ok && !got) fail(what);
        ok = ok && got;
        return ok;
      };
      auto full = [&](int values, int tile) { return need(waitOr(smemAddr(&s.full[stageOf(values, tile)]), phaseOf(values, tile), abortFlag), 2000 + stageOf(values, tile)); };
      auto tileAt = [&](int values, int tile) { return smem0 + Shape::kRing + stageOf(values, tile) * kTileBytes; };
      const bool fixed = fixTile >= 0 && fixTile == n - 1;
      auto scores = [&](int i) {
        if (!full(0, i)) return;
        if (fixed && i == n - 1 && !need(waitOr(smemAddr(&s.fix[0]), 0, abortFlag), 2200)) return;
        tcFenceAfter();
        productOfTiles<T, DP>(tmem, descAlong(smem0), descAlong(tileAt(0, i)));
        ummaCommit(smemAddr(s.first));
      };
      auto doV = [&](int i) {
        if (!full(1, i)) return;
        if (fixed && i == n - 1 && !need(waitOr(smemAddr(&s.fix[1]), 0, abortFlag), 2201)) return;
        tcFenceAfter();
        productOfTiles<T, DP>(tmem + 128 + (i & 1) * 128, descAlong(smem0 + kTileBytes), descAlong(tileAt(1, i)));
        ummaCommit(smemAddr(&s.second[i & 1]));
        ummaCommit(smemAddr(&s.empty[stageOf(1, i)]));
      };
      if (need(waitOr(smemAddr(s.own), 0, abortFlag), 2100)) scores(0);
      if (ok) doV(0);
      for (int i = 0; i < n && ok; ++i) {
        if (i + 1 < n) {
          if (!need(waitOr(smemAddr(s.firstDone), i & 1, abortFlag), 2400)) break;   // scores are in registers
          scores(i + 1);
          if (ok) doV(i + 1);   // over ds of the tile before, whose product is in front of this
        }
        if (!ok || !need(waitOr(smemAddr(&s.secondDone[i & 1]), i >> 1 & 1, abortFlag), 2300)) break;
        tcFenceAfter();
        productWithTmem<T, DP>(tmem + 384, tmem + 128 + (i & 1) * 128, descAcross(tileAt(0, i)), i != 0);
        if (FINE) productWithTmem<T, DP>(tmem + 384, tmem + 160 + (i & 1) * 128, descAcross(tileAt(0, i)), true);
        ummaCommit(smemAddr(&s.empty[stageOf(0, i)]));
      }
      if (ok) ummaCommit(smemAddr(s.outBar));
      if (!ok) {
        ummaCommit(smemAddr(s.drain));
        mbarWait(smemAddr(s.drain), 0, 1u << 20);
      }
    }
  } else if (warp < BackwardWarps::kCompute) {
    regsTake<BackwardWarps::kManyRegs>();
    const int half = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tS = tmem + lanes + half * 64;
    const int tok = tok0 + row / a.group, head = kvHead * a.group + row % a.group;
    const bool valid = row < rows && tok < seq.q, exists = row < rows && tok < a.q;
    const int limit = valid ? visibleOf(a, seq, tok) : 0;
    const float c = a.scale * kLog2e, up = n > 0 ? gradScale<T>(a, b, kvHead) : 1.0f;
    float shift = 0.0f, delta = 0.0f;
    if (n > 0) {
      const float* stats = a.stats + (((size_t)b * a.kvHeads + kvHead) * a.tiles + qTile) * 256;
      shift = stats[row] - Pack<T>::kBackwardBias + log2f(up);   // (up is a power of two)
      delta = stats[128 + row];
    }
    const uint64_t c2 = pair(c, c), shift2 = pair(shift, shift), delta2 = pair(delta, delta);
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const uint32_t tDp = tS + 128 + (i & 1) * 128;
      ok = warpWaitOr(smemAddr(s.first), i & 1, abortFlag);
      if (!ok) {
        if (lane == 0) fail(3000);
        break;
      }
      tcFenceAfter();
      uint32_t x[2][32], y[32], packed[32], rest[FINE ? 32 : 1];
      tmemLd32(tS, x[0]);
      tmemLd32(tS + 32, x[1]);
      tmemLdWait32(x[0]);
      tmemLdWait32(x[1]);
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) mbarArrive(smemAddr(s.firstDone));
      const int k0 = (begin + i) * 128 + half * 64;
      const bool hide = __any_sync(~0u, limit < k0 + 64);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint64_t p[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint64_t z = fma2(packF32x2(x[q][2 * k], x[q][2 * k + 1]), c2, shift2);
          p[k] = pair(exp2Fast(lowOf(z)), exp2Fast(highOf(z)));
        }
        if (q == 0) {
          ok = warpWaitOr(smemAddr(&s.second[i & 1]), i >> 1 & 1, abortFlag);
          if (!ok) {
            if (lane == 0) fail(3001);
            break;
          }
          tcFenceAfter();
        }
        tmemLd32(tDp + q * 32, y);
        tmemLdWait32(y);
#pragma unroll
        for (int k = 0; k < 16; ++k) p[k] = mul2(p[k], add2(packF32x2(y[2 * k], y[2 * k + 1]), delta2));
        if (hide) {
#pragma unroll
          for (int k = 0; k < 16; ++k) p[k] = pair(k0 + q * 32 + 2 * k < limit ? lowOf(p[k]) : 0.0f, k0 + q * 32 + 2 * k + 1 < limit ? highOf(p[k]) : 0.0f);
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          packed[q * 16 + k] = Pack<T>::two(lowOf(p[k]), highOf(p[k]));
          if (FINE) rest[q * 16 + k] = remainderOf<T>(packed[q * 16 + k], lowOf(p[k]), highOf(p[k]));
        }
      }
      if (!ok) break;
      tmemSt32(tDp, packed);
      if constexpr (FINE) tmemSt32(tDp + 32, rest);
      tmemStWait();
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) mbarArrive(smemAddr(&s.secondDone[i & 1]));
    }
    if (ok && n > 0) {
      ok = warpWaitOr(smemAddr(s.outBar), 0, abortFlag);
      if (!ok && lane == 0) fail(3100);
      tcFenceAfter();
    }
    if (!__any_sync(~0u, *abortFlag) && half == 0) {
      const size_t at = ((size_t)b * a.q + tok) * a.heads + head;
      const bool whole = a.qParts == 1;
      storeGradient<T, DP>(a, tmem + lanes + 384, n > 0, a.scale / up, exists, valid, whole ? at : (size_t)part * a.batch * a.q * a.heads + at, whole ? a.dq : a.partDq, !whole || a.gradFp32,
                           whole ? a.addDq : nullptr);
    }
  }
}

// The first CTAs own tiles of keys, the others tiles of queries: neither needs the other's, and where both are few they run beside one another.
template <typename T, int DP, bool FINE>
__global__ void __launch_bounds__(BackwardWarps::kThreads, 1)
attnBackwardKernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmDo, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ AttnArgs a) {
  using Shape = BackwardShape<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, rows = a.tileTokens * a.group;
  const bool ofKeys = blockIdx.x < a.kvCtas;
  const BackwardBars s = backwardSetUp<DP>(smem, warp);
  if (ofKeys && warp < BackwardWarps::kCompute && rows < 128) {
    // rows of a tile that no copy writes are operands of sums over the rows: zero, for good
    const int each = (128 - rows) * 8;
    for (int i = threadIdx.x; i < Shape::kStages * (DP / 64) * each; i += BackwardWarps::kCompute * 32)
      *(uint4*)(smem + Shape::kRing + i / each * kHalfTile + rows * 128 + i % each * 16) = make_uint4(0, 0, 0, 0);
    fenceProxyAsync();
  }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmem = *s.tmemSlot;
  pdlEnter();   // the set-up above overlaps the end of the kernel before
  if (ofKeys) backwardKv<T, DP, FINE>(tmQ, tmDo, tmK, tmV, a, smem, s, tmem, blockIdx.x);
  else backwardQ<T, DP, FINE>(tmQ, tmDo, tmK, tmV, a, smem, s, tmem, blockIdx.x - a.kvCtas);
  tcFenceBefore();
  __syncthreads();
  if (warp == BackwardWarps::kMma) {
    tcFenceAfter();
    tmemDealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------- parts
// dq, dk and dv from the parts' sums, added up in order, and what is there already. A thread has four channels of a row; rows behind a sequence's last are zeros in every part. It reads
// what was just written, mostly from level 2: 12 MB of parts 5 us with its launch.
template <typename T>
__global__ void __launch_bounds__(256) attnSumKernel(const __grid_constant__ AttnArgs a) {
  const int quads = a.dim / 4;
  const size_t qRows = a.qParts > 1 ? (size_t)a.batch * a.q * a.heads : 0, kvRows = a.kvParts > 1 ? (size_t)a.batch * a.kv * a.kvHeads : 0;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  size_t row = i / quads;
  if (row >= qRows + 2 * kvRows) return;
  const int which = row < qRows ? 0 : row < qRows + kvRows ? 1 : 2;   // dq, dk, dv
  if (which) row -= qRows + (which == 2 ? kvRows : 0);
  const int heads = which ? a.kvHeads : a.heads, tokens = which ? a.kv : a.q, parts = which ? a.kvParts : a.qParts;
  const int tok = (int)(row / heads % tokens), b = (int)(row / heads / tokens);
  const size_t at = row * quads + i % quads, stride = (which ? kvRows : qRows) * quads;
  const float4* from = (const float4*)(which == 0 ? a.partDq : which == 1 ? a.partDk : a.partDv) + at;
  const float4* add = (const float4*)(which == 0 ? a.addDq : which == 1 ? a.addDk : a.addDv);
  pdlEnter();
  const int* lengths = which ? a.kvLengths : a.qLengths;
  float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const float4 v = from[p * stride];
    f.x += v.x; f.y += v.y; f.z += v.z; f.w += v.w;
  }
  if (add && (!lengths || tok < lengths[b])) {
    const float4 v = add[at];
    f.x += v.x; f.y += v.y; f.z += v.z; f.w += v.w;
  }
  void* to = which == 0 ? a.dq : which == 1 ? a.dk : a.dv;
  if (a.gradFp32) ((float4*)to)[at] = f;
  else ((uint2*)to)[at] = make_uint2(Pack<T>::two(f.x, f.y), Pack<T>::two(f.z, f.w));
}

// ---------------------------------------------------------------------------------------------- what both need of each row of queries
// Minus <do, o> (unless that is given: minus what is), and minus the log-sum-exp in units of log 2, laid out as the tiles are. Rows that nobody has, and rows that
// see no key, get an infinite log-sum-exp and a delta of zero: their probabilities and ds are zero. A CTA takes a tile, 8 or 16 lanes a row, a pack of 16 bytes each. fp16: the longest
// row of do and the largest delta in it, and by the CTAs behind those the longest of every 128 rows of v. Bound by its instructions, of which 73 % of the slots are issued: a reduction over the lanes for each row (fp16: two), divisions
// by the group and addresses. 4096 tokens of 32 heads of 128 channels 19.6 us (68 MB, 43 % of memory's rate; fp16, with 8 key heads' values, 22.5), 8192 33 us; with loads that a condition
// guards row by row it took twice that.
template <typename T, int LANES>
__global__ void __launch_bounds__(256, 4) attnStatsKernel(const __grid_constant__ AttnStatsArgs a) {
  constexpr int kAtOnce = 256 / LANES, kTurns = 4;   // rows of the CTA, and of a thread with loads on their way
  const int lane = threadIdx.x % LANES, row0 = threadIdx.x / LANES, packs = a.dim / 8;
  const bool has = lane < packs;
  const int channel = has ? lane * 8 : 0;
  auto load = [&](const void* x, long long at) { return *(const uint4*)((const uint16_t*)x + at + channel); };
  auto dot = [&](uint4 x, uint4 y) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = Pack<T>::both(u[i]), q = Pack<T>::both(v[i]);
      sum += p.x * q.x + p.y * q.y;
    }
    sum = has ? sum : 0.0f;
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    return sum;
  };
  const unsigned owners = a.batch * a.kvHeads, qTiles = owners * a.tiles;
  const bool ofV = blockIdx.x >= qTiles;   // 128 rows of v instead of a tile
  const unsigned block = ofV ? blockIdx.x - qTiles : blockIdx.x, owner = block % owners;
  const int tile = block / owners, kvHead = owner % a.kvHeads, b = owner / a.kvHeads;
  uint32_t most = 0, mostDelta = 0;   // the squared norm of the longest row, and the largest |delta|, as bits
  // The CTA's into their places.
  auto largest = [&] {
    __shared__ uint32_t ofWarp[2][8];
    most = __reduce_max_sync(~0u, most);
    mostDelta = __reduce_max_sync(~0u, mostDelta);
    if (threadIdx.x % 32 == 0) {
      ofWarp[0][threadIdx.x / 32] = most;
      ofWarp[1][threadIdx.x / 32] = mostDelta;
    }
    __syncthreads();
    if (threadIdx.x < (ofV ? 1 : 2)) {
      uint32_t all = 0;
      for (int i = 0; i < 8; ++i) all = max(all, ofWarp[threadIdx.x][i]);
      a.bounds[(size_t)owner * (2 * a.tiles + a.vTiles) + (ofV ? 2 * a.tiles + tile : 2 * tile + threadIdx.x)] = all;
    }
  };
  pdlEnter();
  if (ofV) {
    const int used = a.kvLengths ? min(a.kvLengths[b], a.kv) : a.kv;
    if (tile * 128 >= used) {
      largest();
      return;
    }
    const long long base = b * a.vStride[0] + kvHead * a.vStride[2];
    for (int pass = 0; pass < 128; pass += kAtOnce * kTurns) {
      uint4 x[kTurns];
#pragma unroll
      for (int n = 0; n < kTurns; ++n) x[n] = load(a.v, base + min(tile * 128 + pass + row0 + n * kAtOnce, used - 1) * a.vStride[1]);
#pragma unroll
      for (int n = 0; n < kTurns; ++n) {
        most = max(most, __float_as_uint(dot(x[n], x[n])) & 0x7fffffffu);
      }
    }
    largest();
    return;
  }
  const int used = a.qLengths ? max(0, min(a.qLengths[b], a.q)) : a.q, tok0 = tile * a.tileTokens, rows = a.tileTokens * a.group;
  const int some = min(used - tok0, a.tileTokens) * a.group;   // rows that somebody has
  float* to = a.stats + ((size_t)owner * a.tiles + tile) * 256 + row0;
  const size_t base = ((size_t)b * a.heads + kvHead * a.group) * a.q + tok0;   // of lse and delta
  const bool needX = !a.delta || a.bounds;
  for (int pass = 0; pass < 128; pass += kAtOnce * kTurns) {
    uint4 x[kTurns] = {}, y[kTurns] = {};
    float lse[kTurns], delta[kTurns];
    size_t at[kTurns];
#pragma unroll
    for (int n = 0; n < kTurns; ++n) {
      const int row = max(0, min(pass + row0 + n * kAtOnce, some - 1)), t = row / a.group, head = row - t * a.group;   // (a row behind the last stands for it)
      at[n] = base + (size_t)head * a.q + t;
      if (some > 0) {
        if (needX) x[n] = load(a.dout, b * a.doutStride[0] + (tok0 + t) * a.doutStride[1] + (kvHead * a.group + head) * a.doutStride[2]);
        if (!a.delta) y[n] = load(a.out, b * a.outStride[0] + (tok0 + t) * a.outStride[1] + (kvHead * a.group + head) * a.outStride[2]);
        if (a.delta) delta[n] = a.delta[at[n]];
        if (a.stats) lse[n] = a.lse[at[n]];
      }
    }
#pragma unroll
    for (int n = 0; n < kTurns; ++n) {
      const int row = pass + row0 + n * kAtOnce;
      if (!a.delta) delta[n] = dot(x[n], y[n]);
      if (a.bounds) most = max(most, __float_as_uint(dot(x[n], x[n])) & 0x7fffffffu);
      if (row >= some) {
        delta[n] = 0.0f;
        lse[n] = -INFINITY;
      }
      if (a.stats && lse[n] == -INFINITY) delta[n] = 0.0f;   // (of a row that sees no key it may have been given as anything)
      if (a.bounds) mostDelta = max(mostDelta, __float_as_uint(delta[n]) & 0x7fffffffu);
      if (a.stats && lane == 0) {
        to[row - row0] = lse[n] == -INFINITY ? -INFINITY : fmaf(lse[n], -kLog2e, Pack<T>::kBackwardBias);
        to[row - row0 + 128] = -delta[n];
      }
      if (a.deltaOut && lane == 0 && row < rows) {
        const int t = row / a.group;
        if (tok0 + t < a.q) a.deltaOut[base + (size_t)(row - t * a.group) * a.q + t] = delta[n];
      }
    }
  }
  if (a.bounds) largest();
}

}  // namespace

template <typename T> static const void* backwardFn(int dim, bool fine) {
  if (dim <= 64) return fine ? (const void*)attnBackwardKernel<T, 64, true> : (const void*)attnBackwardKernel<T, 64, false>;
  return fine ? (const void*)attnBackwardKernel<T, 128, true> : (const void*)attnBackwardKernel<T, 128, false>;
}
const void* attnBackwardKernelFn(int type, int dim, bool fine) { return type == ATTN_F16 ? backwardFn<__half>(dim, fine) : backwardFn<__nv_bfloat16>(dim, fine); }
const void* attnSumKernelFn(int type) { return type == ATTN_F16 ? (const void*)attnSumKernel<__half> : (const void*)attnSumKernel<__nv_bfloat16>; }
int attnBackwardThreads() { return BackwardWarps::kThreads; }
int attnBackwardRegs() { return BackwardWarps::kLaunchRegs; }
size_t attnBackwardSmemBytes(int dim) { return dim <= 64 ? BackwardShape<64>::kBytes : BackwardShape<128>::kBytes; }
const void* attnStatsKernelFn(int type, int dim) {
  if (dim <= 64) return type == ATTN_F16 ? (const void*)attnStatsKernel<__half, 8> : (const void*)attnStatsKernel<__nv_bfloat16, 8>;
  return type == ATTN_F16 ? (const void*)attnStatsKernel<__half, 16> : (const void*)attnStatsKernel<__nv_bfloat16, 16>;
}

}  // namespace b200
