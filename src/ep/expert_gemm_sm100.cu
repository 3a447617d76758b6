// The experts' products for sm_100a: one matrix product per expert over the rows that dispatch packed for it, bf16 operands, fp32 sums in
// tensor memory. With x [experts][cap][K], W [experts][N][K] and counts[e] rows in use:
//   FORWARD  out[e] = act(x[e] W[e]^T + b[e]) + r[e]        both operands lie along the sum (K-major)
//   DX       dx[e]  = dz[e] W[e]                            W lies across it (MN-major)
//   DW       dw[e]  = dz[e]^T x[e], sums over the rows      both lie across it
// Only the device knows the counts: every CTA reads them, counts the tiles of all experts and walks its share of them, so that one launch
// serves a single token and a full batch alike.
//
// One persistent CTA per SM, 320 threads in three roles:
//   warp 0      TMA producer: 128 x 64 tiles of the first operand and up to 256 x 64 of the second (128-byte swizzle) through a ring in
//               shared memory. Of few rows only the boxes of 32 that hold some are fetched; the rows behind them in shared memory are
//               whatever was there: they reach only results that nobody stores.
//   warp 1      MMA issuer: tcgen05.mma 128 x BN x 16 into one of two accumulators in tensor memory.
//   warps 2-9   epilogue, two warps to 32 rows: bias, activation, residual, rounding, stores of whole 128-byte lines.
// The last step of DW's sum may hold rows behind the expert's last: the issuing warp writes zeros over them in shared memory.
// Every wait is bounded; on expiry the kernel records a status, waits for its copies in flight, frees its tensor memory and returns.
#include "../kernels/common.cuh"
#include "../tp/gemm_sm100.cuh"
#include "moe_math.cuh"
#include "moe_ops.h"

namespace b200 {

using namespace sm100;

namespace {

constexpr int kBM = 128, kBK = 64, kUmmaK = 16, kMaxBN = 256;
constexpr int kThreads = 320, kEpiWarps = 8;
constexpr uint32_t kTmemCols = 512, kAccCols = 256;
constexpr uint32_t kRingBytes = 4 * (kBM + kMaxBN) * kBK * 2;
constexpr int kMaxStages = 12;
constexpr uint32_t kBlockBytes = 64 * kBK * 2;   // of a box of 64 x 64
constexpr size_t kCtrlBytes = 512;
static_assert((2 * kMaxStages + 4) * 8 + 8 <= kCtrlBytes, "control block too small");
constexpr size_t kTableBytes = (kExpertMax + 1) * 4 + 12;
constexpr size_t kSmemBytes = 1024 + kRingBytes + kEpiWarps * 4096 + kCtrlBytes + kTableBytes;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");

__device__ __forceinline__ void tmaLoad3d(uint32_t dstSmem, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dstSmem), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}

// An operand that lies across the sum, in boxes of 64 values x 64 steps with 128-byte swizzle: the next 64 values are a box further, the
// next 8 steps 1024 bytes.
__device__ __forceinline__ uint64_t descAcross(uint32_t smemByteAddr) {
  uint64_t d = 0;
  d |= (uint64_t)((smemByteAddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(kBlockBytes >> 4) << 16;   // leading byte offset: next 64 values
  d |= (uint64_t)(1024 >> 4) << 32;          // stride byte offset: next 8 steps of the sum
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

struct Tile {
  int e, rows, row0, col0, steps;   // expert, its rows in use, first row and column of the result, 64-wide steps of the sum
};

}  // namespace

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
expertGemmKernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmASmall, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmBSmall, const __grid_constant__ ExpertGemmArgs a) {
  constexpr bool kAcrossA = MODE == EXPERT_DW, kAcrossB = MODE != EXPERT_FORWARD;
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smemRaw + 1023) & ~(uintptr_t)1023);
  uint8_t* epiBuf = smem + kRingBytes;
  uint8_t* ctrl = epiBuf + kEpiWarps * 4096;
  uint64_t* fullBar = (uint64_t*)ctrl;              // [kMaxStages]
  uint64_t* emptyBar = fullBar + kMaxStages;        // [kMaxStages]
  uint64_t* accFull = emptyBar + kMaxStages;        // [2]
  uint64_t* accEmpty = accFull + 2;                 // [2]
  uint32_t* tmemSlot = (uint32_t*)(accEmpty + 2);
  volatile uint32_t* abortFlag = tmemSlot + 1;
  int* tileStart = (int*)(ctrl + kCtrlBytes);       // [experts + 1] row tiles in front of each expert's
  int* mostRows = tileStart + kExpertMax + 1;       // of one expert

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) { mbarInit(smemAddr(&fullBar[s]), 1); mbarInit(smemAddr(&emptyBar[s]), 1); }
    for (int b = 0; b < 2; ++b) { mbarInit(smemAddr(&accFull[b]), 1); mbarInit(smemAddr(&accEmpty[b]), kEpiWarps); }
    *abortFlag = 0;
    mbarInitFence();
    prefetchTensorMap(&tmA);
    prefetchTensorMap(&tmB);
  }
  if (warp == 1) {
    tmemAlloc(smemAddr(tmemSlot), kTmemCols);
    tmemRelinquish();
  }
  pdlEnter();   // the set-up above overlaps the end of the kernel before

  auto rowsOf = [&](int e) { return a.counts ? min(max(a.counts[e], 0), a.cap) : a.cap; };
  if (warp == 0) {
    int before = 0, most = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane, rows = e < a.experts ? rowsOf(e) : 0;
      int n = e >= a.experts ? 0 : ((MODE == EXPERT_DW ? a.outRows : rows) + kBM - 1) / kBM;
      most = max(most, rows);
      const int mine = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(~0u, n, o);
        if (lane >= o) n += v;
      }
      if (e < a.experts) tileStart[e] = before + n - mine;
      before += __shfl_sync(~0u, n, 31);
    }
    most = __reduce_max_sync(~0u, most);
    if (lane == 0) {
      tileStart[a.experts] = before;
      *mostRows = most;
    }
  }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmemBase = *tmemSlot;

  // Width of the tiles: the one that the SMs finish first, a wave of tiles taken to cost its columns and a fixed part for the first
  // operand and the start. The sums do not depend on it.
  const int parts = MODE == EXPERT_FORWARD && a.gated ? 2 : 1;
  const int rowTiles = tileStart[a.experts];
  int bn = kMaxBN;
  {
    long long best = 0;
    for (int w = kMaxBN; w >= (MODE == EXPERT_FORWARD && parts == 1 ? 32 : 64); w >>= 1) {
      const long long tiles = (long long)rowTiles * ((a.cols + w / parts - 1) / (w / parts));
      const long long cost = (tiles + gridDim.x - 1) / gridDim.x * (w + 32);
      if (w == kMaxBN || cost < best) { best = cost; bn = w; }
    }
  }
  const int outCols = bn / parts;                       // columns of the result in a tile
  const int tilesN = (a.cols + outCols - 1) / outCols;
  // of the first operand only the boxes that hold rows are fetched: where no expert has many, the ring has more and smaller stages
  const uint32_t aBytes = kAcrossA ? 2 * kBlockBytes : (uint32_t)min(kBM, (*mostRows + 31) / 32 * 32) * 128;
  const uint32_t stageBytes = aBytes + (uint32_t)bn * 128;
  const int stages = (int)min((uint32_t)kMaxStages, kRingBytes / stageBytes);
  const uint32_t ring = smemAddr(smem);
  const int nTiles = rowTiles * tilesN;

  // Tiles of an expert in panels of 8 row tiles: those in flight share both operands.
  auto tileAt = [&](int t) {
    Tile r;
    int lo = 0, hi = a.experts;
    while (hi - lo > 1) {   // the last expert whose tiles begin at or before t, among those with tiles
      const int mid = (lo + hi) / 2;
      if (tileStart[mid] * tilesN <= t) lo = mid;
      else hi = mid;
    }
    r.e = lo;
    r.rows = rowsOf(lo);
    const int j = t - tileStart[lo] * tilesN, mine = tileStart[lo + 1] - tileStart[lo];
    const int panel = j / (8 * tilesN), width = min(8, mine - panel * 8), k = j - panel * 8 * tilesN;
    r.row0 = (panel * 8 + k % width) * kBM;
    r.col0 = k / width * outCols;
    r.steps = ((MODE == EXPERT_DW ? r.rows : a.depth) + kBK - 1) / kBK;
    return r;
  };
  auto fail = [&](uint32_t what) {
    *abortFlag = 1;
    if (a.status && ldRelaxedSys(a.status) == DEV_OK) {
      a.status[1] = WAIT_TILE;
      a.status[2] = what;
      a.status[3] = blockIdx.x;
      __threadfence_system();
      stRelaxedSys(a.status, DEV_TIMEOUT);
    }
  };

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, armed = 0;   // stages that were ever loaded
      uint32_t phase = 0;
      for (int t = blockIdx.x; t < nTiles && !*abortFlag; t += gridDim.x) {
        const Tile c = tileAt(t);
        const int left = (MODE == EXPERT_DW ? a.outRows : c.rows) - c.row0;
        const int aBoxes = kAcrossA ? (left > 64 ? 2 : 1) : min(kBM / 32, (left + 31) / 32);
        const int bLeft = min(outCols, a.cols - c.col0), perPart = outCols >= 64 ? 64 : 32;
        const int bBoxes = kAcrossB ? (bLeft + 63) / 64 : (bLeft + perPart - 1) / perPart;
        const uint32_t bytes = (kAcrossA ? aBoxes * kBlockBytes : aBoxes * 32 * 128) + (kAcrossB ? bBoxes * kBlockBytes : (uint32_t)(parts * bBoxes * perPart) * 128);
        for (int kb = 0; kb < c.steps; ++kb) {
          if (!mbarWait(smemAddr(&emptyBar[s]), phase ^ 1)) { fail(1000 + s); break; }
          if (*abortFlag) break;
          const uint32_t full = smemAddr(&fullBar[s]), sA = ring + s * stageBytes, sB = sA + aBytes;
          mbarExpectTx(full, bytes);
          if (kAcrossA) {
            for (int i = 0; i < aBoxes; ++i) tmaLoad3d(sA + i * kBlockBytes, &tmA, c.row0 + i * 64, kb * kBK, c.e, full);
          } else if (aBoxes == kBM / 32) {
            tmaLoad3d(sA, &tmA, kb * kBK, c.row0, c.e, full);
          } else {
            for (int i = 0; i < aBoxes; ++i) tmaLoad3d(sA + i * 32 * 128, &tmASmall, kb * kBK, c.row0 + i * 32, c.e, full);
          }
          if (kAcrossB) {
            for (int i = 0; i < bBoxes; ++i) tmaLoad3d(sB + i * kBlockBytes, &tmB, c.col0 + i * 64, kb * kBK, c.e, full);
          } else {
            const CUtensorMap* map = perPart == 64 ? &tmB : &tmBSmall;
            for (int p = 0; p < parts; ++p)
              for (int i = 0; i < bBoxes; ++i)
                tmaLoad3d(sB + (p * outCols + i * perPart) * 128, map, kb * kBK, p * a.cols + c.col0 + i * perPart, c.e, full);
          }
          armed = max(armed, s + 1);
          if (++s == stages) { s = 0; phase ^= 1; }
        }
      }
      if (*abortFlag) {
        // copies already issued still write into shared memory: wait for them (bounded). A stage in front of s was loaded in this round, one from s on in the one before
        for (int i = 0; i < armed; ++i) mbarWait(smemAddr(&fullBar[i]), i < s ? phase : phase ^ 1, 1u << 20);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = umInstrBf16(kBM, bn) | (kAcrossA ? 1u << 15 : 0u) | (kAcrossB ? 1u << 16 : 0u);
    int s = 0, it = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x; t < nTiles && !__any_sync(~0u, *abortFlag); t += gridDim.x) {
      const Tile c = tileAt(t);
      if (c.steps == 0) continue;   // nothing to add up: the epilogue writes zeros
      const int buf = it & 1;
      const uint32_t aph = (it >> 1) & 1;
      ++it;
      if (!__all_sync(~0u, mbarWait(smemAddr(&accEmpty[buf]), aph ^ 1))) { if (lane == 0) fail(2000 + buf); break; }
      tcFenceAfter();
      const uint32_t dT = tmemBase + buf * kAccCols;
      const int length = MODE == EXPERT_DW ? c.rows : a.depth;
      bool bad = false;
      for (int kb = 0; kb < c.steps; ++kb) {
        if (!__all_sync(~0u, mbarWait(smemAddr(&fullBar[s]), phase))) { if (lane == 0) fail(3000 + s); bad = true; break; }
        const uint32_t sA = ring + s * stageBytes, sB = sA + aBytes;
        const int left = length - kb * kBK, chunks = min(kBK / kUmmaK, (left + kUmmaK - 1) / kUmmaK);
        if (MODE == EXPERT_DW && left < chunks * kUmmaK) {
          // rows behind the expert's last are somebody's old values: zeros, so that they add nothing (a row is 128 bytes of every box)
          const int rows = chunks * kUmmaK - left, boxes = 2 + bn / 64;
          for (int i = lane; i < boxes * rows * 8; i += 32) {
            const int box = i / (rows * 8), r = i / 8 % rows;
            *(uint4*)(smem + (size_t)s * stageBytes + box * kBlockBytes + (left + r) * 128 + i % 8 * 16) = make_uint4(0, 0, 0, 0);
          }
          fenceProxyAsync();
          __syncwarp();
        }
        tcFenceAfter();
        if (lane == 0) {
          for (int k = 0; k < chunks; ++k) {
            const uint64_t da = kAcrossA ? descAcross(sA + k * kUmmaK * 128) : umDescK128(sA + k * kUmmaK * 2);
            const uint64_t db = kAcrossB ? descAcross(sB + k * kUmmaK * 128) : umDescK128(sB + k * kUmmaK * 2);
            ummaBf16(dT, da, db, idesc, (kb | k) != 0);
          }
          ummaCommit(smemAddr(&emptyBar[s]));
        }
        __syncwarp();
        if (++s == stages) { s = 0; phase ^= 1; }
      }
      if (bad) break;
      if (lane == 0) ummaCommit(smemAddr(&accFull[buf]));
      __syncwarp();
    }
  } else {
    // ---- epilogue: TMEM lanes [32q, 32q+32) belong to the warps with warp % 4 == q; of those two, each takes every other 64 columns
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* wbuf = epiBuf + (size_t)(warp - 2) * 4096;
    int it = 0;
    for (int t = blockIdx.x; t < nTiles && !__any_sync(~0u, *abortFlag); t += gridDim.x) {
      const Tile c = tileAt(t);
      const int buf = it & 1;
      const uint32_t aph = (it >> 1) & 1;
      if (c.steps) {
        ++it;
        if (!__all_sync(~0u, mbarWait(smemAddr(&accFull[buf]), aph))) { if (lane == 0) fail(4000 + buf); break; }
        tcFenceAfter();
      }
      const int row = c.row0 + q * 32, left = (MODE == EXPERT_DW ? a.outRows : c.rows) - row;   // this warp's first row, rows from there on
      const uint32_t tBase = tmemBase + ((uint32_t)(q * 32) << 16) + buf * kAccCols;
      const size_t first = (size_t)c.e * (MODE == EXPERT_DW ? a.outRows : a.cap) + row;
      for (int cc = half * 64; cc < outCols && c.col0 + cc < a.cols && left > 0; cc += 128) {
        const int col = c.col0 + cc, width = min(min(64, outCols - cc), a.cols - col);   // a multiple of 8
        // 64 columns of 32 rows between the lanes (a row each) and whole lines of memory, 16-byte chunks XOR-swizzled by row
        auto chunk = [&](int r, int j) { return (uint4*)(wbuf + r * 128 + ((j ^ (r & 7)) * 16)); };
        auto store = [&](__nv_bfloat16* to, size_t ld) {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int r = k * 4 + (lane >> 3), j = lane & 7;
            if (r < left && j * 8 < width) *(uint4*)(to + (size_t)r * ld + j * 8) = *chunk(r, j);
          }
          __syncwarp();
        };
        auto sums = [&](int part, int h, float (&v)[32]) {
          uint32_t r[32];
          tmemLd32(tBase + part * outCols + cc + h * 32, r);
          tmemLdWait32(r);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
          if (MODE == EXPERT_FORWARD && a.bias) {
            const __nv_bfloat16* b = (const __nv_bfloat16*)a.bias + ((size_t)c.e * parts + part) * a.cols + col + h * 32;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (h * 32 + j * 8 >= width) break;
              float f[8];
              unpackBf16x8(__ldg((const uint4*)b + j), f);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[j * 8 + i] += f[i];
            }
          }
        };
        if (MODE == EXPERT_FORWARD && a.pre) {
          for (int p = 0; p < parts; ++p) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h * 32 >= width) break;
              float v[32];
              sums(p, h, v);
#pragma unroll
              for (int j = 0; j < 4; ++j) *chunk(lane, h * 4 + j) = packBf16x8(v + j * 8);
            }
            store((__nv_bfloat16*)a.pre + (first * parts + p) * a.cols + col, (size_t)parts * a.cols);
          }
        }
        if (MODE == EXPERT_FORWARD && a.residual) {
          const __nv_bfloat16* from = (const __nv_bfloat16*)a.residual + first * a.cols + col;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int r = k * 4 + (lane >> 3), j = lane & 7;
            *chunk(r, j) = r < left && j * 8 < width ? *(const uint4*)(from + (size_t)r * a.cols + j * 8) : make_uint4(0, 0, 0, 0);
          }
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h * 32 >= width) break;
          float v[32];
          if (MODE == EXPERT_DW && c.steps == 0) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.0f;
          } else {
            sums(0, h, v);
          }
          if (MODE == EXPERT_FORWARD) {
            if (parts == 2) {
              float u[32];
              sums(1, h, u);
              const int base = a.act == ACT_SWIGLU ? ACT_SILU : ACT_GELU;
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = activation(base, v[i]) * u[i];
            } else if (a.act != ACT_NONE) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = activation(a.act, v[i]);
            }
            if (a.residual) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float f[8];
                unpackBf16x8(*chunk(lane, h * 4 + j), f);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j * 8 + i] += f[i];
              }
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) *chunk(lane, h * 4 + j) = packBf16x8(v + j * 8);
        }
        store((__nv_bfloat16*)a.out + first * a.cols + col, (size_t)a.cols);
      }
      if (c.steps) {
        tcFenceBefore();
        __syncwarp();
        if (lane == 0) mbarArrive(smemAddr(&accEmpty[buf]));
      }
    }
  }

  tcFenceBefore();
  __syncthreads();
  if (warp == 1) {
    tcFenceAfter();
    tmemDealloc(tmemBase, kTmemCols);
  }
}

const void* expertGemmKernelFn(int mode) {
  return mode == EXPERT_DW ? (const void*)expertGemmKernel<EXPERT_DW> : mode == EXPERT_DX ? (const void*)expertGemmKernel<EXPERT_DX> : (const void*)expertGemmKernel<EXPERT_FORWARD>;
}
size_t expertGemmSmemBytes() { return kSmemBytes; }
int expertGemmThreads() { return kThreads; }

}  // namespace b200
