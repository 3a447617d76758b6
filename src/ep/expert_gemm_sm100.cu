// The experts' products for sm_100a: one matrix product per expert over the rows that dispatch packed for it, bf16 operands, fp32 sums in
// tensor memory. With x [experts][cap][K], W [experts][N][K] and counts[e] rows in use:
//   FORWARD  out[e] = act(x[e] W[e]^T + b[e]) + r[e]        both operands lie along the sum (K-major)
//   DX       dx[e]  = dz[e] W[e]                            W lies across it (MN-major)
//   DW       dw[e]  = dz[e]^T x[e], sums over the rows      both lie across it
// Only the device knows the counts: every CTA reads them, counts the tiles of all experts and walks its share of them, so that one launch
// serves a single token and a full batch alike.
//
// Two kernels. expertGemmPairKernel: CTA pairs (clusters of two, tcgen05 cta_group::2) on tiles of 256 rows x up to 256 columns; each CTA stages
// its 128 rows of the first operand and its half of the second per 64 steps of the sum, and keeps the results of its rows. A CTA alone
// would need 48 KiB where one of a pair needs 32, more than level 2 delivers while the tensor cores work on them (4 x 2048 rows, 4096 x 4096:
// 1142 TFLOP/s; pairs 1530 to 1560). expertGemmKernel: one CTA per tile of 128 rows, where no expert can have more: there the weights are the traffic.
//
// Persistent CTAs, one per SM, in roles:
//   warp 0      TMA producer: operand tiles (128-byte swizzle) through a ring in shared memory
//   warp 1      MMA issuer (of a pair: the first CTA's) into one of two accumulators in tensor memory; a pair's second: the bias's gradient from the slices' sums
//   warps 2-9   epilogue, two warps to 32 rows: bias, activation, residual, rounding, stores
//   warp 10     DW: the last step of a sum may hold rows behind the expert's last; zeros are written over them in shared memory
// Rows of the first operand that were not fetched, or lie behind the last, are whatever shared memory held: they reach only results that nobody stores.
// Every wait is bounded; on expiry the kernel records a status, waits for its copies in flight, frees its tensor memory and returns.
#include "../kernels/common.cuh"
#include "../tp/gemm_sm100.cuh"
#include "moe_math.cuh"
#include "moe_ops.h"

namespace b200 {

using namespace sm100;

namespace {

constexpr int kBK = 64, kUmmaK = 16, kMaxBN = 256;
constexpr int kEpiWarps = 8, kFirstEpiWarp = 2, kFixWarp = kFirstEpiWarp + kEpiWarps;
constexpr int kThreads = kFixWarp * 32, kPairThreads = kThreads + 32;
constexpr uint32_t kTmemCols = 512, kAccCols = 256;
constexpr uint32_t kRingBytes = 224 << 10;
constexpr int kMaxStages = 12, kMaxPairStages = 7;
constexpr uint32_t kHalfBytes = 128 * kBK * 2;   // 128 rows (or columns) of an operand, 64 steps
constexpr uint32_t kBlockBytes = 64 * kBK * 2;   // a box of 64 x 64
constexpr size_t kCtrlBytes = 512, kTableBytes = (kExpertMax + 1) * 4 + 12;
constexpr size_t kSmemBytes = 1024 + kRingBytes + kCtrlBytes + kTableBytes;
static_assert((2 * kMaxStages + 4) * 8 + 8 <= kCtrlBytes && (4 * kMaxPairStages + 4) * 8 + 8 <= kCtrlBytes, "control block too small");
static_assert(kMaxPairStages * 2 * kHalfBytes <= kRingBytes && 6 * 2 * kHalfBytes + kEpiWarps * 4096 <= kRingBytes && kSmemBytes <= 227 * 1024, "shared memory");

__device__ __forceinline__ void tmaLoad3d(uint32_t dstSmem, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dstSmem), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
// The same, counted on an mbarrier of either CTA of the pair (cluster address). No multicast.
__device__ __forceinline__ void tmaLoad3dPair(uint32_t dstSmem, const CUtensorMap* map, int c0, int c1, int c2, uint32_t barCluster) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dstSmem), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(barCluster) : "memory");
}

// Waits of the roles: they end early when another role has given up. The flag is looked at where there is something to wait for, not in every step. `waits`: how
// many waits of the other roles this one may span.
__device__ __forceinline__ bool waitOr(uint32_t bar, uint32_t parity, volatile uint32_t* abortFlag, uint32_t waits = 1) {
  if (mbarTry(bar, parity)) return true;
  for (uint64_t i = 0; i < (uint64_t)waits << 24 && !*abortFlag; ++i)
    if (mbarTry(bar, parity)) return true;
  return false;
}
// The same for a warp of the epilogue: one lane asks, now and then (eight warps that ask all the time slow the others' barriers down).
__device__ __forceinline__ bool warpWaitOr(uint32_t bar, uint32_t parity, volatile uint32_t* abortFlag, int lane) {
  bool ok = true;
  if (lane == 0) {
    ok = mbarTry(bar, parity);
    for (uint32_t i = 0; i < (1u << 24) && !ok && !*abortFlag; ++i) {
      __nanosleep(64);
      ok = mbarTry(bar, parity);
    }
  }
  ok = __shfl_sync(~0u, (int)ok, 0);
  if (ok) mbarTry(bar, parity);   // every lane has seen the phase end
  return ok;
}

// Arrival at an mbarrier of the pair that publishes no memory: with release it waits until all of the warp's stores are done (DW over experts of
// 64 rows, 32 x 4096 x 7168: 598 us, 439 with this one).
__device__ __forceinline__ void mbarArriveRelaxed(uint32_t clusterAddr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(clusterAddr) : "memory");
}
// As waitOr, for what the other CTA of the pair wrote before it arrived.
__device__ __forceinline__ bool waitClusterOr(uint32_t bar, uint32_t parity, volatile uint32_t* abortFlag) {
  for (uint32_t i = 0; i < 1u << 24; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    if (*abortFlag) break;
  }
  return false;
}

// After one of the roles has given up: copies that count on a barrier of the other CTA, and products whose end nobody waited for, may still be on
// their way into memory that this CTA is about to leave. No barrier here shows their end, so they get a millisecond, hundreds of times what they take.
__device__ __noinline__ void letThemLand() {
  const uint64_t from = globalTimerNs();
  for (int i = 0; i < 1 << 16 && globalTimerNs() - from < 1000000; ++i) __nanosleep(1000);
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
template <bool ACROSS> __device__ __forceinline__ uint64_t descOf(uint32_t addr) { return ACROSS ? descAcross(addr) : umDescK128(addr); }
template <bool ACROSS> constexpr uint64_t kNextDesc = (ACROSS ? kUmmaK * 128 : kUmmaK * 2) >> 4;   // 16 steps on, in 16-byte units

template <int MODE> constexpr bool kAcrossA = MODE == EXPERT_DW;
template <int MODE> constexpr bool kAcrossB = MODE != EXPERT_FORWARD;

struct Tile {
  int e, rows, row0, col0, steps;   // expert, its rows in use, first row and column of the result, 64-wide steps of the sum
};

// ceil(2^32 / n): the quotient of numbers below 2^26 by 2 .. 8 is the high word of the product.
__constant__ uint32_t kInverse[9] = {0, 0, 0x80000000u, 0x55555556u, 0x40000000u, 0x33333334u, 0x2aaaaaabu, 0x24924925u, 0x20000000u};

// The tiles of all experts and their order.
template <int MODE, int BM>
struct Tiles {
  const ExpertGemmArgs& a;
  const int* start;          // [experts + 1] row tiles in front of each expert's
  int bn, parts;             // columns of a tile's accumulator, and of how many parts (gate and up) they are
  int outCols, tilesN, count;

  __device__ __forceinline__ static int rowsOf(const ExpertGemmArgs& a, int e) { return a.counts ? min(max(a.counts[e], 0), a.cap) : a.cap; }

  // One warp fills the table.
  __device__ static void fill(const ExpertGemmArgs& a, int* start, int lane) {
    int before = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane;
      const int mine = e < a.experts ? ((MODE == EXPERT_DW ? a.outRows : rowsOf(a, e)) + BM - 1) / BM : 0;
      int n = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(~0u, n, o);
        if (lane >= o) n += v;
      }
      if (e < a.experts) start[e] = before + n - mine;
      before += __shfl_sync(~0u, n, 31);
    }
    if (lane == 0) start[a.experts] = before;
  }

  // Width of the tiles, kMaxBN or half as much and so on: what `workers` CTAs or pairs finish first, a wave of tiles taken to cost `cost(width)`. The
  // sums do not depend on it.
  template <typename Cost>
  __device__ __forceinline__ Tiles(const ExpertGemmArgs& args, const int* table, int workers, int narrowest, Cost cost) : a(args), start(table) {
    parts = MODE == EXPERT_FORWARD && a.gated ? 2 : 1;
    const int rowTiles = start[a.experts];
    float best = 0.0f;
    bn = kMaxBN;
    for (int w = kMaxBN; w >= narrowest; w /= 2) {
      const int n = rowTiles * ((a.cols + w / parts - 1) / (w / parts));
      const float all = (n + workers - 1) / workers * cost(w);
      if (w == kMaxBN || all < best) { best = all; bn = w; }
    }
    outCols = bn / parts;
    tilesN = (a.cols + outCols - 1) / outCols;
    count = rowTiles * tilesN;
  }

  // Panels of 8 row tiles: those in flight share both operands. No search where the expert stays, and no division: with both DW over 32 experts of 64 rows, whose
  // tiles are short, took 415 us, without 332. `from`: an expert at or before t's, as that of the tile before.
  __device__ __forceinline__ Tile at(int t, int from) const {
    Tile r;
    int lo = from;
    if (start[lo + 1] * tilesN <= t) {   // the last expert whose tiles begin at or before t
      int hi = a.experts;
      ++lo;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (start[mid] * tilesN <= t) lo = mid;
        else hi = mid;
      }
    }
    r.e = lo;
    r.rows = rowsOf(a, lo);
    const int first = start[lo], mine = start[lo + 1] - first;
    int k = t - first * tilesN, panel = 0;
    if (mine > 8) {
      panel = k / (8 * tilesN);
      k -= panel * 8 * tilesN;
    }
    const int width = min(8, mine - panel * 8), col = width == 1 ? k : (int)__umulhi((uint32_t)k, kInverse[width]);   // k / width
    r.row0 = (panel * 8 + k - col * width) * BM;
    r.col0 = col * outCols;
    r.steps = ((MODE == EXPERT_DW ? r.rows : a.depth) + kBK - 1) / kBK;
    return r;
  }
  __device__ __forceinline__ int rowLimit(const Tile& c) const { return MODE == EXPERT_DW ? a.outRows : c.rows; }
  __device__ __forceinline__ int length(const Tile& c) const { return MODE == EXPERT_DW ? c.rows : a.depth; }
};

__device__ __forceinline__ void reportTimeout(const ExpertGemmArgs& a, uint32_t what) {
  if (a.status && ldRelaxedSys(a.status) == DEV_OK) {
    a.status[1] = WAIT_TILE;
    a.status[2] = what;
    a.status[3] = blockIdx.x;
    __threadfence_system();
    stRelaxedSys(a.status, DEV_TIMEOUT);
  }
}

// 32 lanes x 8 or 16 columns of an accumulator, and the wait for them.
__device__ __forceinline__ void tmemLd(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmemLd(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmemLd(uint32_t taddr, uint32_t (&r)[32]) { tmemLd32(taddr, r); }
template <int N>
__device__ __forceinline__ void tmemLdReady(uint32_t (&r)[N]) {   // nothing that uses them moves in front
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i])::"memory");
}
template <int N>
__device__ __forceinline__ void asFloat(const uint32_t (&r)[N], float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __uint_as_float(r[i]);
}
// v += N neighbouring bf16.
template <int N>
__device__ __forceinline__ void addBf16(const uint4 (&q)[N / 8], float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N / 8; ++j) {
    float f[8];
    unpackBf16x8(q[j], f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[j * 8 + i] += f[i];
  }
}
// A tile's bias, eight columns to a lane, fetched before the sums are complete: from memory (or level 2) for every step it took longer than the step. All lanes
// ask for the same columns.
struct TileBias {
  uint4 q[2];
  __device__ __forceinline__ void load(const __nv_bfloat16* bias, int cols, int parts, int end, int lane) {
    q[0] = q[1] = make_uint4(0, 0, 0, 0);
    if (lane * 8 < end) {
      q[0] = *(const uint4*)(bias + lane * 8);
      if (parts == 2) q[1] = *(const uint4*)(bias + cols + lane * 8);
    }
  }
  __device__ __forceinline__ uint4 at(int part, int col) const {
    const uint4 m = part ? q[1] : q[0];
    const int from = col / 8;
    return make_uint4(__shfl_sync(~0u, m.x, from), __shfl_sync(~0u, m.y, from), __shfl_sync(~0u, m.z, from), __shfl_sync(~0u, m.w, from));
  }
};
// 16 neighbouring columns of one row, 8 or 16 of them inside the matrix.
__device__ __forceinline__ void storeRow16(__nv_bfloat16* to, const float (&v)[16], bool both, bool wide) {
  const uint4 lo = packBf16x8(v), hi = packBf16x8(v + 8);
  if (wide) {
    st32(to, Pack32{lo, hi});
  } else {
    *(uint4*)to = lo;
    if (both) *(uint4*)(to + 8) = hi;
  }
}

// The same in fp32.
__device__ __forceinline__ void storeRow16(float* to, const float (&v)[16], bool both, bool wide) {
  uint4 q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
  if (wide) {
    st32(to, Pack32{q[0], q[1]});
    st32(to + 8, Pack32{q[2], q[3]});
  } else {
    ((uint4*)to)[0] = q[0];
    ((uint4*)to)[1] = q[1];
    if (both) {
      ((uint4*)to)[2] = q[2];
      ((uint4*)to)[3] = q[3];
    }
  }
}

// Epilogues take an accumulator in small steps in a loop that is not unrolled: each warp passes this code once per tile, and straight through 32 or 64
// columns it did so at the pace at which instructions can be fetched (64 experts of 50 rows, 5000 x 184 with bias and residual: 186 us unrolled, 168 so; 64 of 200, 6656 x
// 432, geglu and bias: 222 and 207).

// Epilogue of one warp for its 32 rows, `row` the first of them, and every other 32 columns of the tile: tBase is the tensor-memory address of the
// warp's first lane and the tile's first column. A lane has a row of the accumulator and stores 16 of its columns at a time, whole sectors straight from
// registers: shared memory is busy with the operands, and its room makes a seventh stage (32 experts of 64 rows, 4096 x 7168: 295 us through shared memory, 285 so).
template <int MODE, typename T, typename Ready>
__device__ __forceinline__ bool storeTile(const ExpertGemmArgs& a, const T& tiles, const Tile& c, int row, uint32_t tBase, int half, int lane, Ready ready) {
  const int parts = tiles.parts, outCols = tiles.outCols;
  const bool mine = row + lane < c.rows;
  const size_t at = ((size_t)c.e * a.cap + row + lane) * a.cols + c.col0;
  const int end = row < c.rows ? min(outCols, a.cols - c.col0) : 0;
  TileBias bias;
  if (MODE == EXPERT_FORWARD && a.bias) bias.load((const __nv_bfloat16*)a.bias + (size_t)c.e * parts * a.cols + c.col0, a.cols, parts, end, lane);
  // the residual of a lane's next columns, on its way while the sums are completed and the columns before are stored (64 experts of 50 rows, 5000 x 184, with a bias: 88 us, read where
  // it is added 96)
  uint4 residual[2];
  auto fetch = [&](int cc) {
    if (MODE != EXPERT_FORWARD || !a.residual || !mine) return;
    const uint4* from = (const uint4*)((const __nv_bfloat16*)a.residual + at + cc);
    residual[0] = cc < end ? from[0] : make_uint4(0, 0, 0, 0);
    residual[1] = cc + 8 < end ? from[1] : make_uint4(0, 0, 0, 0);
  };
  fetch(half * 32);
  if (!ready()) return false;
  if (MODE != EXPERT_FORWARD || (a.act == ACT_NONE && !a.bias && !a.pre && !a.residual)) {
    // the sums as they are: 32 at a time (64 experts of 50 rows, 4992 x 184: 55 us, 63 by the loop below)
#pragma unroll 1
    for (int cc = half * 32; cc < end; cc += 64) {
      uint32_t r[32];
      tmemLd(tBase + cc, r);
      tmemLdReady(r);
#pragma unroll
      for (int j = 0; j < 32; j += 16) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[j + i]);
        if (mine && cc + j < end) storeRow16((__nv_bfloat16*)a.out + at + cc + j, v, cc + j + 8 < end, a.wide);
      }
      __syncwarp();   // together again for the next load from tensor memory
    }
    return true;
  }
#pragma unroll 1
  for (int cc = half * 32, next; cc < end; cc = next) {
    next = cc + (cc & 16 ? 48 : 16);
    const bool both = cc + 8 < end;   // (columns come in eights)
    uint32_t r[16];
    float v[16], u[16];
    auto sums = [&](int part, float (&to)[16]) {
      tmemLd(tBase + part * outCols + cc, r);
      tmemLdReady(r);
      asFloat(r, to);
      if (MODE == EXPERT_FORWARD && a.bias) {
        const uint4 add[2] = {bias.at(part, cc), bias.at(part, cc + 8)};
        addBf16<16>(add, to);
      }
      if (MODE == EXPERT_FORWARD && a.pre) {
        const size_t o = (at - c.col0) * parts + part * a.cols + c.col0 + cc;
        if (mine && a.preFp32) storeRow16((float*)a.pre + o, to, both, a.wide);
        if (mine && !a.preFp32) storeRow16((__nv_bfloat16*)a.pre + o, to, both, a.wide);
        __syncwarp();
      }
    };
    sums(0, v);
    if (MODE == EXPERT_FORWARD) {
      if (parts == 2) sums(1, u);
      activateAll<16>(a.act, v, u);
      if (a.residual && mine) {
        addBf16<16>(residual, v);
        fetch(next);
      }
    }
    if (mine) storeRow16((__nv_bfloat16*)a.out + at + cc, v, both, a.wide);
    __syncwarp();
  }
  return true;
}

// The same through shared memory: 64 columns of 32 rows at a time pass 4 KiB (16-byte chunks XOR-swizzled by row), so that memory sees 128 contiguous bytes of a
// row. For DW, whose results are the traffic: 32 experts of 64 rows, 4096 x 7168, 431 us, with the stores above 501, with bulk copies from shared memory
// 609 (332 us since, 5.7 TB/s written; the framework's fill of the same memory takes 474). And where a lane's own row would be touched 16 bytes at a time, 32 lines by an
// instruction (residual, rows that are not whole packs of 32 bytes): 64 experts of about 140 rows, 2056 x 1400 with a residual, 153 and 145 us.
template <int MODE, typename T, typename Ready>
__device__ __forceinline__ bool storeTileStaged(const ExpertGemmArgs& a, const T& tiles, const Tile& c, int row, uint32_t tBase, uint8_t* wbuf, int half, int lane, Ready ready) {
  const int parts = tiles.parts, outCols = tiles.outCols, left = tiles.rowLimit(c) - row;   // rows from here on
  const size_t first = (size_t)c.e * (MODE == EXPERT_DW ? a.outRows : a.cap) + row;
  const int end = left > 0 ? min(outCols, a.cols - c.col0) : 0;
  TileBias bias;
  if (MODE == EXPERT_FORWARD && a.bias) bias.load((const __nv_bfloat16*)a.bias + (size_t)c.e * parts * a.cols + c.col0, a.cols, parts, end, lane);
  auto chunk = [&](int r, int j) { return (uint4*)(wbuf + r * 128 + ((j ^ (r & 7)) * 16)); };
  const int mine = lane >> 3, j0 = lane & 7;   // of four rows, and of a row's eight chunks
  const bool plain = a.act == ACT_NONE && !a.bias && !a.residual;
  uint4 residual[8];
  auto fetch = [&](int cc) {
    if (MODE != EXPERT_FORWARD || !a.residual) return;
    const __nv_bfloat16* from = (const __nv_bfloat16*)a.residual + (first + mine) * a.cols + c.col0 + cc + j0 * 8;
#pragma unroll
    for (int k = 0; k < 8; ++k) residual[k] = cc + j0 * 8 < end && k * 4 + mine < left ? *(const uint4*)(from + (size_t)(k * 4) * a.cols) : make_uint4(0, 0, 0, 0);
  };
  fetch(half * 64);
  if (!ready()) return false;
#pragma unroll 1
  for (int cc = half * 64; cc < end; cc += 128) {
    const int width = min(64, end - cc), col = c.col0 + cc;   // a multiple of 8
    auto store = [&](auto* to, size_t ld, int columns) {
      constexpr int kPer = 16 / sizeof(*to);   // of a chunk
      __syncwarp();
      to += mine * ld + j0 * kPer;
#pragma unroll
      for (int k = 0; k < 8; ++k, to += 4 * ld)
        if (k * 4 + mine < left && j0 * kPer < columns) *(uint4*)to = *chunk(k * 4 + mine, j0);
      __syncwarp();
    };
    auto sums = [&](int part, int at, float (&v)[8]) {
      uint32_t r[8];
      tmemLd(tBase + part * outCols + cc + at, r);
      tmemLdReady(r);
      asFloat(r, v);
      if (a.bias) {
        const uint4 add[1] = {bias.at(part, cc + at)};
        addBf16<8>(add, v);
      }
    };
    if (MODE == EXPERT_FORWARD && a.pre) {
#pragma unroll 1
      for (int p = 0; p < parts; ++p) {
        const size_t o = (first * parts + p) * a.cols + col;
#pragma unroll 1
        for (int at = 0; at < width; at += 8) {
          float v[8];
          sums(p, at, v);
          if (!a.preFp32) {
            *chunk(lane, at / 8) = packBf16x8(v);
          } else {   // 32 columns fill a row
#pragma unroll
            for (int i = 0; i < 2; ++i)
              *chunk(lane, at / 4 % 8 + i) = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
            if (at % 32 == 24 || at + 8 == width) store((float*)a.pre + o + at / 32 * 32, (size_t)parts * a.cols, at % 32 + 8);
          }
        }
        if (!a.preFp32) store((__nv_bfloat16*)a.pre + o, (size_t)parts * a.cols, width);
      }
    }
    if (MODE == EXPERT_FORWARD && a.residual) {
#pragma unroll
      for (int k = 0; k < 8; ++k) *chunk(k * 4 + mine, j0) = residual[k];
      __syncwarp();
      fetch(cc + 128);
    }
    if (MODE == EXPERT_FORWARD && !plain) {
#pragma unroll 1
      for (int at = 0; at < width; at += 8) {
        float v[8], u[8];
        sums(0, at, v);
        if (parts == 2) sums(1, at, u);
        activateAll<8>(a.act, v, u);
        if (a.residual) {
          const uint4 add[1] = {*chunk(lane, at / 8)};
          addBf16<8>(add, v);
        }
        *chunk(lane, at / 8) = packBf16x8(v);
      }
    } else {   // the sums as they are: 32 at a time
#pragma unroll
      for (int at = 0; at < 64; at += 32) {
        if (at >= width) break;
        uint32_t r[32] = {};
        if (MODE != EXPERT_DW || c.steps) {
          tmemLd(tBase + cc + at, r);
          tmemLdReady(r);
        }
        float v[32];
        asFloat(r, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) *chunk(lane, at / 8 + j) = packBf16x8(v + j * 8);
      }
    }
    store((__nv_bfloat16*)a.out + first * a.cols + col, (size_t)a.cols, width);
  }
  return true;
}

}  // namespace

// ---------------------------------------------------------------------------------------------- one CTA per tile of 128 rows
// No expert has more rows than one tile (cap <= 128): FORWARD and DX. tmA has boxes of 32 rows (of fewer, if cap is less), of which those that hold rows are fetched. tmB has
// boxes of 128 rows of W (DX: 64 x 64), tmBNarrow of 32 (gated: 64) for narrow tiles: one or two boxes make a tile.
template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
expertGemmKernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmBNarrow,
                 const __grid_constant__ ExpertGemmArgs a) {
  static_assert(MODE != EXPERT_DW, "DW runs on pairs");
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smemRaw + 1023) & ~(uintptr_t)1023);
  uint8_t* ctrl = smem + kRingBytes;
  uint64_t* fullBar = (uint64_t*)ctrl;              // [kMaxStages]
  uint64_t* emptyBar = fullBar + kMaxStages;        // [kMaxStages]
  uint64_t* accFull = emptyBar + kMaxStages;        // [2]
  uint64_t* accEmpty = accFull + 2;                 // [2]
  uint32_t* tmemSlot = (uint32_t*)(accEmpty + 2);
  volatile uint32_t* abortFlag = tmemSlot + 1;
  int* table = (int*)(ctrl + kCtrlBytes);

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
  if (warp == 0) Tiles<MODE, 128>::fill(a, table, lane);
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  const uint32_t tmemBase = *tmemSlot;
  // us of a step, where the weights come as fast as they are used. Wide tiles: 32 experts of 16 rows, 4096 x 7168 gated, 256 columns 299 us, 128 373; two
  // experts of one row, 28672 x 4096 80 and 126. Narrow ones where they would leave SMs idle: 4096 x 14336 87, 79 and (64) 52 us
  const Tiles<MODE, 128> tiles(a, table, gridDim.x, MODE != EXPERT_FORWARD ? 64 : a.gated ? 128 : 32,
                               [](int w) { return w == 256 ? 0.33f : w == 128 ? 0.27f : w == 64 ? 0.23f : 0.2f; });
  const int bn = tiles.bn, parts = tiles.parts, outCols = tiles.outCols;
  const bool narrow = MODE == EXPERT_FORWARD && outCols <= 64;
  const int boxRows = MODE != EXPERT_FORWARD ? 64 : !narrow ? 128 : parts == 2 ? 64 : 32, boxes = bn / boxRows;
  const uint32_t aBytes = (uint32_t)((a.cap + 31) / 32 * a.boxRows) * 128, stageBytes = aBytes + (uint32_t)bn * 128;
  const int stages = (int)min((uint32_t)kMaxStages, kRingBytes / stageBytes);
  const uint32_t ring = smemAddr(smem);
  auto fail = [&](uint32_t what) {
    *abortFlag = 1;
    reportTimeout(a, what);
  };

  if (warp == 0) {
    if (electOne()) {
      // one thread feeds the ring: what a step takes here is what the others wait for, so addresses are counted on and not computed
      const uint32_t bars = smemAddr(fullBar), toEmpty = smemAddr(emptyBar) - bars, stride = boxRows * 128;
      uint32_t phase = 0, sA = ring, bar = bars;
      const uint32_t ringEnd = ring + stages * stageBytes;
      bool whole = false;   // every stage was loaded once
      int at = 0;   // expert of the tile before
      for (int t = blockIdx.x; t < tiles.count && !*abortFlag; t += gridDim.x) {
        const Tile c = tiles.at(t, at);
        at = c.e;
        const int second = c.col0 + (parts == 2 ? a.cols : boxRows);   // row of W in a tile's second box
        const int aBoxes = (c.rows + 31) / 32, end = c.steps * kBK;
        const uint32_t bytes = (uint32_t)(aBoxes * a.boxRows + bn) * 128;
        for (int x = 0; x < end; x += kBK) {
          if (!waitOr(bar + toEmpty, phase ^ 1, abortFlag)) { fail(1000); break; }
          mbarExpectTx(bar, bytes);
          tmaLoad3d(sA, &tmA, x, 0, c.e, bar);
          if (aBoxes > 1)
            for (int i = 1; i < aBoxes; ++i) tmaLoad3d(sA + i * 32 * 128, &tmA, x, i * 32, c.e, bar);
          const uint32_t sB = sA + aBytes;
          if (MODE != EXPERT_FORWARD) {
            for (int i = 0; i < boxes; ++i) tmaLoad3d(sB + i * kBlockBytes, &tmB, c.col0 + i * 64, x, c.e, bar);
          } else if (!narrow) {
            tmaLoad3d(sB, &tmB, x, c.col0, c.e, bar);
            if (boxes == 2) tmaLoad3d(sB + stride, &tmB, x, second, c.e, bar);
          } else {
            tmaLoad3d(sB, &tmBNarrow, x, c.col0, c.e, bar);
            if (boxes == 2) tmaLoad3d(sB + stride, &tmBNarrow, x, second, c.e, bar);
          }
          sA += stageBytes;
          bar += 8;
          if (sA == ringEnd) { sA = ring; bar = bars; phase ^= 1; whole = true; }
        }
      }
      if (*abortFlag) {
        // copies already issued still write into shared memory: wait for them (bounded). Stages in front of the next one were loaded in this round, the others in the one before
        for (uint32_t i = bars; i < bars + stages * 8; i += 8)
          if (whole || i < bar) mbarWait(i, i < bar ? phase : phase ^ 1, 1u << 20);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (electOne()) {
      const uint32_t idesc = umInstrBf16(128, bn) | (kAcrossB<MODE> ? 1u << 16 : 0u);
      int s = 0, it = 0;
      uint32_t phase = 0;
      bool bad = false;
      int at = 0;   // expert of the tile before
      for (int t = blockIdx.x; t < tiles.count && !bad && !*abortFlag; t += gridDim.x, ++it) {
        const Tile c = tiles.at(t, at);
        at = c.e;
        const int buf = it & 1;
        if (!waitOr(smemAddr(&accEmpty[buf]), ((it >> 1) & 1) ^ 1, abortFlag)) { fail(2000 + buf); break; }
        tcFenceAfter();
        const uint32_t dT = tmemBase + buf * kAccCols;
        for (int kb = 0; kb < c.steps; ++kb) {
          if (!waitOr(smemAddr(&fullBar[s]), phase, abortFlag)) { fail(3000 + s); bad = true; break; }
          tcFenceAfter();
          const uint32_t sA = ring + s * stageBytes, sB = sA + aBytes;
          const uint64_t da = umDescK128(sA), db = descOf<kAcrossB<MODE>>(sB);
#pragma unroll
          for (int k = 0; k < kBK / kUmmaK; ++k)   // (behind the sum's end are zeros)
            ummaBf16(dT, da + k * kNextDesc<false>, db + k * kNextDesc<kAcrossB<MODE>>, idesc, (kb | k) != 0);
          ummaCommit(smemAddr(&emptyBar[s]));
          if (++s == stages) { s = 0; phase ^= 1; }
        }
        if (!bad) ummaCommit(smemAddr(&accFull[buf]));
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, half = (warp - kFirstEpiWarp) >> 2;   // TMEM lanes [32q, 32q+32) belong to the warps with warp % 4 == q
    int it = 0;
    int at = 0;   // expert of the tile before
    for (int t = blockIdx.x; t < tiles.count && !__any_sync(~0u, *abortFlag); t += gridDim.x, ++it) {
      const Tile c = tiles.at(t, at);
      at = c.e;
      const int buf = it & 1;
      auto ready = [&] {
        const bool ok = warpWaitOr(smemAddr(&accFull[buf]), (it >> 1) & 1, abortFlag, lane);
        tcFenceAfter();
        return ok;
      };
      if (!storeTile<MODE>(a, tiles, c, q * 32, tmemBase + ((uint32_t)(q * 32) << 16) + buf * kAccCols, half, lane, ready)) { if (lane == 0) fail(4000 + buf); break; }
      tcFenceBefore();
      __syncwarp();
      if (lane == 0) mbarArrive(smemAddr(&accEmpty[buf]));
    }
  }

  tcFenceBefore();
  __syncthreads();
  if (*abortFlag) letThemLand();
  if (warp == 1) {
    tcFenceAfter();
    tmemDealloc(tmemBase, kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------- CTA pairs, tiles of 256 rows
// FORWARD: tmB has boxes of 128 rows of W, tmBNarrow of 64, half the width of a tile each; else tmB has boxes of 64 x 64.
//   fullBar[s]   (the first CTA's copy) counts the bytes of both CTAs' loads of ring stage s;
//   emptyBar[s]  in each CTA: a commit that signals both frees the stage;
//   accFull[b]   in each CTA: the same publishes accumulator b to both epilogues;
//   accEmpty[b]  (the first CTA's copy) collects the epilogue warps of both;
//   tailBar[s]   DW, in each CTA: the bytes of its own loads of a stage whose last rows are to be zeroed;
//   fixBar[s]    (the first CTA's copy) the other CTA has written its zeros; the first CTA's warp for that arrives at fullBar then, in the
//                producer's place. (An arrival of both producers in every step, so that fullBar could count two, took half of DW's rate.)
template <int MODE, bool STAGED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
expertGemmPairKernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmBNarrow,
                     const __grid_constant__ ExpertGemmArgs a) {
  constexpr uint32_t kStageBytes = 2 * kHalfBytes;
  constexpr int kPairStages = STAGED ? 6 : 7;   // an epilogue through shared memory takes the room of the seventh
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smemRaw + 1023) & ~(uintptr_t)1023);
  uint8_t* ctrl = smem + kRingBytes;
  uint64_t* fullBar = (uint64_t*)ctrl;              // [kPairStages]
  uint64_t* emptyBar = fullBar + kPairStages;       // [kPairStages]
  uint64_t* tailBar = emptyBar + kPairStages;       // [kPairStages]
  uint64_t* fixBar = tailBar + kPairStages;         // [kPairStages]
  uint64_t* accFull = fixBar + kPairStages;         // [2]
  uint64_t* accEmpty = accFull + 2;                 // [2]
  uint32_t* tmemSlot = (uint32_t*)(accEmpty + 2);
  volatile uint32_t* abortFlag = tmemSlot + 1;
  int* table = (int*)(ctrl + kCtrlBytes);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cr = clusterCtaRank();
  const bool leader = cr == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      for (uint64_t* b : {fullBar, emptyBar, tailBar, fixBar}) mbarInit(smemAddr(&b[s]), 1);
    }
    for (int b = 0; b < 2; ++b) { mbarInit(smemAddr(&accFull[b]), 1); mbarInit(smemAddr(&accEmpty[b]), 2 * kEpiWarps); }
    *abortFlag = 0;
    mbarInitFence();
    prefetchTensorMap(&tmA);
    prefetchTensorMap(&tmB);
  }
  if (warp == 1) {
    tmemAllocPair(smemAddr(tmemSlot), kTmemCols);
    tmemRelinquishPair();
  }
  pdlEnter();   // the set-up above overlaps the end of the kernel before
  if (warp == 0) Tiles<MODE, 256>::fill(a, table, lane);
  tcFenceBefore();
  __syncthreads();
  __syncwarp();
  clusterSync();   // both CTAs' barriers are initialised before either signals the other's
  tcFenceAfter();
  const uint32_t tmemBase = *tmemSlot;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  // us of a step. Half as wide a tile fetches three quarters as much: it pays where whole ones would leave most of the SMs idle
  const Tiles<MODE, 256> tiles(a, table, pairs, 128, [](int w) { return w == 256 ? 0.35f : 0.22f; });
  const int bn = tiles.bn, parts = tiles.parts, halfCols = bn / 2;   // columns that each CTA stages
  const uint32_t ring = smemAddr(smem);
  auto fail = [&](uint32_t what) {
    *abortFlag = 1;
    stSharedCluster(mapaShared(smemAddr((const void*)abortFlag), cr ^ 1), 1u);   // the partner gives up too
    reportTimeout(a, what);
  };
  // Rows of this CTA's half of the first operand in use (DW: of the result), and its first row or column of the second
  auto rowsIn = [&](const Tile& c, int rank) { return min(128, tiles.rowLimit(c) - c.row0 - rank * 128); };
  auto firstB = [&](const Tile& c) { return parts == 2 ? (int)cr * a.cols + c.col0 : c.col0 + (int)cr * halfCols; };
  auto colsIn = [&](const Tile& c, int rank) { return parts == 2 ? min(halfCols, a.cols - c.col0) : min(halfCols, a.cols - c.col0 - rank * halfCols); };
  // Bytes that CTA `rank` loads for a step: nothing of an operand where it has no row or column. With neither it still loads a box from behind the matrix (zeros, no
  // traffic): what keeps a CTA within one round of the ring of its partner is that no step is complete without its bytes.
  auto bytesA = [&](const Tile& c, int rank) {
    const int n = rowsIn(c, rank);
    return n <= 0 ? 0u : kAcrossA<MODE> && n <= 64 ? kBlockBytes : kHalfBytes;
  };
  auto bytesB = [&](const Tile& c, int rank) {
    const int n = colsIn(c, rank);
    return n <= 0 && rowsIn(c, rank) > 0 ? 0u : !kAcrossB<MODE> ? (uint32_t)halfCols * 128 : n <= 64 ? kBlockBytes : kHalfBytes;
  };

  if (warp == 0) {
    if (electOne()) {
      const uint32_t bars = smemAddr(fullBar), toEmpty = smemAddr(emptyBar) - bars, toTail = smemAddr(tailBar) - bars;
      const uint32_t toLeader = mapaShared(bars, 0) - bars, toOwn = mapaShared(bars, cr) - bars;   // cluster addresses of the barriers
      const uint32_t ringEnd = ring + kPairStages * kStageBytes;
      uint32_t phase = 0, sA = ring, bar = bars, tails = 0, tailPhase = 0;   // bit s: the last load of stage s counts on tailBar, and the phase of that
      bool whole = false;                                                    // every stage was loaded once
      int at = 0;   // expert of the tile before
      for (int t = pair; t < tiles.count && !*abortFlag; t += pairs) {
        const Tile c = tiles.at(t, at);
        at = c.e;
        const uint32_t mineA = bytesA(c, cr), mineB = bytesB(c, cr), both = bytesA(c, 0) + bytesA(c, 1) + bytesB(c, 0) + bytesB(c, 1);
        const int row = c.row0 + (int)cr * 128, col = firstB(c), end = c.steps * kBK;
        const int tailAt = MODE == EXPERT_DW && c.rows % kUmmaK != 0 ? end - kBK : -1;
        for (int x = 0; x < end; x += kBK) {
          if (!waitOr(bar + toEmpty, phase ^ 1, abortFlag)) { fail(1000); break; }
          const uint32_t sB = sA + kHalfBytes;
          uint32_t full = bar + toLeader;
          if (MODE == EXPERT_DW && x == tailAt) {
            full = bar + toTail + toOwn;
            mbarExpectTx(bar + toTail, mineA + mineB);
            tails |= 1u << (bar - bars) / 8;
            tailPhase ^= 1u << (bar - bars) / 8;
          } else {
            if (leader) mbarExpectTx(bar, both);
            if (MODE == EXPERT_DW) tails &= ~(1u << (bar - bars) / 8);
          }
          if (kAcrossA<MODE>) {
            if (mineA) tmaLoad3dPair(sA, &tmA, row, x, c.e, full);
            if (mineA > kBlockBytes) tmaLoad3dPair(sA + kBlockBytes, &tmA, row + 64, x, c.e, full);
          } else if (mineA) {
            tmaLoad3dPair(sA, &tmA, x, row, c.e, full);
          }
          if (kAcrossB<MODE>) {
            if (mineB) tmaLoad3dPair(sB, &tmB, col, x, c.e, full);
            if (mineB > kBlockBytes) tmaLoad3dPair(sB + kBlockBytes, &tmB, col + 64, x, c.e, full);
          } else if (mineB) {
            if (bn == 256) tmaLoad3dPair(sB, &tmB, x, col, c.e, full);
            else tmaLoad3dPair(sB, &tmBNarrow, x, col, c.e, full);
          }
          sA += kStageBytes;
          bar += 8;
          if (sA == ringEnd) { sA = ring; bar = bars; phase ^= 1; whole = true; }
        }
      }
      if (*abortFlag) {
        // copies already issued (by either CTA) still write into shared memory: wait for them (bounded). Stages in front of the next one were loaded in this round
        for (int i = 0; i < kPairStages; ++i) {
          const uint32_t at = bars + i * 8;
          if (!whole && at >= bar) break;
          if (tails >> i & 1) mbarWait(at + toTail, (tailPhase >> i & 1) ^ 1, 1u << 20);
          else if (leader) mbarWait(at, at < bar ? phase : phase ^ 1, 1u << 20);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (MODE != EXPERT_FORWARD && !leader && a.partial) biasFromSlices(a.partial, (__nv_bfloat16*)a.dbias, a.sums, a.slices, (size_t)pair * 32 + lane, (size_t)pairs * 32);
    if (leader && electOne()) {
      const uint32_t idesc = umInstrBf16(256, bn) | (kAcrossA<MODE> ? 1u << 15 : 0u) | (kAcrossB<MODE> ? 1u << 16 : 0u);
      int s = 0, it = 0;
      uint32_t phase = 0;
      bool bad = false;
      int at = 0;   // expert of the tile before
      for (int t = pair; t < tiles.count && !bad && !*abortFlag; t += pairs) {
        const Tile c = tiles.at(t, at);
        at = c.e;
        if (c.steps == 0) continue;   // nothing to add up: the epilogue writes zeros
        const int buf = it & 1;
        if (!waitOr(smemAddr(&accEmpty[buf]), ((it >> 1) & 1) ^ 1, abortFlag)) { fail(2000 + buf); break; }
        ++it;
        tcFenceAfter();
        const uint32_t dT = tmemBase + buf * kAccCols;
        const int last = (tiles.length(c) - (c.steps - 1) * kBK + kUmmaK - 1) / kUmmaK;   // sixteens in the last step
        for (int kb = 0; kb < c.steps; ++kb) {
          if (!waitOr(smemAddr(&fullBar[s]), phase, abortFlag)) { fail(3000 + s); bad = true; break; }
          tcFenceAfter();
          const uint32_t sA = ring + s * kStageBytes;
          const uint64_t da = descOf<kAcrossA<MODE>>(sA), db = descOf<kAcrossB<MODE>>(sA + kHalfBytes);
          const int chunks = kb == c.steps - 1 ? last : kBK / kUmmaK;
#pragma unroll
          for (int k = 0; k < kBK / kUmmaK; ++k)
            if (k < chunks) ummaBf16Pair(dT, da + k * kNextDesc<kAcrossA<MODE>>, db + k * kNextDesc<kAcrossB<MODE>>, idesc, (kb | k) != 0);
          ummaCommitPair(smemAddr(&emptyBar[s]), 3);
          if (++s == kPairStages) { s = 0; phase ^= 1; }
        }
        if (!bad) ummaCommitPair(smemAddr(&accFull[buf]), 3);
      }
    }
    __syncwarp();
  } else if (warp < kFixWarp) {
    const int q = warp & 3, half = (warp - kFirstEpiWarp) >> 2;   // TMEM lanes [32q, 32q+32) belong to the warps with warp % 4 == q
    int it = 0;
    int at = 0;   // expert of the tile before
    for (int t = pair; t < tiles.count && !__any_sync(~0u, *abortFlag); t += pairs) {
      const Tile c = tiles.at(t, at);
      at = c.e;
      const int buf = it & 1;
      const int row = c.row0 + (int)cr * 128 + q * 32;
      const uint32_t tBase = tmemBase + ((uint32_t)(q * 32) << 16) + buf * kAccCols;
      auto ready = [&] {   // (nothing to wait for where there was nothing to add up)
        const bool ok = c.steps == 0 || warpWaitOr(smemAddr(&accFull[buf]), (it >> 1) & 1, abortFlag, lane);
        tcFenceAfter();
        return ok;
      };
      bool ok;
      if constexpr (STAGED) ok = storeTileStaged<MODE>(a, tiles, c, row, tBase, smem + 6 * kStageBytes + (warp - kFirstEpiWarp) * 4096, half, lane, ready);
      else ok = storeTile<MODE>(a, tiles, c, row, tBase, half, lane, ready);
      if (!ok) { if (lane == 0) fail(4000 + buf); break; }
      if (c.steps) {
        ++it;
        tcFenceBefore();
        __syncwarp();
        if (lane == 0) mbarArriveRelaxed(mapaShared(smemAddr(&accEmpty[buf]), 0));
      }
    }
  } else if (MODE == EXPERT_DW) {
    // rows behind the expert's last are somebody's old values: zeros up to the next sixteen, so that they add nothing (a row is 128 bytes of every box)
    int done = 0;   // steps of the tiles before
    uint32_t phases = 0, since = 1;   // tiles since the last one that had such rows
    int at = 0;   // expert of the tile before
    for (int t = pair; t < tiles.count && !__any_sync(~0u, *abortFlag); t += pairs) {
      const Tile c = tiles.at(t, at);
      at = c.e;
      if (c.steps == 0) continue;
      const int s = (done + c.steps - 1) % kPairStages, rows = (kUmmaK - c.rows % kUmmaK) % kUmmaK;
      done = (done + c.steps) % kPairStages;
      if (rows == 0) {
        ++since;
        continue;
      }
      const uint32_t parity = phases >> s & 1;
      phases ^= 1u << s;
      // (all lanes ask: a step waits for this warp, and one lane that tells the others costs 32 experts of 61 rows, 4096 x 7168, 4 %)
      if (!__all_sync(~0u, waitOr(smemAddr(&tailBar[s]), parity, abortFlag, since))) { if (lane == 0) fail(5000 + s); break; }
      since = 1;
      const int from = c.rows - (c.steps - 1) * kBK;
      for (int i = lane; i < 4 * rows * 8; i += 32) {
        const int box = i / (rows * 8), r = i / 8 % rows;
        *(uint4*)(smem + (size_t)s * kStageBytes + box * kBlockBytes + (from + r) * 128 + i % 8 * 16) = make_uint4(0, 0, 0, 0);
      }
      fenceProxyAsync();
      __syncwarp();
      if (!leader) {
        if (lane == 0) mbarArriveCluster(mapaShared(smemAddr(&fixBar[s]), 0));
      } else {
        if (!__all_sync(~0u, waitClusterOr(smemAddr(&fixBar[s]), parity, abortFlag))) { if (lane == 0) fail(6000 + s); break; }
        if (lane == 0) mbarArrive(smemAddr(&fullBar[s]));
      }
    }
  }

  // the pair meets: nobody touches the partner's shared or tensor memory afterwards
  tcFenceBefore();
  __syncthreads();
  if (*abortFlag) letThemLand();
  __syncwarp();
  clusterSync();
  if (warp == 1) {
    tcFenceAfter();
    tmemDeallocPair(tmemBase, kTmemCols);
  }
}

const void* expertGemmKernelFn(int mode) { return mode == EXPERT_DX ? (const void*)expertGemmKernel<EXPERT_DX> : (const void*)expertGemmKernel<EXPERT_FORWARD>; }
const void* expertGemmPairKernelFn(int mode, bool staged) {
  if (mode == EXPERT_DW) return (const void*)expertGemmPairKernel<EXPERT_DW, true>;
  if (mode == EXPERT_DX) return staged ? (const void*)expertGemmPairKernel<EXPERT_DX, true> : (const void*)expertGemmPairKernel<EXPERT_DX, false>;
  return staged ? (const void*)expertGemmPairKernel<EXPERT_FORWARD, true> : (const void*)expertGemmPairKernel<EXPERT_FORWARD, false>;
}
size_t expertGemmSmemBytes() { return kSmemBytes; }
int expertGemmThreads(bool pair) { return pair ? kPairThreads : kThreads; }

}  // namespace b200
