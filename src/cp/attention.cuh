// Building blocks of the attention kernels: tiles of 128 rows, tcgen05 products with an operand in tensor memory, bounded waits, exponentials.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../kernels/common.cuh"
#include "../tp/gemm_sm100.cuh"
#include "cp.h"

namespace b200 {
namespace attn {

using namespace sm100;

// Warps of a CTA: those that hold rows, then the producer, the issuer of products and two without a role (registers are dealt out to groups of four warps: they move
// from the last group to those that hold rows).
template <int COMPUTE, int LAUNCH, int FEW, int MANY> struct Warps {
  static constexpr int kCompute = COMPUTE, kProducer = COMPUTE, kMma = COMPUTE + 1, kThreads = (COMPUTE + 4) * 32, kLaunchRegs = LAUNCH, kFewRegs = FEW, kManyRegs = MANY;
  static_assert(COMPUTE % 4 == 0 && COMPUTE * MANY + 4 * FEW <= (COMPUTE + 4) * LAUNCH && (COMPUTE + 4) * 32 * LAUNCH <= 65536, "registers");
};
using ForwardWarps = Warps<8, 168, 80, 208>;
using BackwardWarps = Warps<8, 168, 80, 208>;
constexpr uint32_t kHalfTile = 128 * 128;          // bytes of 128 rows x 64 channels
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// ---------------------------------------------------------------- types
template <typename T> struct Pack;
template <> struct Pack<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1;
  // Unnormalised probabilities may be multiplied by a power of two that keeps small ones of 16 bits normal numbers; bf16 has fp32's range.
  static constexpr float kForwardBias = 0.0f, kBackwardBias = 0.0f;
  __device__ static __forceinline__ uint32_t two(float a, float b) { __nv_bfloat162 v = __floats2bfloat162_rn(a, b); return *(uint32_t*)&v; }
  __device__ static __forceinline__ float2 both(uint32_t u) { return __bfloat1622float2(*(__nv_bfloat162*)&u); }
};
template <> struct Pack<__half> {
  static constexpr uint32_t kFormat = 0;
  // forward: at most 2^8 (the maximum lags by up to that), times 2^7; backward: at most 1 (and a rounding more), times 2^15
  static constexpr float kForwardBias = 7.0f, kBackwardBias = 15.0f;
  __device__ static __forceinline__ uint32_t two(float a, float b) { __half2 v = __floats2half2_rn(a, b); return *(uint32_t*)&v; }
  __device__ static __forceinline__ float2 both(uint32_t u) { return __half22float2(*(__half2*)&u); }
};

// What rounding two numbers to 16 bits left, in 16 bits.
template <typename T>
__device__ __forceinline__ uint32_t remainderOf(uint32_t rounded, float a, float b) {
  const float2 r = Pack<T>::both(rounded);
  return Pack<T>::two(a - r.x, b - r.y);
}

// kind::f16, fp32 sums; B along the sum (K-major) or across it.
template <typename T> constexpr uint32_t instr(int N, bool acrossB) {
  return (1u << 4) | (Pack<T>::kFormat << 7) | (Pack<T>::kFormat << 10) | ((acrossB ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((128u >> 4) << 24);
}

// A tile of 128 rows lies in boxes of 128 rows x 64 channels with 128-byte swizzle. As an operand whose sum runs over the channels: rows of 128 bytes, the next 8 of them 1024
// bytes on. As one whose sum runs over the rows: the next 64 channels are a box further, the next 8 rows 1024 bytes. The lower word of a descriptor has the address in units of
// 16 bytes (and the leading offset above it), so that steps along the sum add a constant to it; the upper word is the same for all.
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t descAlong(uint32_t addr) { return (addr & 0x3FFFF) >> 4 | 1u << 16; }
__device__ __forceinline__ uint32_t descAcross(uint32_t addr) { return (addr & 0x3FFFF) >> 4 | (kHalfTile >> 4) << 16; }

// The first step of a sum says at run time whether it is added to what is there, the others add.
template <bool FIRST>
__device__ __forceinline__ void mmaSS(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 x, y;\n"
      "setp.ne.b32 p, %5, 0;\n"
      "mov.b64 x, {%1, %4};\n"
      "mov.b64 y, {%2, %4};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(kDescHigh), "n"(FIRST ? 0 : 1) : "memory");
}
__device__ __forceinline__ void mmaTS(uint32_t d, uint32_t aTmem, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 y;\n"
      "setp.ne.b32 p, %5, 0;\n"
      "mov.b64 y, {%2, %4};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}"
      ::"r"(d), "r"(aTmem), "r"(b), "r"(idesc), "r"(kDescHigh), "r"(accumulate) : "memory");
}
// D[128 x N] = A B^T over DP channels of two tiles in shared memory, from the lower words of their descriptors (descAlong).
// AHalf: bytes from A's first 64 channels to the next.
template <typename T, int DP, int N = 128, uint32_t AHalf = kHalfTile>
__device__ __forceinline__ void productOfTiles(uint32_t d, uint32_t a, uint32_t b) {
  mmaSS<true>(d, a, b, instr<T>(N, false));
#pragma unroll
  for (int k = 1; k < DP / 16; ++k) {
    mmaSS<false>(d, a + (((k / 4) * AHalf + (k % 4) * 32) >> 4), b + (((k / 4) * kHalfTile + (k % 4) * 32) >> 4), instr<T>(N, false));
  }
}
// D[128 x DP] (+)= A B with A [128 x 128] in tensor memory, 16 bits a value, columns [0, 64) of the sum at `a`, the others 64 columns on; B (descAcross) 128 rows of DP channels.
template <typename T, int DP>
__device__ __forceinline__ void productWithTmem(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  mmaTS(d, a, b, instr<T>(DP, true), accumulate);
#pragma unroll
  for (int k = 1; k < 8; ++k) mmaTS(d, a + k / 4 * 64 + k % 4 * 8, b + (k * 2048 >> 4), instr<T>(DP, true), 1);
}

// ---------------------------------------------------------------- copies
__device__ __forceinline__ void tmaLoad4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
// A tile of rows from token `tok` on; `head0`: the first head (queries: of the group).
template <int DP>
__device__ __forceinline__ void loadTile(uint32_t dst, const CUtensorMap* map, int tok, int head0, int b, uint32_t bar) {
#pragma unroll
  for (int h = 0; h < DP / 64; ++h) tmaLoad4d(dst + h * kHalfTile, map, h * 64, head0, tok, b, bar);
}
// Rows [from, 128) of a tile become zero, by one warp; ordered in front of the products by a fence and the arrival that follows.
template <int DP>
__device__ __forceinline__ void clearRows(uint8_t* tile, int from, int lane) {
#pragma unroll
  for (int h = 0; h < DP / 64; ++h)
    for (int i = from * 8 + lane; i < 128 * 8; i += 32) *(uint4*)(tile + h * kHalfTile + i * 16) = make_uint4(0, 0, 0, 0);   // (the swizzle stays within a row's 128 bytes)
  fenceProxyAsync();
  __syncwarp();
}

// ---------------------------------------------------------------- tensor memory
__device__ __forceinline__ void tmemSt32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmemStWait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---------------------------------------------------------------- arithmetic
__device__ __forceinline__ float exp2Fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
// Two fp32 operations in one instruction, each rounded like the single one.
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) { return packF32x2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float lowOf(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float highOf(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// ---------------------------------------------------------------- sequences
struct Sequence {
  int q, kv, offset;   // tokens in use, and how far a query's position is ahead of its index
};
__device__ __forceinline__ Sequence sequenceOf(const AttnArgs& a, int b) {
  Sequence s;
  s.q = a.qLengths ? min(max(a.qLengths[b], 0), a.q) : a.q;
  s.kv = a.kvLengths ? min(max(a.kvLengths[b], 0), a.kv) : a.kv;
  s.offset = a.causal == 2 ? s.kv - s.q : a.offset;
  return s;
}
// Keys that the query at `tok` sees: those in front of this one.
__device__ __forceinline__ int visibleOf(const AttnArgs& a, const Sequence& s, int tok) { return a.causal ? max(0, min(s.kv, tok + s.offset + 1)) : s.kv; }

// ---------------------------------------------------------------- waits
__device__ __forceinline__ void reportTimeout(uint32_t* status, uint32_t what) {
  if (status && ldRelaxedSys(status) == DEV_OK) {
    status[1] = WAIT_TILE;
    status[2] = what;
    status[3] = blockIdx.x;
    __threadfence_system();
    stRelaxedSys(status, DEV_TIMEOUT);
  }
}
// Bounded; ends early when another role has given up.
__device__ __forceinline__ bool waitOr(uint32_t bar, uint32_t parity, volatile uint32_t* abortFlag) {
  if (mbarTry(bar, parity)) return true;
  for (uint32_t i = 0; i < (1u << 24) && !*abortFlag; ++i)
    if (mbarTry(bar, parity)) return true;
  return false;
}
// The same for a whole warp, with one answer.
__device__ __forceinline__ bool warpWaitOr(uint32_t bar, uint32_t parity, volatile uint32_t* abortFlag) {
  return __all_sync(~0u, waitOr(bar, parity, abortFlag));
}

// A barrier of N threads that tells them all whether all are well.
template <int N> __device__ __forceinline__ bool allWell(int id, bool well) {
  uint32_t all;
  asm volatile(
      "{\n.reg .pred p, q;\n"
      "setp.ne.u32 p, %3, 0;\n"
      "barrier.cta.red.and.pred q, %1, %2, p;\n"
      "selp.u32 %0, 1, 0, q;\n}"
      : "=r"(all) : "r"(id), "n"(N), "r"((uint32_t)well) : "memory");
  return all != 0;
}

}  // namespace attn
}  // namespace b200
