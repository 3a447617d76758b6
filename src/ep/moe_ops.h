// Internal interface between the host code of the mixture-of-experts operators (moe_ops.cc) and their kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

// ---------------------------------------------------------------- routing (route.cu)
constexpr int kRouteMaxExperts = 1024, kRouteMaxTopk = 16, kRouteMaxGroups = 32;
constexpr int kRouteMaxPerLane = 64;   // 1024 experts in a little more than half as many groups as there are lane shares

struct RouteArgs {
  const void* logits;         // [tokens][experts]
  const float* bias;          // [experts] or null
  int64_t* idx;               // [tokens][topk], -1 = no expert
  float* weights;             // [tokens][topk]
  const float* dweights;      // backward: [tokens][topk]
  void* dlogits;              // backward: [tokens][experts]
  int tokens, experts, topk;
  int groups, keep, perGroup; // groups of perGroup experts next to each other, of which `keep` stay
  int lanes, perLane;         // lanes of a warp for each group (a power of two), and experts of a lane
  int sigmoid, top2, renormalize;
  float scale;
  int wide, wideBias;         // rows of logits, and the bias, may be read in packs of 16 bytes
};

enum RouteType : int { ROUTE_F32 = 0, ROUTE_F16 = 1, ROUTE_BF16 = 2 };
const void* routeKernelFn(int type, int perLane);
const void* routeBackwardKernelFn(int type, int perLane);
int routeWarps();             // warps of a CTA, one token each

// ---------------------------------------------------------------- the experts' products (expert_gemm_sm100.cu)
enum ExpertAct : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3, ACT_SWIGLU = 4, ACT_GEGLU = 5 };
inline bool actGated(int act) { return act == ACT_SWIGLU || act == ACT_GEGLU; }

// Which of the three products of a linear layer: rows x W^T, their gradient dz W, or the weights' gradient dz^T x.
enum ExpertMode : int { EXPERT_FORWARD = 0, EXPERT_DX = 1, EXPERT_DW = 2 };

constexpr int kExpertMax = 256;   // experts of a call: the tile counts of all of them are held in shared memory

struct ExpertGemmArgs {
  const int* counts;          // [experts] rows in use (null: all of them)
  int experts, cap;           // rows that the tensors have for each expert
  int outRows;                // DW: rows of the result (of W); else the rows in use
  int cols;                   // columns of the result
  int depth;                  // length of the sums (DW: cap; the rows in use count)
  int boxRows;                // rows of a box of the first operand (the kernel on single CTAs)
  int wide;                   // rows of out and pre may be stored in packs of 32 bytes
  int gated, act;             // forward: gate rows of W, then up rows, `cols` of each
  const void* bias;           // bf16 [experts][cols, twice when gated] or null
  const void* residual;       // bf16, laid out like out, or null
  void* out;                  // bf16 [experts][cap or outRows][cols]
  void* pre;                  // bf16 or fp32 [experts][cap][cols, twice when gated]: what the activation is applied to, or null
  int preFp32;
  const float* partial;       // backward, on pairs: sums for the bias's gradient, [slices][sums], that a warp without other work adds up, or null
  void* dbias;                // bf16 [sums]
  size_t sums;                // a multiple of 8
  int slices;
  uint32_t* status;           // {code, kind, what, CTA} of the communicator, written when a wait runs out
};

constexpr int kExpertOneCtaRows = 128;   // an expert with more rows takes the kernel on CTA pairs
const void* expertGemmKernelFn(int mode);       // FORWARD, DX; tensor maps of A, B and B in boxes of 32 rows (gated: 64)
const void* expertGemmPairKernelFn(int mode, bool staged);   // tensor maps of A, B and B in boxes of 64 rows; clusters of two. staged: results go through shared memory (DW: always)
size_t expertGemmSmemBytes();
int expertGemmThreads(bool pair);

// ---------------------------------------------------------------- row kernels (moe_backward.cu)
struct ExpertActArgs {
  const int* counts;
  const void* dout;           // bf16 [experts][cap][cols]
  const void* pre;            // bf16 or fp32 [experts][cap][cols, twice when gated]; not read without an activation
  void* dz;                   // bf16, laid out like pre; null without an activation
  float* partial;             // [slices][experts][cols, twice when gated] sums of dz over the rows of a slice, or null
  void* dbias;                // bf16 [experts][cols, twice when gated] or null
  int experts, cap, cols, act, slices;
};
const void* expertActKernelFn(int act, bool preFp32);
const void* expertBiasKernelFn();
constexpr int kActCols = 256, kActThreads = 256;   // columns and threads of a CTA

struct MoeRowsArgs {
  const void* dout;           // [tokens][hidden] bf16
  const void* y;              // rows of the experts, bf16
  const float* weights;       // [tokens][topk]
  const int* rows;            // [tokens][topk], negative = no row
  void* dy;
  float* dweights;
  void* dx;                   // dispatch's backward: [tokens][hidden]
  int tokens, topk, hidden, numRows;
};
const void* combineBackwardKernelFn(int topk);
const void* dispatchBackwardKernelFn();
constexpr int kMoeRowThreads = 256;

struct DispatchRowsArgs {
  const int64_t* idx;         // [tokens][topk] of the last dispatch
  const int* rowOf;
  const int2* srcInfo;
  const int* counts;
  int* rows;
  size_t entries;
  int experts, cap, rank;
};
const void* dispatchRowsKernelFn();

}  // namespace b200
