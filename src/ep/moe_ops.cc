// Host side of the mixture-of-experts operators around dispatch and combine: routing, the experts' products, and the gradients that
// cross the exchange. Checks of arguments, tensor maps and launches; the kernels are in route.cu, expert_gemm_sm100.cu and moe_backward.cu.
#include "moe_ops.h"

#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "ep_group.h"

using namespace b200;

static bool routeConfigOk(const ncclEpRouteConfig_t* c) { return c && c->magic == NCCL_EP_MAGIC && c->size == sizeof(*c); }

static bool aligned(std::initializer_list<const void*> ps, size_t to) {
  uintptr_t all = 0;
  for (const void* p : ps) all |= (uintptr_t)p;
  return all % to == 0;
}

// The group's GPU is the current one while this lives.
struct OnDevice {
  int before = -1, dev;
  cudaError_t rc;
  explicit OnDevice(int d) : dev(d) {
    rc = cudaGetDevice(&before);
    if (rc == cudaSuccess && before != dev) rc = cudaSetDevice(dev);
  }
  ~OnDevice() { if (before >= 0 && before != dev) cudaSetDevice(before); }
};
#define B200_ON_DEVICE(g)              \
  OnDevice onDevice((g)->comm->cudaDev); \
  CUDACHECK(onDevice.rc)

static ncclResult_t launchMoe(ncclEpGroup* g, const void* fn, dim3 grid, int threads, size_t smem, void** args, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  if (devPlanePdl()) {
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  if (smem > 40000) CUDACHECK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
  if (e != cudaSuccess) {
    WARN("mixture-of-experts kernel launch failed: %s", cudaGetErrorString(e));
    (void)cudaGetLastError();
    return ncclUnhandledCudaError;
  }
  if (g->comm->devPlane) g->comm->devPlane->launches++;
  return ncclSuccess;
}

// ---------------------------------------------------------------- routing
static ncclResult_t fillRoute(const char* what, ncclDataType_t type, int tokens, int experts, int topk, const ncclEpRouteConfig_t* c, RouteArgs* a, int* kind) {
  *kind = type == ncclFloat32 ? ROUTE_F32 : type == ncclFloat16 ? ROUTE_F16 : type == ncclBfloat16 ? ROUTE_BF16 : -1;
  if (*kind < 0) { WARN("%s: logits must be fp32, fp16 or bf16", what); return ncclInvalidArgument; }
  if (!routeConfigOk(c)) { WARN("%s: configuration was not initialised", what); return ncclInvalidArgument; }
  if (c->score != NCCL_EP_SCORE_SOFTMAX && c->score != NCCL_EP_SCORE_SIGMOID) { WARN("%s: unknown score %d", what, (int)c->score); return ncclInvalidArgument; }
  if (tokens < 0 || experts <= 0 || topk <= 0 || topk > kRouteMaxTopk || topk > experts || experts > kRouteMaxExperts) {
    WARN("%s: %d tokens, top-%d of %d experts (at most %d experts, top-%d)", what, tokens, topk, experts, kRouteMaxExperts, kRouteMaxTopk);
    return ncclInvalidArgument;
  }
  if (!(c->scale > 0.0f) || !std::isfinite(c->scale)) { WARN("%s: scale must be positive and finite", what); return ncclInvalidArgument; }
  memset(a, 0, sizeof(*a));
  a->tokens = tokens;
  a->experts = experts;
  a->topk = topk;
  a->groups = a->keep = 1;
  a->perGroup = experts;
  a->sigmoid = c->score == NCCL_EP_SCORE_SIGMOID;
  a->renormalize = c->renormalize != 0;
  a->scale = c->scale;
  return ncclSuccess;
}

// Deals the warp's lanes out to the groups. Packs: where every lane has as many experts as its registers hold, and they begin at whole packs of 16 bytes (or of the
// lane's share, where that is less).
static void dealLanes(RouteArgs* a, int kind, std::initializer_list<const void*> ps) {
  a->lanes = 32;
  while (a->lanes * a->groups > 32) a->lanes /= 2;
  a->perLane = (a->perGroup + a->lanes - 1) / a->lanes;
  const int size = kind == ROUTE_F32 ? 4 : 2, bytes = std::min(16, a->perLane * size);
  a->wide = (a->perLane & (a->perLane - 1)) == 0 && a->perGroup * size % bytes == 0 && aligned(ps, bytes);
}

static ncclResult_t launchRoute(ncclEpGroup* g, const void* fn, RouteArgs* a, cudaStream_t stream) {
  void* args[1] = {a};
  return launchMoe(g, fn, dim3(((unsigned)a->tokens + routeWarps() - 1) / routeWarps()), routeWarps() * 32, 0, args, stream);
}

// ---------------------------------------------------------------- the experts' products
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encodeFn() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess) return (EncodeTiledFn)p;
    (void)cudaGetLastError();
    return (EncodeTiledFn) nullptr;
  }();
  return fn;
}

// bf16 [experts][rows][inner], boxes of boxRows x 64 values of one expert with 128-byte swizzle.
static ncclResult_t makeMap(CUtensorMap* map, const void* base, int inner, int rows, int experts, int boxRows) {
  EncodeTiledFn enc = encodeFn();
  if (!enc) { WARN("cuTensorMapEncodeTiled is not available"); return ncclUnhandledCudaError; }
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)experts};
  cuuint64_t strides[2] = {(cuuint64_t)inner * 2, (cuuint64_t)inner * 2 * (cuuint64_t)rows};
  cuuint32_t box[3] = {64, (cuuint32_t)boxRows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, (void*)base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { WARN("cuTensorMapEncodeTiled failed (%d)", (int)r); return ncclUnhandledCudaError; }
  return ncclSuccess;
}

// The activation without the flag beside it.
static int actOf(ncclEpActivation_t a) { return (int)a & ~(int)NCCL_EP_ACT_PRE_FP32; }
static bool preInFp32(ncclEpActivation_t a) { return ((int)a & (int)NCCL_EP_ACT_PRE_FP32) != 0; }

static ncclResult_t checkLinear(const ncclEpGroup* g, const char* what, int experts, int rows, int n, int k, int act) {
  if (g->comm->compCap < 100) { WARN("%s needs compute capability 10.0 (found %d)", what, g->comm->compCap); return ncclInvalidUsage; }
  if (act < ACT_NONE || act > ACT_GEGLU) { WARN("%s: unknown activation %d", what, act); return ncclInvalidArgument; }
  const int unit = actGated(act) ? 16 : 8;
  if (experts <= 0 || experts > kExpertMax || rows < 0 || n <= 0 || k <= 0 || n % unit || k % 8) {
    WARN("%s: %d experts (at most %d), %d rows, n=%d must be a multiple of %d, k=%d of 8", what, experts, kExpertMax, rows, n, unit, k);
    return ncclInvalidArgument;
  }
  // sums of more steps would outlast the kernels' waits; and a tile is numbered with 31 bits, whatever its width
  const int longest = 1 << 24;
  const double tilesN = (n + 31) / 32, tilesK = (k + 31) / 32, most = 1 << 30;
  if ((double)experts * ((rows + 127) / 128) * std::max(tilesN, tilesK) > most || (double)experts * ((n + 127) / 128) * tilesK > most || rows > longest || n > longest || k > longest) {
    WARN("%s: %d experts x %d rows x n=%d, k=%d are too many tiles", what, experts, rows, n, k);
    return ncclInvalidArgument;
  }
  return ncclSuccess;
}

// Pairs that can be resident at once: with more the last ones would start when the first have finished all their tiles.
static int pairsAtOnce(ncclEpGroup* g) {
  int n = g->expertPairs.load(std::memory_order_relaxed);
  if (n >= 0) return n;
  n = g->smCount / 2;
  for (int form = 0; form < 5; ++form) {
    const void* fn = expertGemmPairKernelFn(form % 3, form >= 3);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(g->smCount & ~1);
    cfg.blockDim = dim3(expertGemmThreads(true));
    cfg.dynamicSmemBytes = expertGemmSmemBytes();
    int clusters = 0;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)expertGemmSmemBytes()) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&clusters, fn, &cfg) == cudaSuccess && clusters > 0)
      n = std::min(n, clusters);
    else
      (void)cudaGetLastError();
  }
  g->expertPairs.store(n, std::memory_order_relaxed);
  return n;
}

// A product of [experts][rowsA][innerA] and [experts][rowsB][innerB]; see expert_gemm_sm100.cu for what each mode makes of them. The host knows how many
// rows an expert may have, not how many it has: where a tile of 128 holds them all, single CTAs take a tile each, else pairs tiles of 256.
static ncclResult_t launchExpertGemm(ncclEpGroup* g, int mode, const void* A, int innerA, int rowsA, const void* B, int innerB, int rowsB, ExpertGemmArgs* a, cudaStream_t stream) {
  const bool pair = mode == EXPERT_DW || a->cap > kExpertOneCtaRows;
  a->boxRows = pair ? 128 : std::min(32, (a->cap + 7) / 8 * 8);
  a->wide = a->cols % 16 == 0 && aligned({a->out, a->pre}, 32);
  a->status = g->comm->devStatusDev;
  CUtensorMap maps[3];
  NCCLCHECK(makeMap(&maps[0], A, innerA, rowsA, a->experts, mode == EXPERT_DW ? 64 : a->boxRows));
  NCCLCHECK(makeMap(&maps[1], B, innerB, rowsB, a->experts, mode == EXPERT_FORWARD ? 128 : 64));
  if (mode == EXPERT_FORWARD) NCCLCHECK(makeMap(&maps[2], B, innerB, rowsB, a->experts, pair || a->gated ? 64 : 32));
  else maps[2] = maps[1];
  void* args[4] = {&maps[0], &maps[1], &maps[2], a};
  // no more CTAs than the narrowest tiles of all rows
  const double rows = mode == EXPERT_DW ? a->outRows : a->cap, tilesN = (a->cols + 31) / 32;
  if (pair) {
    const double tiles = (double)a->experts * (int)((rows + 255) / 256) * tilesN;
    const int pairs = (int)std::min<double>(pairsAtOnce(g), tiles);
    // Through shared memory go results that a lane would touch 16 bytes at a time (a residual, rows that are not whole packs of 32 bytes). With `pre` that makes the
    // sums twice, which pays where there may be many tiles (of 256 columns, eight for each pair): 16 experts of 1800 rows, 4696 x 328, there and back 668 us straight from registers,
    // 517 so; five of 310 rows, 2200 x 1000, 86 and 100.
    const bool staged = (a->residual || !a->wide) && (!a->pre || tiles / 8 > 8.0 * pairs);
    return launchMoe(g, expertGemmPairKernelFn(mode, staged), dim3(2 * pairs), expertGemmThreads(true), expertGemmSmemBytes(), args, stream);
  }
  const int ctas = (int)std::min<double>(g->smCount, (double)a->experts * tilesN);
  return launchMoe(g, expertGemmKernelFn(mode), dim3(ctas), expertGemmThreads(false), expertGemmSmemBytes(), args, stream);
}

// Slices of rows that the activation's backward works on at a time: enough CTAs to fill the chip four times over.
static int actSlices(const ncclEpGroup* g, int experts, int rows, int cols) {
  const long long perSlice = (long long)experts * ((cols + kActCols - 1) / kActCols);
  const long long want = ((long long)g->smCount * 4 + perSlice - 1) / perSlice, most = (rows + 7) / 8;
  return (int)std::max<long long>(1, std::min<long long>({want, most, 64}));
}

static size_t dzBytes(int experts, int rows, int n, int act) { return act == ACT_NONE ? 0 : ((size_t)experts * rows * n * 2 + 255) / 256 * 256; }

extern "C" {

ncclResult_t ncclEpRoute(ncclEpGroup_t g, const void* logits, ncclDataType_t type, const float* bias, int64_t* idx, float* weights, int tokens, int experts, int topk,
                         const ncclEpRouteConfig_t* c, cudaStream_t stream) {
  if (!g) return ncclInvalidArgument;
  RouteArgs a;
  int kind;
  NCCLCHECK(fillRoute("ncclEpRoute", type, tokens, experts, topk, c, &a, &kind));
  if (c->groups <= 0 || c->groups > kRouteMaxGroups || experts % c->groups || c->keep_groups <= 0 || c->keep_groups > c->groups) {
    WARN("ncclEpRoute: %d experts in %d groups (at most %d), %d kept", experts, c->groups, kRouteMaxGroups, c->keep_groups);
    return ncclInvalidArgument;
  }
  if (c->group_score != NCCL_EP_GROUP_SCORE_MAX && c->group_score != NCCL_EP_GROUP_SCORE_TOP2) { WARN("ncclEpRoute: unknown group score %d", (int)c->group_score); return ncclInvalidArgument; }
  const int perGroup = experts / c->groups;
  if (topk > c->keep_groups * perGroup) { WARN("ncclEpRoute: top-%d of %d groups of %d experts", topk, c->keep_groups, perGroup); return ncclInvalidArgument; }
  if (tokens == 0) return ncclSuccess;
  if (!logits || !idx || !weights) return ncclInvalidArgument;
  if (!aligned({logits}, kind == ROUTE_F32 ? 4 : 2) || !aligned({bias, weights}, 4) || !aligned({idx}, 8)) { WARN("ncclEpRoute: misaligned tensors"); return ncclInvalidArgument; }
  const size_t entries = (size_t)tokens * topk, logitBytes = (size_t)tokens * experts * (kind == ROUTE_F32 ? 4 : 2);
  if (overlap({{idx, entries * 8}, {weights, entries * 4}}, {{logits, logitBytes}, {bias, (size_t)experts * 4}}) || overlap({{idx, entries * 8}}, {{weights, entries * 4}})) {
    WARN("ncclEpRoute: an output shares memory with another tensor");
    return ncclInvalidArgument;
  }
  a.logits = logits;
  a.bias = bias;
  a.idx = idx;
  a.weights = weights;
  // with every group kept they change nothing
  if (c->keep_groups < c->groups) {
    a.groups = c->groups;
    a.keep = c->keep_groups;
    a.perGroup = perGroup;
  }
  a.top2 = c->group_score == NCCL_EP_GROUP_SCORE_TOP2 && perGroup > 1;
  dealLanes(&a, kind, {logits});
  a.wideBias = a.perLane % 4 == 0 && a.perGroup % 4 == 0 && aligned({bias}, 16);
  B200_ON_DEVICE(g);
  return launchRoute(g, routeKernelFn(kind, a.perLane), &a, stream);
}

ncclResult_t ncclEpRouteBackward(ncclEpGroup_t g, const float* dweights, const void* logits, ncclDataType_t type, const int64_t* idx, void* dlogits, int tokens, int experts, int topk,
                                 const ncclEpRouteConfig_t* c, cudaStream_t stream) {
  if (!g) return ncclInvalidArgument;
  RouteArgs a;
  int kind;
  NCCLCHECK(fillRoute("ncclEpRouteBackward", type, tokens, experts, topk, c, &a, &kind));
  if (tokens == 0) return ncclSuccess;
  if (!dweights || !logits || !idx || !dlogits) return ncclInvalidArgument;
  if (!aligned({logits, dlogits}, kind == ROUTE_F32 ? 4 : 2) || !aligned({dweights}, 4) || !aligned({idx}, 8)) { WARN("ncclEpRouteBackward: misaligned tensors"); return ncclInvalidArgument; }
  const size_t entries = (size_t)tokens * topk, logitBytes = (size_t)tokens * experts * (kind == ROUTE_F32 ? 4 : 2);
  // a token's row is read before its gradient is written: the one may take the other's place
  if (overlap({{dlogits, logitBytes}}, {{logits == dlogits ? nullptr : logits, logitBytes}, {dweights, entries * 4}, {idx, entries * 8}})) {
    WARN("ncclEpRouteBackward: the output shares memory with an input (it may take the logits' place)");
    return ncclInvalidArgument;
  }
  a.logits = logits;
  a.idx = (int64_t*)idx;
  a.dweights = dweights;
  a.dlogits = dlogits;
  dealLanes(&a, kind, {logits, dlogits});
  B200_ON_DEVICE(g);
  return launchRoute(g, routeBackwardKernelFn(kind, a.perLane), &a, stream);
}

ncclResult_t ncclEpExpertLinear(ncclEpGroup_t g, const void* x, const void* w, const int* counts, const void* bias, const void* residual, void* out, void* pre, int experts,
                                int rows, int n, int k, ncclEpActivation_t activation, cudaStream_t stream) {
  if (!g) return ncclInvalidArgument;
  const int act = actOf(activation);
  NCCLCHECK(checkLinear(g, "ncclEpExpertLinear", experts, rows, n, k, act));
  if (rows == 0) return ncclSuccess;
  if (!x || !w || !out) return ncclInvalidArgument;
  if (!aligned({x, w, bias, residual, out, pre}, 16) || !aligned({counts}, 4)) { WARN("ncclEpExpertLinear: tensors must be 16-byte aligned"); return ncclInvalidArgument; }
  const size_t er = (size_t)experts * rows, outBytes = er * (actGated(act) ? n / 2 : n) * 2, preBytes = er * n * (preInFp32(activation) ? 4 : 2);
  if (overlap({{out, outBytes}, {pre, preBytes}}, {{x, er * k * 2}, {w, (size_t)experts * n * k * 2}, {counts, (size_t)experts * 4}, {bias, (size_t)experts * n * 2},
                                                   {residual == out ? nullptr : residual, outBytes}}) ||
      overlap({{pre, preBytes}}, {{out, outBytes}, {residual, outBytes}})) {
    WARN("ncclEpExpertLinear: an output shares memory with another tensor (the residual may be the output itself)");
    return ncclInvalidArgument;
  }
  NCCLCHECK(devPlaneCheckStatus(g->comm));
  B200_ON_DEVICE(g);
  ExpertGemmArgs a;
  memset(&a, 0, sizeof(a));
  a.counts = counts;
  a.experts = experts;
  a.cap = rows;
  a.gated = actGated(act);
  a.act = act;
  a.cols = a.gated ? n / 2 : n;
  a.depth = k;
  a.bias = bias;
  a.residual = residual;
  a.out = out;
  a.pre = pre;
  a.preFp32 = preInFp32(activation);
  return launchExpertGemm(g, EXPERT_FORWARD, x, k, rows, w, k, n, &a, stream);
}

size_t ncclEpExpertLinearBackwardWork(ncclEpGroup_t g, int experts, int rows, int n, ncclEpActivation_t activation, int withBias) {
  if (!g || experts <= 0 || experts > kExpertMax || rows <= 0 || n <= 0) return 0;
  const int act = actOf(activation);
  const int cols = actGated(act) ? n / 2 : n;
  return dzBytes(experts, rows, n, act) + (withBias ? (size_t)actSlices(g, experts, rows, cols) * experts * n * sizeof(float) : 0);
}

ncclResult_t ncclEpExpertLinearBackward(ncclEpGroup_t g, const void* dout, const void* x, const void* w, const int* counts, const void* pre, void* dx, void* dw, void* dbias,
                                        void* work, int experts, int rows, int n, int k, ncclEpActivation_t activation, cudaStream_t stream) {
  if (!g) return ncclInvalidArgument;
  const int act = actOf(activation);
  NCCLCHECK(checkLinear(g, "ncclEpExpertLinearBackward", experts, rows, n, k, act));
  const bool needDz = act != ACT_NONE;
  if (!aligned({dout, x, w, pre, dx, dw, dbias, work}, 16) || !aligned({counts}, 4)) { WARN("ncclEpExpertLinearBackward: tensors must be 16-byte aligned"); return ncclInvalidArgument; }
  if (rows > 0 && (!dout || (needDz && !pre) || (dx && !w) || (dw && !x) || ((needDz || dbias) && !work))) {
    WARN("ncclEpExpertLinearBackward: a tensor that the wanted gradients need is missing");
    return ncclInvalidArgument;
  }
  const size_t er = (size_t)experts * rows, weights = (size_t)experts * n * k * 2, biases = (size_t)experts * n * 2;
  const Span given[] = {{dout, er * (actGated(act) ? n / 2 : n) * 2}, {x, er * k * 2}, {w, weights}, {counts, (size_t)experts * 4}, {pre, er * n * (preInFp32(activation) ? 4 : 2)}};
  const Span made[] = {{dx, er * k * 2}, {dw, weights}, {dbias, biases}, {work, ncclEpExpertLinearBackwardWork(g, experts, rows, n, activation, dbias != nullptr)}};
  for (const Span& o : made) {
    for (const Span& i : given)
      if (overlap({o}, {i})) { WARN("ncclEpExpertLinearBackward: an output shares memory with an input"); return ncclInvalidArgument; }
    for (const Span& i : made)
      if (&i != &o && overlap({o}, {i})) { WARN("ncclEpExpertLinearBackward: two outputs share memory"); return ncclInvalidArgument; }
  }
  NCCLCHECK(devPlaneCheckStatus(g->comm));
  B200_ON_DEVICE(g);
  if (rows == 0) {   // nothing to add up
    if (dw) CUDACHECK(cudaMemsetAsync(dw, 0, (size_t)experts * n * k * 2, stream));
    if (dbias) CUDACHECK(cudaMemsetAsync(dbias, 0, (size_t)experts * n * 2, stream));
    return ncclSuccess;
  }
  const int gated = actGated(act), cols = gated ? n / 2 : n;
  const void* dz = needDz ? work : dout;
  // products on CTA pairs have warps to spare for the last step of the bias's gradient: a launch less (5 experts of 310 rows, 2200 x 1000, there and back 81 us,
  // 79 without)
  const bool dxOnPairs = dx && rows > kExpertOneCtaRows, biasAside = dbias && (dxOnPairs || dw);
  if (needDz || dbias) {
    ExpertActArgs e;
    memset(&e, 0, sizeof(e));
    e.counts = counts;
    e.dout = dout;
    e.pre = pre;
    e.dz = needDz ? work : nullptr;
    e.experts = experts;
    e.cap = rows;
    e.cols = cols;
    e.act = act;
    e.slices = actSlices(g, experts, rows, cols);
    e.partial = dbias ? (float*)((char*)work + dzBytes(experts, rows, n, act)) : nullptr;
    e.dbias = dbias;
    void* args[1] = {&e};
    NCCLCHECK(launchMoe(g, expertActKernelFn(act, preInFp32(activation)), dim3((cols + kActCols - 1) / kActCols, experts, e.slices), kActThreads, 0, args, stream));
    if (dbias && !biasAside)
      NCCLCHECK(launchMoe(g, expertBiasKernelFn(), dim3((unsigned)std::min<size_t>(((size_t)experts * n / 4 + kActThreads - 1) / kActThreads, (size_t)g->smCount * 8)), kActThreads, 0, args, stream));
  }
  ExpertGemmArgs a;
  memset(&a, 0, sizeof(a));
  if (biasAside) {
    a.partial = (const float*)((char*)work + dzBytes(experts, rows, n, act));
    a.dbias = dbias;
    a.sums = (size_t)experts * n;
    a.slices = actSlices(g, experts, rows, cols);
  }
  a.counts = counts;
  a.experts = experts;
  a.cap = rows;
  a.cols = k;
  if (dx) {
    a.depth = n;
    a.out = dx;
    NCCLCHECK(launchExpertGemm(g, EXPERT_DX, dz, n, rows, w, k, n, &a, stream));
    if (dxOnPairs) a.partial = nullptr;   // done
  }
  if (dw) {
    a.depth = rows;
    a.outRows = n;
    a.out = dw;
    NCCLCHECK(launchExpertGemm(g, EXPERT_DW, dz, n, rows, x, k, rows, &a, stream));
  }
  return ncclSuccess;
}

ncclResult_t ncclEpDispatchRows(ncclEpHandle_t h, int* rows, cudaStream_t stream) {
  if (!h) return ncclInvalidArgument;
  ncclEpGroup* g = h->g;
  if (!h->rowOf) { WARN("ncclEpDispatchRows: needs a group of one rank and the expert-major layout"); return ncclInvalidUsage; }
  // (a combine that waits for its other half does not touch the rows)
  if (!h->sentIdx || h->pending == 1) { WARN("ncclEpDispatchRows: no dispatch has been completed on this handle"); return ncclInvalidUsage; }
  if (h->sentT == 0) return ncclSuccess;
  if (!rows || !aligned({rows}, 4)) return ncclInvalidArgument;
  B200_ON_DEVICE(g);
  DispatchRowsArgs a;
  a.idx = h->sentIdx;
  a.rowOf = h->rowOf;
  a.srcInfo = h->srcInfo;
  a.counts = h->expertCount;
  a.rows = rows;
  a.entries = (size_t)h->sentT * h->K;
  a.experts = g->E;
  a.cap = g->maxTokens;
  a.rank = g->comm->rank;
  void* args[1] = {&a};
  return launchMoe(g, dispatchRowsKernelFn(), dim3((unsigned)std::min<size_t>((a.entries + kMoeRowThreads - 1) / kMoeRowThreads, (size_t)g->smCount * 4)), kMoeRowThreads, 0, args, stream);
}

static ncclResult_t checkRows(const char* what, int tokens, int topk, int hidden, int numRows) {
  if (tokens < 0 || topk <= 0 || topk > kRouteMaxTopk || hidden <= 0 || hidden % 8 || numRows < 0) {
    WARN("%s: %d tokens, top-%d (at most %d), hidden=%d must be a multiple of 8, %d rows", what, tokens, topk, kRouteMaxTopk, hidden, numRows);
    return ncclInvalidArgument;
  }
  return ncclSuccess;
}

ncclResult_t ncclEpCombineBackward(ncclEpGroup_t g, const void* dout, const void* y, const float* weights, const int* rows, void* dy, float* dweights, int tokens, int topk,
                                   int hidden, int numRows, cudaStream_t stream) {
  if (!g) return ncclInvalidArgument;
  NCCLCHECK(checkRows("ncclEpCombineBackward", tokens, topk, hidden, numRows));
  if (tokens == 0) return ncclSuccess;
  if (!dout || !weights || !rows || !dweights || (numRows > 0 && (!y || !dy))) return ncclInvalidArgument;
  if (!aligned({dout, y, dy}, 16) || !aligned({weights, rows, dweights}, 4)) { WARN("ncclEpCombineBackward: tensors must be 16-byte aligned"); return ncclInvalidArgument; }
  const size_t T = tokens, rowBytes = (size_t)hidden * 2, entries = T * topk * 4;
  // dy may take y's place: a row is read and written by the same threads
  if (overlap({{dy, numRows * rowBytes}, {dweights, entries}}, {{dout, T * rowBytes}, {y == dy ? nullptr : y, numRows * rowBytes}, {weights, entries}, {rows, entries}}) ||
      overlap({{dweights, entries}}, {{y, numRows * rowBytes}, {dy, numRows * rowBytes}})) {
    WARN("ncclEpCombineBackward: an output shares memory with another tensor (the rows' gradients may take the rows' place)");
    return ncclInvalidArgument;
  }
  B200_ON_DEVICE(g);
  MoeRowsArgs a;
  memset(&a, 0, sizeof(a));
  a.dout = dout;
  a.y = y;
  a.weights = weights;
  a.rows = rows;
  a.dy = dy;
  a.dweights = dweights;
  a.tokens = tokens;
  a.topk = topk;
  a.hidden = hidden;
  a.numRows = numRows;
  void* args[1] = {&a};
  return launchMoe(g, combineBackwardKernelFn(topk), dim3(std::min(tokens, g->smCount * 16)), kMoeRowThreads, 0, args, stream);
}

ncclResult_t ncclEpDispatchBackward(ncclEpGroup_t g, const void* dtoks, const int* rows, void* dx, int tokens, int topk, int hidden, int numRows, cudaStream_t stream) {
  if (!g) return ncclInvalidArgument;
  NCCLCHECK(checkRows("ncclEpDispatchBackward", tokens, topk, hidden, numRows));
  if (tokens == 0) return ncclSuccess;
  if (!rows || !dx || (numRows > 0 && !dtoks)) return ncclInvalidArgument;
  if (!aligned({dtoks, dx}, 16) || !aligned({rows}, 4)) { WARN("ncclEpDispatchBackward: tensors must be 16-byte aligned"); return ncclInvalidArgument; }
  if (overlap({{dx, (size_t)tokens * hidden * 2}}, {{dtoks, (size_t)numRows * hidden * 2}, {rows, (size_t)tokens * topk * 4}})) {
    WARN("ncclEpDispatchBackward: the output shares memory with an input");
    return ncclInvalidArgument;
  }
  B200_ON_DEVICE(g);
  MoeRowsArgs a;
  memset(&a, 0, sizeof(a));
  a.y = dtoks;
  a.rows = rows;
  a.dx = dx;
  a.tokens = tokens;
  a.topk = topk;
  a.hidden = hidden;
  a.numRows = numRows;
  void* args[1] = {&a};
  return launchMoe(g, dispatchBackwardKernelFn(), dim3(std::min(tokens, g->smCount * 16)), kMoeRowThreads, 0, args, stream);
}

}  // extern "C"
