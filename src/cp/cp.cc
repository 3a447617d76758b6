// Host side of the context-parallel operators: checks of arguments, plans, tensor maps and launches. See include/nccl_cp.h for the API; the kernels are in
// attention_forward.cu, attention_backward.cu and rotary.cu.
#include "cp.h"

#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>
#include <new>

#include "../comm/device_plane.h"
#include "nccl_cp.h"

using namespace b200;

struct ncclCpContext {
  ncclComm* comm = nullptr;
  int smCount = 0;
  std::atomic<const void*> ready[32] = {};   // kernels with tiles that have been set up on this GPU
};

// The context's GPU is the current one while this lives.
namespace {
struct OnDevice {
  int before = -1, dev;
  cudaError_t rc;
  explicit OnDevice(int d) : dev(d) {
    rc = cudaGetDevice(&before);
    if (rc == cudaSuccess && before != dev) rc = cudaSetDevice(dev);
  }
  ~OnDevice() { if (before >= 0 && before != dev) cudaSetDevice(before); }
};
}  // namespace
#define B200_ON_DEVICE(cp)               \
  OnDevice onDevice((cp)->comm->cudaDev); \
  CUDACHECK(onDevice.rc)

static bool aligned(std::initializer_list<const void*> ps, size_t to) {
  uintptr_t all = 0;
  for (const void* p : ps) all |= (uintptr_t)p;
  return all % to == 0;
}

// Once for each kernel that moves registers between its warps: registers that nobody was launched with would be waited for without end.
static ncclResult_t setUp(ncclCpContext* cp, const void* fn, size_t smem, int regs) {
  std::atomic<const void*>* place = nullptr;
  for (auto& r : cp->ready) {
    const void* p = r.load(std::memory_order_relaxed);
    if (p == fn) return ncclSuccess;
    if (!p) { place = &r; break; }
  }
  cudaFuncAttributes built;
  CUDACHECK(cudaFuncGetAttributes(&built, fn));
  if (built.numRegs < regs) { WARN("an attention kernel was built with %d registers instead of %d", built.numRegs, regs); return ncclInternalError; }
  CUDACHECK(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  if (place) place->store(fn, std::memory_order_relaxed);   // (two threads that come here at once do the same)
  return ncclSuccess;
}

// `regs`: what a thread of a kernel that moves registers between its warps has to be launched with.
static ncclResult_t launchCp(ncclCpContext* cp, const void* fn, unsigned grid, unsigned gridY, int threads, size_t smem, void** args, cudaStream_t stream, int regs = 0) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  cfg.gridDim = dim3(grid, gridY);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  if (devPlanePdl()) {
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  if (regs) NCCLCHECK(setUp(cp, fn, smem, regs));
  const cudaError_t e = cudaLaunchKernelExC(&cfg, fn, args);
  if (e != cudaSuccess) {
    WARN("context-parallel kernel launch failed: %s", cudaGetErrorString(e));
    (void)cudaGetLastError();
    return ncclUnhandledCudaError;
  }
  if (cp->comm->devPlane) cp->comm->devPlane->launches++;
  return ncclSuccess;
}

// ---------------------------------------------------------------- memory that tensors span
namespace {
struct Span {
  const void* p;
  size_t bytes;
};
}  // namespace
static bool meets(const Span& a, const Span& b) {
  return a.p && b.p && a.bytes && b.bytes && (uintptr_t)a.p < (uintptr_t)b.p + b.bytes && (uintptr_t)b.p < (uintptr_t)a.p + a.bytes;
}
static bool overlap(std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
  for (const Span* a = outs.begin(); a != outs.end(); ++a) {
    for (const Span& b : ins)
      if (meets(*a, b)) return true;
    for (const Span* b = a + 1; b != outs.end(); ++b)
      if (meets(*a, *b)) return true;
  }
  return false;
}
// [batch][tokens][heads][dim] with strides of the first three in elements.
static Span spanOf(const void* p, int batch, int tokens, int heads, int dim, const long long* stride, size_t size) {
  if (!p || batch <= 0 || tokens <= 0 || heads <= 0) return {p, 0};
  return {p, ((size_t)(batch - 1) * stride[0] + (size_t)(tokens - 1) * stride[1] + (size_t)(heads - 1) * stride[2] + dim) * size};
}

// Rows of a tensor that is turned: [batch][tokens][heads], strides in elements (0 where there is one).
struct Rows {
  const void* at;
  const int* sizes;
  const long long* stride;
};
// Whether rows of that many elements at these places never meet: each dimension steps over all that the smaller ones reach.
static bool nest(const int* sizes, const long long* stride, unsigned dims, __int128 extent) {
  for (int i = 0; i < 3; ++i)
    if (sizes[i] <= 1) dims &= ~(1u << i);
  while (dims) {
    int least = -1;
    for (int i = 0; i < 3; ++i)
      if (dims >> i & 1 && (least < 0 || stride[i] < stride[least])) least = i;
    if (stride[least] < extent) return false;
    extent += (__int128)(sizes[least] - 1) * stride[least];
    dims &= ~(1u << least);
  }
  return true;
}
// Whether rows of two tensors of the same batch and tokens never meet: with some dimensions stepping alike, what the others reach is apart (a projection's queries and keys).
static bool apart(Rows a, Rows b, int dim, int size) {
  if ((uintptr_t)a.at > (uintptr_t)b.at) std::swap(a, b);
  const __int128 distance = (__int128)((uintptr_t)b.at - (uintptr_t)a.at) / size;
  for (unsigned alike = 0; alike < 8; ++alike) {
    __int128 reachA = dim, reachB = dim;
    int sizes[3];
    long long stride[3];
    bool same = true;
    for (int i = 0; i < 3; ++i) {
      sizes[i] = std::max(a.sizes[i], b.sizes[i]);
      stride[i] = std::max(a.stride[i], b.stride[i]);
      if (alike >> i & 1) {
        same = same && (a.sizes[i] == 1 || b.sizes[i] == 1 || a.stride[i] == b.stride[i]);
      } else {
        reachA += (__int128)(a.sizes[i] - 1) * a.stride[i];
        reachB += (__int128)(b.sizes[i] - 1) * b.stride[i];
      }
    }
    if (same && reachA <= distance && nest(sizes, stride, alike, distance + reachB)) return true;
  }
  return false;
}

// ---------------------------------------------------------------- attention
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

static bool isFp16(const ncclCpAttention_t* c) { return c->type == ncclFloat16; }

// [batch][tokens][heads][dim], boxes of `boxTokens` tokens x `boxHeads` heads x 64 channels with 128-byte swizzle. A tensor without tokens is never read, and its strides are anything:
// its map names one row.
static ncclResult_t makeMap(CUtensorMap* map, const ncclCpAttention_t* c, const void* base, int tokens, int heads, const long long* stride, int boxTokens, int boxHeads) {
  EncodeTiledFn enc = encodeFn();
  if (!enc) { WARN("cuTensorMapEncodeTiled is not available"); return ncclUnhandledCudaError; }
  const int sizes[3] = {tokens ? heads : 1, tokens ? tokens : 1, tokens ? c->batch : 1};
  cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)sizes[0], (cuuint64_t)sizes[1], (cuuint64_t)sizes[2]};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) strides[i] = sizes[i] > 1 ? (cuuint64_t)stride[2 - i] * 2 : (cuuint64_t)c->head_dim * 2;   // (of one there is no next)
  cuuint32_t box[4] = {64, (cuuint32_t)boxHeads, (cuuint32_t)boxTokens, 1}, estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, isFp16(c) ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, (void*)base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { WARN("cuTensorMapEncodeTiled failed (%d)", (int)r); return ncclUnhandledCudaError; }
  return ncclSuccess;
}

static ncclResult_t checkShape(const char* what, const ncclCpAttention_t* c) {
  if (!c || c->magic != NCCL_CP_MAGIC || c->size != sizeof(*c)) { WARN("%s: shape was not initialised", what); return ncclInvalidArgument; }
  if (c->type != ncclFloat16 && c->type != ncclBfloat16) { WARN("%s: q, k and v must be fp16 or bf16", what); return ncclInvalidArgument; }
  if (c->result_type != c->type && c->result_type != ncclFloat32) { WARN("%s: results must be of the inputs' type or fp32", what); return ncclInvalidArgument; }
  if (c->batch < 0 || c->q_tokens < 0 || c->kv_tokens < 0 || c->heads <= 0 || c->kv_heads <= 0 || c->heads % c->kv_heads || c->heads / c->kv_heads > kAttnRows || c->head_dim <= 0 ||
      c->head_dim % 8 || c->head_dim > kAttnMaxDim || c->q_tokens > kAttnMaxTokens || c->kv_tokens > kAttnMaxTokens) {
    WARN("%s: batch %d, %d queries and %d keys (at most %d), %d heads over %d (at most %d to one), head_dim %d (a multiple of 8, at most %d)", what, c->batch, c->q_tokens, c->kv_tokens,
         kAttnMaxTokens, c->heads, c->kv_heads, kAttnRows, c->head_dim, kAttnMaxDim);
    return ncclInvalidArgument;
  }
  if (c->mask != NCCL_CP_FULL && c->mask != NCCL_CP_CAUSAL && c->mask != NCCL_CP_CAUSAL_END) { WARN("%s: unknown mask %d", what, (int)c->mask); return ncclInvalidArgument; }
  if (!(c->scale > 0.0f) || !std::isfinite(c->scale)) { WARN("%s: scale must be positive and finite", what); return ncclInvalidArgument; }
  // CTAs are counted with 31 bits, rows of a result with 40
  const double tiles = (double)c->batch * c->kv_heads * (((double)c->q_tokens * (c->heads / c->kv_heads) + c->kv_tokens) / 64 + 2);
  if (tiles * kAttnMaxSplits > 2147483647.0) { WARN("%s: too many tiles", what); return ncclInvalidArgument; }
  return ncclSuccess;
}

// An operand as the tensor maps take it.
static ncclResult_t checkOperand(const char* what, const char* name, const void* p, int batch, int tokens, int heads, const long long* stride) {
  const int sizes[3] = {batch, tokens, heads};
  bool ok = p && aligned({p}, 16);
  for (int i = 0; i < 3; ++i)
    if (sizes[i] > 1) ok = ok && stride[i] > 0 && stride[i] % 8 == 0 && stride[i] < 1ll << 38;
  if (!ok) { WARN("%s: %s must be there, at 16 bytes, with positive strides of multiples of 8 elements", what, name); return ncclInvalidArgument; }
  return ncclSuccess;
}

static void fillAttention(const ncclCpAttention_t* c, const int* qLengths, const int* kvLengths, AttnArgs* a) {
  memset(a, 0, sizeof(*a));
  a->batch = c->batch;
  a->q = c->q_tokens;
  a->kv = c->kv_tokens;
  a->heads = c->heads;
  a->kvHeads = c->kv_heads;
  a->dim = c->head_dim;
  a->group = c->heads / c->kv_heads;
  a->tileTokens = std::min(kAttnRows / a->group, std::max(c->q_tokens, 1));
  a->tiles = (c->q_tokens + a->tileTokens - 1) / a->tileTokens;
  a->vTiles = (c->kv_tokens + kAttnRows - 1) / kAttnRows;
  a->causal = (int)c->mask;
  // further out nothing changes any more (and a query's token, its offset and one more stay within 31 bits)
  a->offset = (int)std::max<long long>(-(long long)c->q_tokens, std::min<long long>(c->offset, std::max(c->kv_tokens - 1, 0)));
  a->scale = c->scale;
  a->qLengths = qLengths;
  a->kvLengths = kvLengths;
  a->splits = 1;
}

// How a forward call is cut up: CTAs with two tiles of queries each ("pairs"), with one whose keys their two halves share, or with at most 32 rows, two to an SM ("few"); and with few
// CTAs, or long keys, into how many parts the keys of a tile.
//
// (All of it measured at 128 channels where nothing else is said; at 64 a tile costs half, and the units with it.)
// Pairs move half as many keys, CTAs with one tile fill the SMs better. Both are estimated in units of what a pair takes for a tile of keys (2 us, 128 channels): waves of CTAs, each
// with the mean number of tiles (of which a CTA with one tile of queries makes two at a time, for 1.15 of the time), the longest CTA at least, and a constant for a CTA's beginning
// and end. Measured with inputs from memory, us, pairs and single tiles (32 heads over 8 of 128 channels where nothing else is said): 2048 x 2048 78, 94; the same, causal 49, 66;
// 4096 causal 139, 168; 1024 x 4096 70, 80; 1500 x 8192 242, 205; 3000 x 3000 of 10 heads over 2, causal 55, 41; 3 x 777 x 1013 of 12 heads over 4, 80 channels 27, 37.
// Parts cost a second kernel and the partial results, and pay where they save more tiles than that, 5 to 9 by the number of rows (few: 3 to 7); then as many as there are places for.
// Measured on inputs in L2, us, one part and by the rule (where it makes none: in parts): 256 of 4 heads over 2 on 1024 (14.6; 15.6), on 1280 16.1, 15.4; 1024 of 4 heads on 1024
// (14.8; 16.9), on 2048 21.8, 19.2; one head of 2048 x 2048 21.5, 16.1; 33 on 4000, 28 heads over 4 35.3, 16.6; 300 on 4000, 4 heads 35.6, 17.9; 128 on 65536, one head 445, 20.5 (32
// parts 27).
//
// Few rows, 32 heads over 8: the single form and this one, single queries on keys for all lengths from one on: 128 on up to 1024 92, 68; 64 on up to 8192 186, 183; 20 on up to 16384 134, 123;
// 16 on up to 4096 39, 41; 8 heads of 64 channels, 256 on up to 2048 184, 125. On 4096 keys one query 15, 12; 16 each 50, 50. Where lengths differ a CTA of a long sequence
// would be waited for, hence parts of about 16 tiles there, for no more than 7 CTAs to a place, whatever the lengths, which only the GPU knows: in one part 64 on up to 8192 198 and 20 on
// up to 16384 211, but of 8192 keys each 64 take 316 and not 327. One query on 768 keys in one part 13.6, by the rule 10.2; on 512 10.5 in one, which stays so.
struct ForwardPlan {
  AttnForm form;
  int splits;
};
static double estimate(double ctas, int sms, double mean, double longest, double constant) {
  // (CTAs of different lengths, the longest first, leave less than half of a last wave empty)
  const double waves = mean < 0.9 * longest ? std::min(std::ceil(ctas / sms), ctas / sms + 0.5) : std::ceil(ctas / sms);
  return std::max(waves * mean, longest) + waves * constant;
}
static ForwardPlan forwardPlan(const ncclCpContext* cp, const ncclCpAttention_t* c) {
  AttnArgs a;
  fillAttention(c, nullptr, nullptr, &a);
  const long long owners = (long long)c->batch * c->kv_heads, ctas = owners * a.tiles, pairCtas = owners * ((a.tiles + 1) / 2);
  const int sms = cp->smCount;
  // tiles of keys that the last and the first tile of queries see (all rows of all sequences being there)
  const long long offset = c->mask == NCCL_CP_CAUSAL_END ? (long long)c->kv_tokens - c->q_tokens : a.offset;
  const auto tilesUpTo = [&](long long tok) { return (double)((c->mask == NCCL_CP_FULL ? c->kv_tokens : std::max(0ll, std::min<long long>(c->kv_tokens, tok + offset))) + 127) / 128; };
  const double longest = std::floor(tilesUpTo(c->q_tokens)), mean = (longest + std::floor(tilesUpTo(a.tileTokens))) / 2;
  ForwardPlan p;
  const bool pairs = a.tiles > 1 && estimate(pairCtas, sms, mean, longest, 1.0) <= estimate(ctas, sms, 1.15 * mean / 2, 1.15 * longest / 2, 2.0);
  p.form = pairs ? ATTN_PAIRS : a.tiles * a.tileTokens * a.group <= kFewRows ? ATTN_FEW : ATTN_SINGLE;
  p.splits = 1;
  const int places = p.form == ATTN_FEW ? 2 * sms : sms;
  if (pairs || !ctas) return p;
  long long most = places / ctas;
  if (p.form == ATTN_FEW) most = std::max(most, std::min((long long)longest / 16, 7 * places / ctas));
  most = std::min({most, (long long)longest / 2, (long long)kAttnMaxSplits});
  if (most > 1 && longest * (1.0 - 1.0 / most) > (p.form == ATTN_FEW ? 3.0 : 5.0) + std::min(4.0, (double)c->batch * c->q_tokens * c->heads / 500)) p.splits = (int)most;
  return p;
}
// How many threads share four channels of a row's parts in the kernel that joins them: as many as there are parts while that makes no more than 512 threads for an SM, and for each no
// more than kAttnJoinTurns parts. One head of 2048 x 2048 in 8 parts takes 16.1 us so, with up to 1024 threads 17.2, with 2048 20.0, with a thread for each part 26.4.
static int joinShares(const ncclCpContext* cp, size_t rows, int quads, int splits) {
  int shares = 1;
  while (shares * kAttnJoinTurns < splits || (2 * shares <= std::min(256 / quads, splits) && 2 * shares * rows * quads <= (size_t)cp->smCount * 512)) shares *= 2;
  return shares;
}
static size_t forwardWork(const ncclCpAttention_t* c, const ForwardPlan& p) {
  return p.splits == 1 ? 0 : (size_t)p.splits * c->batch * c->q_tokens * c->heads * (c->head_dim + 1) * 4;
}

// Into how many parts a backward call cuts the partners of its tiles: where CTAs are few, and the longest of them would be waited for. In units of what a CTA that owns queries takes
// for a tile of keys (1.1 us; one that owns keys takes 1.3 of that for a tile of queries): what all CTAs take on all SMs and half of a last one beside others, the longest one at least, a
// constant for a CTA's beginning and end, and for parts a launch and the traffic of their sums, once there and once back. Measured with inputs from memory, us, without parts and by
// this rule: 2048 causal tokens of 32 heads over one 735, 135; 4096 of 8 over 2 205, 131; 128 queries on 16384 keys of 8 heads 211, 104; 33 on 4000, 28 heads over 4, causal 63, 43;
// 512 causal tokens of 8 heads over one, 64 channels 55, 23; where it makes none parts would cost: 509 x 641, 3 times 12 heads over 4, 96 channels 53, in two parts 62 and more.
//
// Gradients have two roundings to 16 bits: of ds (dv: of the probabilities) and of what is stored, 1.4 times the second alone on average. Where an output has few rows, or few terms
// that cancel, that is 1.55 times now and then. Calls that do not fill the GPU multiply what the first rounding left as well ("fine"). Each product of tiles is made by two CTAs, one that
// owns the keys and one that owns the queries: while the SMs have a place for each of them, more products only make a CTA longer; beyond they add to what all SMs have to do. us, without
// and with, on 148 SMs: 1 query on 512 keys 16.0, 17.7; 2 x 256 causal tokens of 8 heads of 64 10.9, 12.7; 250 of 18 heads of 64 (72 products, with by this rule) 10.8, 12.8, of 19 (76,
// without) 10.8, 12.9; 512 of 8 heads (128) 18.5, 23.6, of 64 channels 13.4, 17.3; 1024 of 4 heads (256) 23.6, 36.4.
struct BackwardPlan {
  int kvParts, qParts;
};
static bool fineProducts(const ncclCpContext* cp, const ncclCpAttention_t* c, const AttnArgs& a) {
  return 2.0 * c->batch * c->kv_heads * a.tiles * a.vTiles <= cp->smCount;   // tiles of queries and of keys that meet, masks aside
}
static BackwardPlan backwardPlan(const ncclCpContext* cp, const ncclCpAttention_t* c, const AttnArgs& a) {
  const double owners = (double)c->batch * c->kv_heads, keyTiles = std::ceil(c->kv_tokens / 128.0), sms = cp->smCount;
  const long long offset = c->mask == NCCL_CP_CAUSAL_END ? (long long)c->kv_tokens - c->q_tokens : a.offset;
  // partners of the tile that has the most and of the one that has the fewest, all rows being there
  const auto keys = [&](long long tok) { return std::ceil((c->mask == NCCL_CP_FULL ? c->kv_tokens : std::max(0ll, std::min<long long>(c->kv_tokens, tok + offset))) / 128.0); };
  const auto queries = [&](long long key) { return std::ceil((c->mask == NCCL_CP_FULL ? c->q_tokens : std::max(0ll, std::min<long long>(c->q_tokens, c->q_tokens - key + offset))) / (double)a.tileTokens); };
  const double qLongest = keys(c->q_tokens), qMean = (qLongest + keys(a.tileTokens)) / 2, kvLongest = 1.3 * queries(0), kvMean = (kvLongest + 1.3 * queries(c->kv_tokens - 128)) / 2;
  const double dq = (double)c->batch * c->q_tokens * c->heads * c->head_dim * 4, dkv = (double)c->batch * c->kv_tokens * c->kv_heads * c->head_dim * 8, constant = 4.0;
  BackwardPlan best = {1, 1};
  if (owners * (keyTiles + a.tiles) > 4 * sms && std::max(kvLongest, qLongest) < (owners * (keyTiles * kvMean + a.tiles * qMean)) / sms) return best;   // enough to do for all
  double least = 0.0;
  for (int kvParts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    if (kvParts > 1 && kvParts * 2.6 > kvLongest) break;
    for (int qParts : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      if (qParts > 1 && qParts * 2 > qLongest) break;
      const double kvCtas = owners * keyTiles * kvParts, qCtas = owners * a.tiles * qParts, qEach = qMean / qParts + constant;
      const double all = (kvCtas * (kvMean / kvParts + constant) + qCtas * qEach) / sms + (kvCtas + qCtas > sms ? 0.5 * qEach : 0.0);
      double t = std::max({all, kvLongest / kvParts + constant, qLongest / qParts + constant});
      if (kvParts > 1 || qParts > 1) t += 2.5 + 2 * ((kvParts > 1 ? kvParts * dkv : 0.0) + (qParts > 1 ? qParts * dq : 0.0)) / 12e6;
      if (least == 0.0 || t < 0.95 * least) {
        least = t;
        best = {kvParts, qParts};
      }
    }
  }
  return best;
}

static size_t statsBytes(const AttnArgs& a) { return (size_t)a.batch * a.kvHeads * a.tiles * 256 * 4; }
static size_t boundsBytes(const ncclCpAttention_t* c, const AttnArgs& a) { return isFp16(c) ? ((size_t)c->batch * c->kv_heads * (2 * a.tiles + a.vTiles) * 4 + 255) / 256 * 256 : 0; }
static size_t dqBytes(const ncclCpAttention_t* c) { return (size_t)c->batch * c->q_tokens * c->heads * c->head_dim * 4; }
static size_t dkBytes(const ncclCpAttention_t* c) { return (size_t)c->batch * c->kv_tokens * c->kv_heads * c->head_dim * 4; }
// Numbers of each row, norms, and the sums of parts.
static size_t backwardWork(const ncclCpAttention_t* c, const AttnArgs& a, const BackwardPlan& p) {
  return statsBytes(a) + boundsBytes(c, a) + (p.qParts > 1 ? p.qParts * dqBytes(c) : 0) + (p.kvParts > 1 ? 2 * p.kvParts * dkBytes(c) : 0);
}

static ncclResult_t needsGpu(const ncclCpContext* cp, const char* what) {
  if (cp->comm->compCap < 100) { WARN("%s needs compute capability 10.0 (found %d)", what, cp->comm->compCap); return ncclInvalidUsage; }
  return ncclSuccess;
}

static ncclResult_t launchStats(ncclCpContext* cp, const ncclCpAttention_t* c, AttnStatsArgs* a, cudaStream_t stream) {
  const unsigned ctas = (unsigned)a->batch * a->kvHeads * (a->tiles + (a->bounds ? a->vTiles : 0));
  if (!ctas) return ncclSuccess;
  void* args[1] = {a};
  return launchCp(cp, attnStatsKernelFn(isFp16(c) ? ATTN_F16 : ATTN_BF16, c->head_dim), ctas, 1, 256, 0, args, stream);
}

static void fillStats(const ncclCpAttention_t* c, const AttnArgs& a, AttnStatsArgs* s) {
  memset(s, 0, sizeof(*s));
  s->batch = a.batch;
  s->q = a.q;
  s->kv = a.kv;
  s->heads = a.heads;
  s->kvHeads = a.kvHeads;
  s->dim = a.dim;
  s->group = a.group;
  s->tileTokens = a.tileTokens;
  s->tiles = a.tiles;
  s->vTiles = a.vTiles;
  s->qLengths = a.qLengths;
  s->kvLengths = a.kvLengths;
  memcpy(s->doutStride, c->dout_stride, sizeof(s->doutStride));
  memcpy(s->outStride, c->out_stride, sizeof(s->outStride));
  memcpy(s->vStride, c->v_stride, sizeof(s->vStride));
}

extern "C" {

ncclResult_t ncclCpCreate(ncclComm_t comm, ncclCp_t* out) {
  if (!out) return ncclInvalidArgument;
  *out = nullptr;
  if (!commValid(comm) || comm->hostOnly) { WARN("ncclCpCreate needs a GPU communicator"); return ncclInvalidArgument; }
  NCCLCHECK(commEnsureReady(comm));
  int sms = 0;
  CUDACHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, comm->cudaDev));
  ncclCpContext* cp = new (std::nothrow) ncclCpContext;
  if (!cp) return ncclSystemError;
  cp->comm = comm;
  cp->smCount = std::max(sms, 1);
  *out = cp;
  return ncclSuccess;
}

ncclResult_t ncclCpDestroy(ncclCp_t cp) {
  delete cp;
  return ncclSuccess;
}

size_t ncclCpAttentionWork(ncclCp_t cp, const ncclCpAttention_t* c) {
  if (!cp || checkShape("ncclCpAttentionWork", c) != ncclSuccess) return 0;
  return forwardWork(c, forwardPlan(cp, c));
}

ncclResult_t ncclCpAttention(ncclCp_t cp, const ncclCpAttention_t* c, const void* q, const void* k, const void* v, const int* qLengths, const int* kvLengths, const float* joinOut,
                             const float* joinLse, void* out, float* lse, void* work, cudaStream_t stream) {
  const char* what = "ncclCpAttention";
  if (!cp) return ncclInvalidArgument;
  NCCLCHECK(checkShape(what, c));
  NCCLCHECK(needsGpu(cp, what));
  if (!c->batch || !c->q_tokens) return ncclSuccess;
  NCCLCHECK(checkOperand(what, "q", q, c->batch, c->q_tokens, c->heads, c->q_stride));
  if (c->kv_tokens) {
    NCCLCHECK(checkOperand(what, "k", k, c->batch, c->kv_tokens, c->kv_heads, c->k_stride));
    NCCLCHECK(checkOperand(what, "v", v, c->batch, c->kv_tokens, c->kv_heads, c->v_stride));
  } else {
    k = v = q;   // not read
  }
  const ForwardPlan plan = forwardPlan(cp, c);
  const size_t rows = (size_t)c->batch * c->q_tokens * c->heads, workBytes = forwardWork(c, plan), lengthBytes = (size_t)c->batch * 4;
  if (!out || !lse || (workBytes && !work) || !joinOut != !joinLse || !aligned({out, joinOut}, 16) || !aligned({lse, joinLse, qLengths, kvLengths}, 4) || !aligned({work}, 256)) {
    WARN("%s: out, lse and (for %zu bytes) work must be there and aligned, join_out and join_lse come as a pair", what, workBytes);
    return ncclInvalidArgument;
  }
  const size_t outBytes = rows * c->head_dim * (c->result_type == ncclFloat32 ? 4 : 2);
  const Span joined = {(const void*)joinOut == out && c->result_type == ncclFloat32 ? nullptr : joinOut, rows * c->head_dim * 4};   // a row is read before it is written, by the same thread
  if (overlap({{out, outBytes}, {lse, rows * 4}, {workBytes ? work : nullptr, workBytes}},
              {spanOf(q, c->batch, c->q_tokens, c->heads, c->head_dim, c->q_stride, 2), c->kv_tokens ? spanOf(k, c->batch, c->kv_tokens, c->kv_heads, c->head_dim, c->k_stride, 2) : Span{nullptr, 0},
               c->kv_tokens ? spanOf(v, c->batch, c->kv_tokens, c->kv_heads, c->head_dim, c->v_stride, 2) : Span{nullptr, 0}, joined, {joinLse == lse ? nullptr : joinLse, rows * 4},
               {qLengths, lengthBytes}, {kvLengths, lengthBytes}})) {
    WARN("%s: an output shares memory with another tensor", what);
    return ncclInvalidArgument;
  }
  AttnArgs a;
  fillAttention(c, qLengths, kvLengths, &a);
  a.out = out;
  a.outFp32 = c->result_type == ncclFloat32;
  a.lse = lse;
  a.joinOut = joinOut;
  a.joinLse = joinLse;
  a.splits = plan.splits;
  a.partOut = (float*)work;
  a.partLse = (float*)work + (size_t)plan.splits * rows * c->head_dim;
  a.status = cp->comm->devStatusDev;
  const int type = isFp16(c) ? ATTN_F16 : ATTN_BF16;
  B200_ON_DEVICE(cp);
  CUtensorMap maps[3];
  NCCLCHECK(makeMap(&maps[0], c, q, c->q_tokens, c->heads, c->q_stride, a.tileTokens, a.group));
  NCCLCHECK(makeMap(&maps[1], c, k, c->kv_tokens, c->kv_heads, c->k_stride, kAttnRows, 1));
  NCCLCHECK(makeMap(&maps[2], c, v, c->kv_tokens, c->kv_heads, c->v_stride, kAttnRows, 1));
  void* args[4] = {&maps[0], &maps[1], &maps[2], &a};
  const unsigned grid = (unsigned)c->batch * c->kv_heads * (plan.form == ATTN_PAIRS ? (a.tiles + 1) / 2 : a.tiles) * plan.splits;
  NCCLCHECK(launchCp(cp, attnForwardKernelFn(type, c->head_dim, plan.form), grid, 1, attnForwardThreads(plan.form), attnForwardSmemBytes(c->head_dim, plan.form), args, stream,
                     attnForwardRegs(plan.form)));
  if (plan.splits == 1) return ncclSuccess;
  const int quads = c->head_dim / 4;
  a.joinShares = joinShares(cp, rows, quads, plan.splits);
  const int perCta = 256 / (quads * a.joinShares);
  void* join[1] = {&a};
  return launchCp(cp, attnJoinKernelFn(type), (unsigned)((rows + perCta - 1) / perCta), 1, 256, 0, join, stream);
}

size_t ncclCpAttentionBackwardWork(ncclCp_t cp, const ncclCpAttention_t* c) {
  if (!cp || checkShape("ncclCpAttentionBackwardWork", c) != ncclSuccess) return 0;
  AttnArgs a;
  fillAttention(c, nullptr, nullptr, &a);
  return backwardWork(c, a, backwardPlan(cp, c, a));
}

ncclResult_t ncclCpAttentionBackward(ncclCp_t cp, const ncclCpAttention_t* c, const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse,
                                     const float* delta, const int* qLengths, const int* kvLengths, const float* addDq, const float* addDk, const float* addDv, void* dq, void* dk,
                                     void* dv, void* work, cudaStream_t stream) {
  const char* what = "ncclCpAttentionBackward";
  if (!cp) return ncclInvalidArgument;
  NCCLCHECK(checkShape(what, c));
  NCCLCHECK(needsGpu(cp, what));
  if (!c->batch || (!c->q_tokens && !c->kv_tokens)) return ncclSuccess;
  const bool some = c->q_tokens && c->kv_tokens;
  const size_t rows = (size_t)c->batch * c->q_tokens * c->heads, cols = (size_t)c->batch * c->kv_tokens * c->kv_heads, lengthBytes = (size_t)c->batch * 4;
  const size_t size = c->result_type == ncclFloat32 ? 4 : 2, D = c->head_dim;
  AttnArgs a;
  fillAttention(c, qLengths, kvLengths, &a);
  const BackwardPlan plan = backwardPlan(cp, c, a);
  const size_t workBytes = backwardWork(c, a, plan);
  if (c->q_tokens) {
    NCCLCHECK(checkOperand(what, "q", q, c->batch, c->q_tokens, c->heads, c->q_stride));
    NCCLCHECK(checkOperand(what, "d_out", dout, c->batch, c->q_tokens, c->heads, c->dout_stride));
    if (!delta || out) NCCLCHECK(checkOperand(what, "out", out, c->batch, c->q_tokens, c->heads, c->out_stride));
  }
  if (c->kv_tokens) {
    NCCLCHECK(checkOperand(what, "k", k, c->batch, c->kv_tokens, c->kv_heads, c->k_stride));
    NCCLCHECK(checkOperand(what, "v", v, c->batch, c->kv_tokens, c->kv_heads, c->v_stride));
  }
  const bool adds = addDq || addDk || addDv;
  if ((c->q_tokens && (!lse || !dq)) || (c->kv_tokens && (!dk || !dv)) || (workBytes && !work) || (adds && ((c->q_tokens && !addDq) || (c->kv_tokens && (!addDk || !addDv)))) ||
      !aligned({dq, dk, dv, addDq, addDk, addDv}, 16) || !aligned({lse, delta, qLengths, kvLengths}, 4) || !aligned({work}, 256)) {
    WARN("%s: lse, d_q, d_k, d_v and work must be there and aligned, add_dq, add_dk and add_dv come together", what);
    return ncclInvalidArgument;
  }
  // a gradient's row is read before it is written, by the same thread
  const auto added = [&](const float* p, const void* to, size_t n) { return Span{(const void*)p == to && size == 4 ? nullptr : p, n * D * 4}; };
  const auto operand = [&](const void* p, int tokens, int heads, const long long* stride) { return tokens ? spanOf(p, c->batch, tokens, heads, c->head_dim, stride, 2) : Span{nullptr, 0}; };
  if (overlap({{dq, rows * D * size}, {dk, cols * D * size}, {dv, cols * D * size}, {workBytes ? work : nullptr, workBytes}},
              {operand(q, c->q_tokens, c->heads, c->q_stride), operand(dout, c->q_tokens, c->heads, c->dout_stride), operand(out, c->q_tokens, c->heads, c->out_stride),
               operand(k, c->kv_tokens, c->kv_heads, c->k_stride), operand(v, c->kv_tokens, c->kv_heads, c->v_stride), {lse, rows * 4}, {delta, rows * 4}, {qLengths, lengthBytes},
               {kvLengths, lengthBytes}, added(addDq, dq, rows), added(addDk, dk, cols), added(addDv, dv, cols)})) {
    WARN("%s: an output shares memory with another tensor", what);
    return ncclInvalidArgument;
  }
  const int type = isFp16(c) ? ATTN_F16 : ATTN_BF16;
  a.gradFp32 = size == 4;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.addDq = addDq;
  a.addDk = addDk;
  a.addDv = addDv;
  a.stats = (const float*)work;
  a.bounds = isFp16(c) ? (const uint32_t*)((const char*)work + statsBytes(a)) : nullptr;
  a.kvParts = plan.kvParts;
  a.qParts = plan.qParts;
  a.partDq = (float*)((char*)work + statsBytes(a) + boundsBytes(c, a));
  a.partDk = (float*)((char*)a.partDq + (plan.qParts > 1 ? plan.qParts * dqBytes(c) : 0));
  a.partDv = (float*)((char*)a.partDk + plan.kvParts * dkBytes(c));
  a.status = cp->comm->devStatusDev;
  B200_ON_DEVICE(cp);
  if (some) {
    AttnStatsArgs s;
    fillStats(c, a, &s);
    s.dout = dout;
    s.out = out;
    s.v = v;
    s.lse = lse;
    s.delta = delta;
    s.stats = (float*)work;
    s.bounds = (uint32_t*)a.bounds;
    NCCLCHECK(launchStats(cp, c, &s, stream));
  }
  if (!c->q_tokens) q = dout = k;   // not read
  if (!c->kv_tokens) k = v = q;
  CUtensorMap maps[6];
  NCCLCHECK(makeMap(&maps[0], c, q, c->q_tokens, c->heads, c->q_stride, a.tileTokens, a.group));
  NCCLCHECK(makeMap(&maps[1], c, dout, c->q_tokens, c->heads, c->dout_stride, a.tileTokens, a.group));
  NCCLCHECK(makeMap(&maps[2], c, k, c->kv_tokens, c->kv_heads, c->k_stride, kAttnRows, 1));
  NCCLCHECK(makeMap(&maps[3], c, v, c->kv_tokens, c->kv_heads, c->v_stride, kAttnRows, 1));
  void* args[5] = {&maps[0], &maps[1], &maps[2], &maps[3], &a};
  const unsigned owners = (unsigned)c->batch * c->kv_heads, keyTiles = (c->kv_tokens + kAttnRows - 1) / kAttnRows;
  a.kvCtas = owners * keyTiles * plan.kvParts;
  NCCLCHECK(launchCp(cp, attnBackwardKernelFn(type, c->head_dim, fineProducts(cp, c, a)), a.kvCtas + owners * a.tiles * plan.qParts, 1, attnBackwardThreads(),
                     attnBackwardSmemBytes(c->head_dim), args, stream, attnBackwardRegs()));
  const size_t sumRows = (plan.qParts > 1 ? rows : 0) + (plan.kvParts > 1 ? 2 * cols : 0);
  if (!sumRows) return ncclSuccess;
  void* sum[1] = {&a};
  return launchCp(cp, attnSumKernelFn(type), (unsigned)((sumRows * (D / 4) + 255) / 256), 1, 256, 0, sum, stream);
}

ncclResult_t ncclCpAttentionDelta(ncclCp_t cp, const ncclCpAttention_t* c, const void* dout, const void* out, const int* qLengths, float* delta, cudaStream_t stream) {
  const char* what = "ncclCpAttentionDelta";
  if (!cp) return ncclInvalidArgument;
  NCCLCHECK(checkShape(what, c));
  if (!c->batch || !c->q_tokens) return ncclSuccess;
  NCCLCHECK(checkOperand(what, "d_out", dout, c->batch, c->q_tokens, c->heads, c->dout_stride));
  NCCLCHECK(checkOperand(what, "out", out, c->batch, c->q_tokens, c->heads, c->out_stride));
  if (!delta || !aligned({delta, qLengths}, 4)) return ncclInvalidArgument;
  if (overlap({{delta, (size_t)c->batch * c->q_tokens * c->heads * 4}}, {spanOf(dout, c->batch, c->q_tokens, c->heads, c->head_dim, c->dout_stride, 2),
                                                                          spanOf(out, c->batch, c->q_tokens, c->heads, c->head_dim, c->out_stride, 2), {qLengths, (size_t)c->batch * 4}})) {
    WARN("%s: delta shares memory with another tensor", what);
    return ncclInvalidArgument;
  }
  AttnArgs a;
  fillAttention(c, qLengths, nullptr, &a);
  AttnStatsArgs s;
  fillStats(c, a, &s);
  s.dout = dout;
  s.out = out;
  s.deltaOut = delta;
  B200_ON_DEVICE(cp);
  return launchStats(cp, c, &s, stream);
}

// ---------------------------------------------------------------- rotary positions
ncclResult_t ncclCpRotary(ncclCp_t cp, const ncclCpRotary_t* c, const void* x0, const void* x1, void* y0, void* y1, const void* positions, const double* turns, cudaStream_t stream) {
  const char* what = "ncclCpRotary";
  if (!cp) return ncclInvalidArgument;
  if (!c || c->magic != NCCL_CP_MAGIC || c->size != sizeof(*c)) { WARN("%s: shape was not initialised", what); return ncclInvalidArgument; }
  const int type = c->type == ncclFloat16 ? ATTN_F16 : c->type == ncclBfloat16 ? ATTN_BF16 : c->type == ncclFloat32 ? ATTN_F32 : -1;
  if (type < 0) { WARN("%s: tensors must be fp16, bf16 or fp32", what); return ncclInvalidArgument; }
  const int size = type == ATTN_F32 ? 4 : 2, E = 16 / size;
  if (c->batch < 0 || c->tokens < 0 || c->head_dim <= 0 || c->half <= 0 || c->half > 512 || 2 * c->half > c->head_dim || c->heads[0] <= 0 || c->heads[1] < 0 || c->head_dim > 1 << 20 ||
      (long long)c->batch * c->tokens > 0x7fffffff || ((long long)c->heads[0] + c->heads[1]) * c->head_dim > 1 << 30) {
    WARN("%s: batch %d, %d tokens (2^31 together), %d and %d heads of %d channels, %d pairs (at most 512)", what, c->batch, c->tokens, c->heads[0], c->heads[1], c->head_dim, c->half);
    return ncclInvalidArgument;
  }
  if (!std::isfinite(c->amplitude)) { WARN("%s: amplitude must be finite", what); return ncclInvalidArgument; }
  if (!c->batch || !c->tokens) return ncclSuccess;
  if (!x0 || !y0 || (c->heads[1] && (!x1 || !y1)) || !turns || !aligned({turns}, 8) || !aligned({positions}, c->positions64 ? 8 : 4) || !aligned({x0, y0, c->heads[1] ? x1 : nullptr, c->heads[1] ? y1 : nullptr}, size)) {
    WARN("%s: tensors must be there and aligned to their elements", what);
    return ncclInvalidArgument;
  }
  RotaryArgs a;
  memset(&a, 0, sizeof(a));
  Span in[2] = {}, out[2] = {};
  bool inPlace[2] = {};
  int sizes[2][3];
  a.wide = c->head_dim % E == 0 && (c->interleaved ? 2 * c->half : c->half) % E == 0;
  const int tensors = c->heads[1] ? 2 : 1;
  for (int t = 0; t < tensors; ++t) {
    a.x[t] = t ? x1 : x0;
    a.y[t] = t ? y1 : y0;
    a.heads[t] = c->heads[t];
    for (int i = 0; i < 3; ++i) sizes[t][i] = i == 0 ? c->batch : i == 1 ? c->tokens : c->heads[t];
    inPlace[t] = a.x[t] == a.y[t];
    for (int i = 0; i < 3; ++i) {
      const long long xs = c->x_stride[t][i], ys = c->y_stride[t][i];
      if (sizes[t][i] > 1) {
        if (xs < 0 || xs >= 1ll << 40 || ys < c->head_dim || ys >= 1ll << 40) { WARN("%s: strides must not be negative, and rows of a result not overlap", what); return ncclInvalidArgument; }
        a.wide = a.wide && xs % E == 0 && ys % E == 0;
        inPlace[t] = inPlace[t] && xs == ys;
      }
      a.inStride[t][i] = sizes[t][i] > 1 ? xs : 0;
      a.outStride[t][i] = sizes[t][i] > 1 ? ys : 0;
    }
    if (!nest(sizes[t], a.outStride[t], 7, c->head_dim)) { WARN("%s: rows of a result overlap", what); return ncclInvalidArgument; }
    a.wide = a.wide && aligned({a.x[t], a.y[t]}, 16);
    in[t] = spanOf(a.x[t], c->batch, c->tokens, c->heads[t], c->head_dim, a.inStride[t], size);
    out[t] = spanOf(a.y[t], c->batch, c->tokens, c->heads[t], c->head_dim, a.outStride[t], size);
  }
  const Span other[2] = {{positions, (size_t)0}, {turns, (size_t)c->half * 8}};
  for (int t = 0; t < tensors; ++t) {
    bool bad = meets(out[t], other[1]);
    if (positions) {
      const long long s0 = c->batch > 1 ? c->position_stride[0] : 0, s1 = c->tokens > 1 ? c->position_stride[1] : 0;
      if (s0 < 0 || s1 < 0 || s0 >= 1ll << 40 || s1 >= 1ll << 40) { WARN("%s: strides must not be negative", what); return ncclInvalidArgument; }
      bad = bad || meets(out[t], {positions, ((size_t)(c->batch - 1) * s0 + (size_t)(c->tokens - 1) * s1 + 1) * (c->positions64 ? 8 : 4)});
    }
    // a tensor that is turned in place may lie between another's rows (one projection's queries and keys), not on them
    for (int u = 0; u < tensors; ++u) {
      if (!inPlace[t]) bad = bad || meets(out[t], in[u]);
      else if (u != t) bad = bad || !apart({a.y[t], sizes[t], a.outStride[t]}, {a.x[u], sizes[u], a.inStride[u]}, c->head_dim, size);
      if (u != t && !(inPlace[t] && inPlace[u])) bad = bad || meets(out[t], out[u]);
    }
    if (bad) { WARN("%s: an output shares memory with another tensor", what); return ncclInvalidArgument; }
  }
  a.batch = c->batch;
  a.tokens = c->tokens;
  a.dim = c->head_dim;
  a.half = c->half;
  a.positions = positions;
  a.positionStride[0] = c->position_stride[0];
  a.positionStride[1] = c->position_stride[1];
  a.positions64 = c->positions64;
  a.offset = c->offset;
  a.turns = turns;
  a.amplitude = c->amplitude;
  a.interleaved = c->interleaved != 0;
  a.inverse = c->inverse != 0;
  B200_ON_DEVICE(cp);
  // A CTA takes as many tokens as it computes angles for at a time; where tokens are few, several share the heads of one.
  const int tokens = c->batch * c->tokens, heads = c->heads[0] + c->heads[1], width = a.wide ? E : 1;
  a.items = (a.interleaved && a.wide ? 2 * a.half : a.half) / width + (a.dim - 2 * a.half) / width;
  const int most = std::max(1, kRotaryAngles / a.half);
  a.tokensAtOnce = std::max(1, std::min(most, tokens / (4 * cp->smCount)));
  const int blocks = (tokens - 1) / a.tokensAtOnce + 1;   // (tokens may be 2^31 - 1)
  const int shares = std::max(1, std::min({cp->smCount / blocks, (heads * a.items + 255) / 256, 64}));
  void* args[1] = {&a};
  return launchCp(cp, rotaryKernelFn(type), (unsigned)blocks, (unsigned)shares, 256, 0, args, stream);
}

}  // extern "C"
