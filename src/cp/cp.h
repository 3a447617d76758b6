// Internal interface between the host code of the context-parallel operators (cp.cc) and their kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

constexpr int kAttnRows = 128;       // rows of a tile: (token, head of a group) pairs of queries, or keys
constexpr int kAttnMaxDim = 128;     // channels of a head
constexpr int kAttnMaxTokens = 1 << 30;
constexpr int kAttnMaxSplits = 64;   // parts of the keys that CTAs work on at the same time
constexpr int kAttnJoinTurns = 8;    // of them, that a thread joins

// Rows of queries are packed: the heads that share keys and values lie next to each other, so that a tile holds `tileTokens` tokens of the `group` heads
// of one key head, row = token * group + head. tileTokens * group <= 128; rows behind that are nobody's.
struct AttnArgs {
  int batch, q, kv, heads, kvHeads, dim;
  int group, tileTokens;
  int causal;                 // 0: no, 1: key j is visible to query i where j <= i + offset, 2: the same with offset = kv length - q length of the sequence
  int offset;
  float scale;
  const int* qLengths;        // [batch] or null
  const int* kvLengths;
  // forward
  void* out;                  // [batch][q][heads][dim], of the inputs' type or fp32
  int outFp32;
  float* lse;                 // [batch][heads][q]
  const float* joinOut;       // what other keys gave, or null
  const float* joinLse;
  int splits;                 // above 1: fp32 results of each part of the keys go to partOut [splits][batch * q * heads][dim], partLse [splits][rows]
  float* partOut;
  float* partLse;
  int joinShares;             // threads with the same channels of a row
  // backward
  const float* stats;         // [batch][kvHeads][tiles][2][128]: minus the log-sum-exp in units of log 2 and minus <d(out), out> of each row
  int tiles;                  // of the queries of a key head
  const uint32_t* bounds;     // fp16: [batch][kvHeads][tiles of queries: squared norm of the longest row of d(out), largest |delta|; then tiles of v: squared norm], as bits
  int vTiles;
  void *dq, *dk, *dv;         // contiguous, of the inputs' type or fp32
  int gradFp32;
  const float *addDq, *addDk, *addDv;
  unsigned kvCtas;            // the first CTAs, which own tiles of keys; the others own tiles of queries
  int kvParts, qParts;        // CTAs that share the queries of a tile of keys, the keys of a tile of queries: above 1 their fp32 sums go to
  float *partDk, *partDv;     // [kvParts][rows of dk][dim]
  float* partDq;              // [qParts][rows of dq][dim]
  uint32_t* status;           // {code, kind, what, CTA} of the communicator, written when a wait runs out
};

struct AttnStatsArgs {
  const void *dout, *out, *v;
  long long doutStride[3], outStride[3], vStride[3];   // batch, token, head
  const float* lse;
  const float* delta;         // [batch][heads][q], or null: computed here
  float* deltaOut;            // only that, or null
  float* stats;
  uint32_t* bounds;           // fp16, else null
  int vTiles;
  int batch, q, kv, heads, kvHeads, dim, group, tileTokens, tiles;
  const int* qLengths;
  const int* kvLengths;
};

struct RotaryArgs {
  const void* x[2];           // [batch][tokens][heads][dim]
  void* y[2];
  long long inStride[2][3], outStride[2][3];           // batch, token, head
  int heads[2];
  const void* positions;      // [batch][tokens] of 32 or 64 bits, or null: offset + token
  long long positionStride[2];
  int positions64;
  long long offset;
  const double* turns;        // [half] turns of one step
  float amplitude;
  int batch, tokens, dim, half;
  int interleaved, inverse;
  int wide;                   // channels of a pack (16 bytes) may be moved together
  int tokensAtOnce;           // of a CTA
  int items;                  // of a head: packs (or channels) of both of a pair, and those that are copied
};
constexpr int kRotaryAngles = 256;   // of a CTA at a time

enum AttnType : int { ATTN_F16 = 0, ATTN_BF16 = 1, ATTN_F32 = 2 };
// Two tiles of queries for each CTA; one, whose keys its two halves share; or one of at most kFewRows rows, for two CTAs to an SM.
enum AttnForm : int { ATTN_PAIRS = 0, ATTN_SINGLE = 1, ATTN_FEW = 2 };
constexpr int kFewRows = 32;
// dim <= 64 or <= 128.
const void* attnForwardKernelFn(int type, int dim, AttnForm form);
size_t attnForwardSmemBytes(int dim, AttnForm form);
const void* attnJoinKernelFn(int type);
const void* attnBackwardKernelFn(int type, int dim, bool fine);
size_t attnBackwardSmemBytes(int dim);
int attnForwardThreads(AttnForm form);
int attnBackwardThreads();
int attnForwardRegs(AttnForm form);   // that a thread is launched with
int attnBackwardRegs();
const void* attnSumKernelFn(int type);
const void* attnStatsKernelFn(int type, int dim);
const void* rotaryKernelFn(int type);

}  // namespace b200
