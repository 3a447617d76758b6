/*
 * Operators of attention over a sequence that is cut across ranks, on sm_100a: what a rank computes on its own rows of the sequence and
 * on the blocks of keys and values that come to it (ring of ncclSend / ncclRecv) or on its heads of the whole sequence
 * (ncclAlltoAll before and after).
 *
 *   ncclCpRotary              rotary positions of queries and keys, and of their gradients
 *   ncclCpAttention           softmax(scale q k^T) v and its log-sum-exp; can join what other keys gave
 *   ncclCpAttentionBackward   gradients, with the probabilities computed again; can add to gradients under way
 *   ncclCpAttentionDelta      the one number per row that all of a row's backward calls share
 *
 * All are local to the communicator's GPU, run in stream order and need no other rank. They extend the reference API, which has no compute
 * kernels: it serves such programs through ncclSend / ncclRecv and ncclAlltoAll.
 */
#ifndef NCCL_CP_H_
#define NCCL_CP_H_

#include "nccl.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ncclCpContext* ncclCp_t;

ncclResult_t ncclCpCreate(ncclComm_t comm, ncclCp_t* cp);
ncclResult_t ncclCpDestroy(ncclCp_t cp);

#define NCCL_CP_MAGIC 0xc9a77e17u

/* Which keys a query sees, beside those behind its sequence's last. */
typedef enum {
  NCCL_CP_FULL = 0,          /* all */
  NCCL_CP_CAUSAL = 1,        /* query i: keys j <= i + offset (offset: how far the block of queries lies behind the block of keys) */
  NCCL_CP_CAUSAL_END = 2     /* the same with offset = keys - queries of the sequence: the last query sees every key */
} ncclCpMask_t;

/* Sizes of a call: queries [batch, q_tokens, heads, head_dim], keys and values [batch, kv_tokens, kv_heads, head_dim]; head h reads key head
 * h / (heads / kv_heads). type: ncclFloat16 or ncclBfloat16. Strides of batch, token and head in elements: positive multiples of 8, channels next to each
 * other, addresses of 16 bytes. head_dim: a multiple of 8, at most 128; heads / kv_heads: at most 128. scale: positive and finite. */
typedef struct {
  unsigned int size;
  unsigned int magic;
  ncclDataType_t type;
  ncclDataType_t result_type;   /* of out, or of the gradients: `type` or ncclFloat32 */
  int batch, q_tokens, kv_tokens, heads, kv_heads, head_dim;
  ncclCpMask_t mask;
  float scale;
  long long offset;
  long long q_stride[3], k_stride[3], v_stride[3];
  long long dout_stride[3], out_stride[3];   /* backward: of d_out and of out */
} ncclCpAttention_t;

/* out [batch, q_tokens, heads, head_dim] (contiguous) and lse [batch, heads, q_tokens] (fp32, natural logarithm; -inf and a row of zeros where a query sees
 * no key). q_lengths, kv_lengths: int32 [batch] on the device, or null: how many rows of each sequence are there. Rows behind them
 * may hold anything; their results are zeros (lse: -inf). join_out (fp32, laid out like out) and join_lse, or null: the result over other keys, which
 * this one is joined with; they may be out and lse. work: ncclCpAttentionWork bytes, aligned to 256 (null for none); not
 * read by later calls. */
size_t ncclCpAttentionWork(ncclCp_t cp, const ncclCpAttention_t* shape);
ncclResult_t ncclCpAttention(ncclCp_t cp, const ncclCpAttention_t* shape, const void* q, const void* k, const void* v, const int* q_lengths, const int* kv_lengths,
                             const float* join_out, const float* join_lse, void* out, float* lse, void* work, cudaStream_t stream);

/* d_q, d_k, d_v: contiguous, laid out like q, k and v, of result_type; rows behind the lengths are zeros. out and lse: the result over ALL keys of the queries (of a ring: the
 * joined one). delta (fp32 [batch, heads, q_tokens]): what ncclCpAttentionDelta gives, or null: computed from out. With delta, out may be null. add_dq, add_dk, add_dv
 * (fp32, all three or none): gradients so far, to which these are added; they may be d_q, d_k and d_v. The order of all sums is fixed. */
size_t ncclCpAttentionBackwardWork(ncclCp_t cp, const ncclCpAttention_t* shape);
ncclResult_t ncclCpAttentionBackward(ncclCp_t cp, const ncclCpAttention_t* shape, const void* d_out, const void* q, const void* k, const void* v, const void* out, const float* lse,
                                     const float* delta, const int* q_lengths, const int* kv_lengths, const float* add_dq, const float* add_dk, const float* add_dv, void* d_q,
                                     void* d_k, void* d_v, void* work, cudaStream_t stream);
/* delta = <d_out, out> of each row (zero behind the lengths). A gradient of lse itself is subtracted from it, whatever its size; of queries that see no key delta is not used. */
ncclResult_t ncclCpAttentionDelta(ncclCp_t cp, const ncclCpAttention_t* shape, const void* d_out, const void* out, const int* q_lengths, float* delta, cudaStream_t stream);

/* Rotary positions. The first 2 * half channels of a head are pairs (i, i + half), with `interleaved` (2 i, 2 i + 1); pair (a, b) becomes
 * amplitude * (a cos - b sin, b cos + a sin) at the angle 2 pi * position * turns[i], with `inverse` at the angle's negative (which is also how gradients go back).
 * Channels behind them are copied. turns: `half` fp64 on the device. Up to two tensors (queries and keys) [batch, tokens, heads, head_dim] of type
 * fp16, bf16 or fp32 with strides of batch, token and head; x[1] and heads[1] may be null and 0. y may be x with the same strides. positions: [batch, tokens] int32 or (positions64)
 * int64 with strides, or null: offset + token. */
typedef struct {
  unsigned int size;
  unsigned int magic;
  ncclDataType_t type;
  int batch, tokens, head_dim, half;
  int heads[2];
  int interleaved, inverse, positions64;
  float amplitude;
  long long offset;
  long long position_stride[2];
  long long x_stride[2][3], y_stride[2][3];
} ncclCpRotary_t;
ncclResult_t ncclCpRotary(ncclCp_t cp, const ncclCpRotary_t* shape, const void* x0, const void* x1, void* y0, void* y1, const void* positions, const double* turns, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
