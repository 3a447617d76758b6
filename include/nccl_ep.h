/*
 * Expert-parallel (MoE) dispatch / combine over a communicator.
 *
 * API shape of the reference extension (contrib/nccl_ep/include/nccl_ep.h): tensors are described
 * by ncclEpTensor_t, configuration structs start with {size, magic}, a group owns the symmetric
 * buffers, a handle owns the routing of one batch, dispatch sends tokens to the ranks of their
 * selected experts and combine brings the expert outputs back as a weighted sum.
 *
 * This implementation serves ranks that can map each other's memory (one NVLink domain) with one
 * fused kernel per direction; the layout of dispatched tokens is expert-major:
 *   tokens   [num_local_experts, num_ranks * max_dispatch_tokens_per_rank, hidden]
 *   scales   [num_local_experts, num_ranks * max_dispatch_tokens_per_rank, hidden / 128]  (fp8 dispatch)
 *   expert_counters[num_local_experts] = rows in use per expert.
 * Passing an output `scales` tensor selects fp8 (e4m3, one fp32 scale per 128 channels) dispatch.
 */
#ifndef NCCL_EP_H_
#define NCCL_EP_H_

#include "nccl.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NCCL_EP_MAJOR 0
#define NCCL_EP_MINOR 1
#define NCCL_EP_PATCH 0
#define NCCL_EP_VERSION_CODE (NCCL_EP_MAJOR * 10000 + NCCL_EP_MINOR * 100 + NCCL_EP_PATCH)
#define NCCL_EP_API_VERSION 1
#define NCCL_EP_MAGIC 0xC00FFFEEu
#define NCCL_EP_TENSOR_MAGIC 0xCAFECAFE
#define NCCL_EP_AUTO 0

typedef enum { NCCL_EP_ALGO_LOW_LATENCY = 0, NCCL_EP_ALGO_HIGH_THROUGHPUT = 1 } ncclEpAlgorithm_t;
typedef enum { NCCL_EP_LAYOUT_UNSET = NCCL_EP_AUTO, NCCL_EP_LAYOUT_EXPERT_MAJOR, NCCL_EP_LAYOUT_RANK_MAJOR, NCCL_EP_LAYOUT_FLAT } ncclEpLayout_t;
typedef enum { NCCL_EP_FWD_PASS = 0, NCCL_EP_BWD_PASS = 1 } ncclEpPassDir_t;

typedef struct ncclEpTensor {
  unsigned int size;
  unsigned int magic;
  unsigned int ndim;
  ncclDataType_t datatype;
  void* data;
  ncclWindow_t win_hdl;
  uint64_t win_offset;
  size_t* sizes;
} ncclEpTensor_t;

typedef struct { unsigned int size; unsigned int magic; } ncclEpTensorAllocConfig_t;

typedef cudaError_t (*ncclEpAllocFn_t)(void** ptr, size_t size, void* context);
typedef cudaError_t (*ncclEpFreeFn_t)(void* ptr, void* context);
typedef struct { ncclEpAllocFn_t alloc_fn; ncclEpFreeFn_t free_fn; void* context; } ncclEpAllocConfig_t;

typedef struct {
  unsigned int size;
  unsigned int magic;
  unsigned int version;
  ncclEpAlgorithm_t algorithm;
  unsigned int num_experts;
  unsigned int max_dispatch_tokens_per_rank;
  unsigned int max_recv_tokens_per_rank;
  unsigned int max_token_bytes;          /* bytes of one bf16 token row: 2 * hidden */
  unsigned long int rdma_buffer_size;
  unsigned int num_qp_per_rank;
  unsigned int num_channels;
  unsigned int max_num_sms;
  ncclEpAllocConfig_t alloc;
  unsigned int enable_mask;
  uint64_t timeout_ns;
} ncclEpGroupConfig_t;

typedef struct ncclEpGroup* ncclEpGroup_t;
typedef struct ncclEpHandle* ncclEpHandle_t;

typedef struct {
  unsigned int size;
  unsigned int magic;
  ncclEpTensor_t* expert_counters;
  ncclEpTensor_t* src_rank_counters;
  ncclEpTensor_t* expert_offsets;
  ncclEpTensor_t* recv_total_counter;
} ncclEpLayoutInfo_t;

typedef struct { unsigned int size; unsigned int magic; ncclEpTensor_t* tokens; ncclEpTensor_t* topk_weights; ncclEpTensor_t* scales; } ncclEpDispatchInputs_t;
typedef struct { unsigned int size; unsigned int magic; ncclEpTensor_t* tokens; ncclEpTensor_t* topk_weights; ncclEpTensor_t* scales; ncclEpTensor_t* topk_idx; } ncclEpDispatchOutputs_t;
typedef struct { unsigned int size; unsigned int magic; ncclEpTensor_t* tokens; ncclEpTensor_t* topk_weights; } ncclEpCombineInputs_t;
typedef struct { unsigned int size; unsigned int magic; ncclEpTensor_t* tokens; ncclEpTensor_t* topk_weights; } ncclEpCombineOutputs_t;
typedef struct { unsigned int size; unsigned int magic; size_t dispatch_output_per_expert_alignment; } ncclEpHandleConfig_t;
typedef struct { unsigned int size; unsigned int magic; unsigned int send_only; unsigned int round_scales; ncclEpPassDir_t pass_direction; } ncclEpDispatchConfig_t;
typedef struct { unsigned int size; unsigned int magic; unsigned int send_only; ncclEpPassDir_t pass_direction; } ncclEpCombineConfig_t;
typedef struct ncclEpCompleteConfig { unsigned int size; unsigned int magic; } ncclEpCompleteConfig_t;

ncclResult_t ncclEpGetVersion(int* version);
ncclResult_t ncclEpTensorAlloc(ncclEpTensor_t** tensor, unsigned int ndim, ncclDataType_t datatype, const size_t* sizes, const ncclEpTensorAllocConfig_t* config);
ncclResult_t ncclEpTensorDestroy(ncclEpTensor_t* tensor);
ncclResult_t ncclEpCreateGroup(ncclEpGroup_t* ep_group, ncclComm_t comm, const ncclEpGroupConfig_t* config);
ncclResult_t ncclEpGroupDestroy(ncclEpGroup_t ep_group);
ncclResult_t ncclEpHandleMemSize(ncclEpGroup_t ep_group, ncclEpLayout_t layout, const ncclEpHandleConfig_t* config, size_t* size_out, int num_topk);
ncclResult_t ncclEpInitHandle(ncclEpHandle_t* handle, ncclEpGroup_t ep_group, ncclEpLayout_t layout, const ncclEpHandleConfig_t* config, int num_topk, const ncclEpTensor_t* handle_mem);
ncclResult_t ncclEpUpdateHandle(ncclEpHandle_t handle, const ncclEpTensor_t* topk_idx, const ncclEpLayoutInfo_t* layout_info, cudaStream_t stream);
ncclResult_t ncclEpCreateHandle(ncclEpHandle_t* handle, ncclEpGroup_t ep_group, ncclEpLayout_t layout, const ncclEpTensor_t* topk_idx, const ncclEpLayoutInfo_t* layout_info, const ncclEpHandleConfig_t* config, cudaStream_t stream);
ncclResult_t ncclEpHandleDestroy(ncclEpHandle_t handle);
ncclResult_t ncclEpDispatch(ncclEpHandle_t handle, const ncclEpDispatchInputs_t* inputs, const ncclEpDispatchOutputs_t* outputs, const ncclEpLayoutInfo_t* layout_info, const ncclEpDispatchConfig_t* config, cudaStream_t stream);
ncclResult_t ncclEpCombine(ncclEpHandle_t handle, const ncclEpCombineInputs_t* inputs, const ncclEpCombineOutputs_t* outputs, const ncclEpCombineConfig_t* config, cudaStream_t stream);
ncclResult_t ncclEpComplete(ncclEpHandle_t handle, const ncclEpCompleteConfig_t* config, cudaStream_t stream);
ncclResult_t ncclEpMaskQuery(ncclEpGroup_t ep_group, int* mask_status, cudaStream_t stream);
ncclResult_t ncclEpMaskUpdate(ncclEpGroup_t ep_group, const int* mask, cudaStream_t stream);
ncclResult_t ncclEpMaskClean(ncclEpGroup_t ep_group, cudaStream_t stream);
ncclResult_t ncclEpGetAsyncError(ncclEpGroup_t ep_group, int* error_out);
ncclResult_t ncclEpErrorClear(ncclEpGroup_t ep_group);

/* ---- Operators of a mixture-of-experts layer around dispatch and combine -------------------------
 * All are local to this GPU, run in stream order and need no other rank; pointers are 16-byte aligned unless said otherwise. */

/* Routing. s = softmax or sigmoid of the logits [num_tokens, num_experts] (dispatch takes as many as its group has); experts are ranked by s + bias (fp32, or null),
 * and taken from the keep_groups best of `groups` equal runs of neighbouring experts (by the best expert's value, or the two best ones'
 * sum). topk_idx gets the num_topk best, best first, equal ones by index; topk_weights scale * s, divided by the sum over the taken
 * ones when `renormalize`. An expert whose logit (or s + bias) is -inf or NaN is never taken; an entry that finds none is -1, weight 0.
 * logits: fp32, fp16 or bf16, at their own alignment. At most 1024 experts, num_topk 16, groups 32. */
typedef enum { NCCL_EP_SCORE_SOFTMAX = 0, NCCL_EP_SCORE_SIGMOID = 1 } ncclEpScore_t;
typedef enum { NCCL_EP_GROUP_SCORE_MAX = 0, NCCL_EP_GROUP_SCORE_TOP2 = 1 } ncclEpGroupScore_t;
typedef struct { unsigned int size; unsigned int magic; ncclEpScore_t score; int groups; int keep_groups; ncclEpGroupScore_t group_score; int renormalize; float scale; } ncclEpRouteConfig_t;
ncclResult_t ncclEpRoute(ncclEpGroup_t ep_group, const void* logits, ncclDataType_t type, const float* bias, int64_t* topk_idx, float* topk_weights, int num_tokens, int num_experts, int num_topk, const ncclEpRouteConfig_t* config, cudaStream_t stream);
/* d(logits) (type of the logits, all of it written; it may take the logits' place) from d(topk_weights); of the configuration score, renormalize and scale count. */
ncclResult_t ncclEpRouteBackward(ncclEpGroup_t ep_group, const float* d_weights, const void* logits, ncclDataType_t type, const int64_t* topk_idx, void* d_logits, int num_tokens, int num_experts, int num_topk, const ncclEpRouteConfig_t* config, cudaStream_t stream);

/* The experts' products over rows packed as dispatch packs them (expert-major): for every expert e and its first counts[e] rows
 *   out[e] = act(x[e] w[e]^T + bias[e]) + residual[e]
 * x [experts, rows, k], w [experts, n, k], bias [experts, n], out and residual [experts, rows, n], all bf16; n and k are multiples of 8.
 * The gated activations take w as [gate rows | up rows] (n a multiple of 16) and give silu(gate) * up or gelu(gate) * up: out and residual have n / 2
 * columns. counts: int32 on the device, null: all rows. Rows behind an expert's last are neither read into a result nor written.
 * bias, residual and pre may be null; pre [experts, rows, n] gets x w^T + bias for the backward pass, in bf16, or in fp32 where
 * NCCL_EP_ACT_PRE_FP32 is added to the activation (gradients are then as exact as one rounding of the activation's gradient to bf16 leaves them).
 * residual may be out. At most 256 experts, and 2^24 rows, n and k. */
typedef enum { NCCL_EP_ACT_NONE = 0, NCCL_EP_ACT_RELU = 1, NCCL_EP_ACT_GELU = 2, NCCL_EP_ACT_SILU = 3, NCCL_EP_ACT_SWIGLU = 4, NCCL_EP_ACT_GEGLU = 5, NCCL_EP_ACT_PRE_FP32 = 256 } ncclEpActivation_t;
ncclResult_t ncclEpExpertLinear(ncclEpGroup_t ep_group, const void* x, const void* w, const int* counts, const void* bias, const void* residual, void* out, void* pre, int num_experts, int num_rows, int n, int k, ncclEpActivation_t activation, cudaStream_t stream);
/* Gradients: d_x [experts, rows, k] (the rows in use), d_w [experts, n, k] and d_bias [experts, n] (of every expert, zeros where it has no
 * rows), each unless null, all bf16. pre: as the forward call gave it, with the same activation (null without one). work: ncclEpExpertLinearBackwardWork bytes. */
size_t ncclEpExpertLinearBackwardWork(ncclEpGroup_t ep_group, int num_experts, int num_rows, int n, ncclEpActivation_t activation, int with_bias);
ncclResult_t ncclEpExpertLinearBackward(ncclEpGroup_t ep_group, const void* d_out, const void* x, const void* w, const int* counts, const void* pre, void* d_x, void* d_w, void* d_bias, void* work, int num_experts, int num_rows, int n, int k, ncclEpActivation_t activation, cudaStream_t stream);

/* Where the handle's last dispatch put each entry: rows [tokens, num_topk] int32, a row of [experts * capacity, hidden] or -1. Groups of one
 * rank, expert-major; the routing of that dispatch must still be in place. */
ncclResult_t ncclEpDispatchRows(ncclEpHandle_t handle, int* rows, cudaStream_t stream);
/* Gradients of combine: d_y[rows[t,k]] = weights[t,k] * d_out[t], d_weights[t,k] = <d_out[t], y[rows[t,k]]> (0 without a row). d_out [tokens, hidden], y and d_y
 * [num_rows, hidden] bf16, hidden a multiple of 8; rows of d_y that no entry names are not written, and d_y may be y where every row is named once. */
ncclResult_t ncclEpCombineBackward(ncclEpGroup_t ep_group, const void* d_out, const void* y, const float* weights, const int* rows, void* d_y, float* d_weights, int num_tokens, int num_topk, int hidden, int num_rows, cudaStream_t stream);
/* Gradient of dispatch: d_x[t] = sum over k of d_tokens[rows[t,k]], bf16 [tokens, hidden]. */
ncclResult_t ncclEpDispatchBackward(ncclEpGroup_t ep_group, const void* d_tokens, const int* rows, void* d_x, int num_tokens, int num_topk, int hidden, int num_rows, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
