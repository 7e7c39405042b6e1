/*
 * mi_experts: MI355X (gfx950) operators around the experts of a mixture-of-
 * experts layer, C ABI (libmi_experts.so). Unlike mi_moe.h, whose libraries
 * are built per layer definition, sizes here are arguments.
 *
 *   tokens to expert order and back:  mi_experts_sort, mi_experts_permute,
 *     mi_experts_unpermute, mi_experts_unpermute_backward
 *   8-bit integer products with a scale per token and per output channel:
 *     mi_experts_quantize_int8, mi_experts_int8_matmul
 *
 * All pointers are device pointers owned by the caller, workspaces included.
 * The library never allocates device memory, never synchronises the host,
 * keeps no pointer after a call, and enqueues all work on the given stream of
 * the current device. Every check runs before the first launch: a rejected
 * call enqueues nothing. Calls are reentrant; calls that run concurrently
 * need workspaces of their own. No counterpart in the reference, whose one
 * entry point is the whole layer.
 */
#ifndef MI_EXPERTS_H_
#define MI_EXPERTS_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes (those of mi_moe.h). */
#define MI_EXPERTS_OK 0
#define MI_EXPERTS_ERR_INVALID 1   /* bad pointer, size, alignment or type */
#define MI_EXPERTS_ERR_WORKSPACE 2 /* workspace too small */
#define MI_EXPERTS_ERR_HIP 3       /* a HIP launch failed */

/* Element types of float tensors. */
#define MI_EXPERTS_BF16 0
#define MI_EXPERTS_F32 1
#define MI_EXPERTS_F16 2

/* Limits: experts of a shard, experts per token, slots (tokens x top_k) and
 * the inner length of an integer product (|sum| <= 2^14 K stays in 32 bits). */
#define MI_EXPERTS_MAX_EXPERTS 1024
#define MI_EXPERTS_MAX_TOP_K 64
#define MI_EXPERTS_MAX_SLOTS (1 << 27)
#define MI_EXPERTS_MAX_K 131071

/* Slots sorted by local expert. topk_ids int32 [T, top_k] holds global expert
 * ids in any order (repeats allowed); ids outside [expert_offset,
 * expert_offset + num_experts) are another shard's. Rows are grouped by local
 * expert, ascending in t * top_k + j inside one; the slots of other shards
 * follow in the same order. Writes
 *   expert_offsets int32 [E+1]  first row of each expert; [E] = S, the local rows
 *   token_of_row int32 [T * top_k]
 *   row_of_slot int32 [T, top_k]
 * Stable and without atomics on memory: two calls give the same tables. */
size_t mi_experts_sort_workspace_size(int64_t num_slots, int32_t num_experts);
int mi_experts_sort(const int32_t* topk_ids, int64_t num_tokens, int32_t top_k, int32_t num_experts,
                    int64_t expert_offset, int32_t* expert_offsets, int32_t* token_of_row,
                    int32_t* row_of_slot, void* workspace, size_t workspace_bytes, void* stream);

/* rows[row_of_slot[t, j]] = x[t] for the slots whose row is below *num_rows
 * (expert_offsets + E of the sort). Rows at and past *num_rows are zeroed
 * with zero_rest, else left as they are. Any element type: rows are row_bytes
 * bytes, strides in bytes. rows has num_tokens * top_k rows. */
int mi_experts_permute(const void* x, int64_t x_stride, int64_t num_tokens, int32_t top_k,
                       int64_t row_bytes, const int32_t* row_of_slot, const int32_t* num_rows,
                       void* rows, int64_t rows_stride, int32_t zero_rest, void* stream);

/* out[t] = sum over j ascending of weights[t, j] * rows[row_of_slot[t, j]], in
 * fp32 and rounded once, over the slots whose row is below *num_rows; zeros
 * for a token without one. weights fp32 [T, top_k], or NULL for ones. Strides
 * in elements. This is also the gradient of mi_experts_permute (weights
 * NULL). */
int mi_experts_unpermute(int32_t dtype, const void* rows, int64_t rows_stride, int64_t num_tokens,
                         int32_t top_k, int64_t row_len, const int32_t* row_of_slot,
                         const int32_t* num_rows, const float* weights, void* out,
                         int64_t out_stride, void* stream);

/* Gradients of mi_experts_unpermute: grad_rows[row] = weights[t, j] * grad[t]
 * (rounded once; rows at and past *num_rows zeroed with zero_rest) and
 * grad_weights[t, j] = sum over columns of grad[t] * rows[row] in fp32, 0 for
 * slots of other shards. Either may be NULL; rows may be NULL without
 * grad_weights. */
int mi_experts_unpermute_backward(int32_t dtype, const void* grad, int64_t grad_stride,
                                  const void* rows, int64_t rows_stride, int64_t num_tokens,
                                  int32_t top_k, int64_t row_len, const int32_t* row_of_slot,
                                  const int32_t* num_rows, const float* weights, void* grad_rows,
                                  int64_t grad_rows_stride, int32_t zero_rest, float* grad_weights,
                                  void* stream);

/* int8 rows with a scale each: scale[m] = max(amax, 1e-10) / 127, q = x / scale
 * rounded to nearest even. swiglu: x has 2 * row_len columns and each row is
 * first silu(x[row_len:]) * x[:row_len] in fp32 (the layer's SwiGLU,
 * solution/triton/kernel.py:297-330). A row that holds a NaN or an infinity
 * gets a scale that is not finite and zeros, so its products are NaN. With
 * num_rows (device int32, may be NULL) rows at and past it get zeros (and a
 * scale of 0) with zero_rest, else they are left as they are. x_stride,
 * q_stride in elements. */
int mi_experts_quantize_int8(int32_t dtype, const void* x, int64_t x_stride, int64_t num_rows_max,
                             int64_t row_len, int32_t swiglu, const int32_t* num_rows,
                             int32_t zero_rest, int8_t* q, int64_t q_stride, float* scale,
                             void* stream);

/* out[m, n] = (sum_k a[m, k] * b[n, k]) * a_scale[m] * b_scale[n] + bias[n],
 * the sum exact in int32, the rest in fp32, rounded once to out's type.
 * num_experts = 0: b [N, K], a [M, K], out [M, N]. Else b [E, N, K], b_scale
 * [E, N], out row m (m < rows) has the expert whose [expert_offsets[e],
 * expert_offsets[e+1]) holds it, and rows before the first expert's and behind
 * the last one's are zeroed with zero_rest, else left as they are. row_ids (int32 [rows], may be NULL): row m of the product is row
 * row_ids[m] of a and of a_scale; an id outside [0, a_rows) gives NaN rows.
 * Offsets are clamped to [0, rows]. Any strides (in elements) and alignment;
 * 16-byte ones of a and b are fast. */
typedef struct mi_experts_int8_args {
    const int8_t* a;
    const float* a_scale;
    const int8_t* b;
    const float* b_scale;
    const void* bias;              /* [N] of bias_dtype, or NULL; dense products only */
    void* out;
    const int32_t* expert_offsets; /* [E+1], grouped products */
    const int32_t* row_ids;        /* [rows] or NULL, grouped products */
    int64_t a_rows;                /* rows of a; M of a dense product */
    int64_t rows;                  /* rows of out; = a_rows without row_ids */
    int64_t N, K;
    int64_t a_stride, b_stride, b_expert_stride, out_stride;
    int32_t num_experts;           /* 0: dense */
    int32_t out_dtype;             /* MI_EXPERTS_* */
    int32_t bias_dtype;
    int32_t zero_rest;             /* grouped products */
    void* workspace;               /* of the call below, 256-byte aligned; NULL where it says 0 */
    size_t workspace_bytes;
} mi_experts_int8_args;
/* 0 but for large dense products whose K is no multiple of 16: their rows are
 * copied to aligned ones first. */
size_t mi_experts_int8_workspace_size(int64_t rows, int64_t N, int64_t K, int32_t num_experts);
int mi_experts_int8_matmul(const mi_experts_int8_args* args, void* stream);

/* Message of the last error on the calling thread ("" if none). */
const char* mi_experts_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* MI_EXPERTS_H_ */
