/*
 * mi_layer: MI355X (gfx950) operators for the inside of a mixture-of-experts
 * layer of a caller's own, C ABI (libmi_layer.so). Sizes are arguments.
 *
 *   the router's balance loss:  mi_layer_balance, mi_layer_balance_backward
 *   the gate between an expert's products, with dropout:  mi_layer_swiglu,
 *     mi_layer_swiglu_backward
 *   products with 4-bit weights and a scale per group:  mi_layer_pack_int4,
 *     mi_layer_quantize_int4, mi_layer_int4_matmul
 *
 * The rules are those of mi_experts.h: all pointers are device pointers owned
 * by the caller, workspaces included; the library never allocates device
 * memory, never synchronises the host, keeps no pointer after a call, and
 * enqueues all work on the given stream of the current device. Every check
 * runs before the first launch. Calls are reentrant; calls that run
 * concurrently need workspaces of their own. No counterpart in the reference.
 */
#ifndef MI_LAYER_H_
#define MI_LAYER_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes and element types (those of mi_experts.h). */
#define MI_LAYER_OK 0
#define MI_LAYER_ERR_INVALID 1   /* bad pointer, size, alignment or type */
#define MI_LAYER_ERR_WORKSPACE 2 /* workspace too small */
#define MI_LAYER_ERR_HIP 3       /* a HIP launch failed */
#define MI_LAYER_BF16 0
#define MI_LAYER_F32 1
#define MI_LAYER_F16 2

#define MI_LAYER_MAX_EXPERTS 1024
#define MI_LAYER_MAX_TOP_K 64
#define MI_LAYER_SCORE_SOFTMAX 0
#define MI_LAYER_SCORE_SIGMOID 1

/* ------------------------------------------------------------ balance loss
 *
 * P[t, :] is the softmax of logits[t], or its sigmoids divided by their sum. A
 * row without a finite score (all -inf) has P = 0. Sequence s has the tokens
 * seq_offsets[s] .. seq_offsets[s + 1] - 1 (int32, non-decreasing; entries are
 * clamped to 0 .. num_tokens; tokens in no sequence do not count), or, with
 * seq_offsets NULL, one sequence has all. mask (NULL: all) holds a byte for
 * each token, 0: it does not count. With n_s the tokens of s that count and
 * c_se their slots in topk_ids [T, top_k] that name expert e (ids outside 0 ..
 * E - 1 count nowhere):
 *
 *   loss = mean over the sequences with n_s > 0 of
 *          sum_e (E c_se / (top_k n_s)) (sum_t P[t, e] / n_s)
 *
 * (0 if there is none). Writes loss[0], counts int32 [S, E], and weights fp32
 * [S, E] with dloss / dP[t, e] for a token t of s. Sums are fp32 in a fixed
 * order (per chunk of tokens, then over chunks): the same call gives the same
 * bits. */
typedef struct mi_layer_balance_args {
    const void* logits;         /* [T, E], rows logits_stride apart */
    const int32_t* topk_ids;    /* [T, top_k] contiguous */
    const int32_t* seq_offsets; /* [S + 1], or NULL (then num_seqs is 1) */
    const uint8_t* mask;        /* [T], or NULL */
    float* loss;                /* [1] */
    int32_t* counts;            /* [S, E] */
    float* weights;             /* [S, E] */
    int64_t num_tokens;
    int64_t num_seqs;
    int64_t logits_stride;
    int32_t num_experts;
    int32_t top_k;
    int32_t dtype;              /* of logits */
    int32_t score;              /* MI_LAYER_SCORE_* */
    void* workspace;
    size_t workspace_bytes;
} mi_layer_balance_args;
size_t mi_layer_balance_workspace_size(int64_t num_tokens, int64_t num_seqs, int32_t num_experts);
int mi_layer_balance(const mi_layer_balance_args* args, void* stream);

/* grad_logits[t, :] = *grad_loss * dloss / dlogits[t, :] (zeros for a token
 * that does not count), from what mi_layer_balance read and the weights it
 * wrote. args: logits, seq_offsets, mask, weights, sizes, dtype and score;
 * the other fields are not looked at. */
int mi_layer_balance_backward(const mi_layer_balance_args* args, const float* grad_loss,
                              void* grad_logits, int64_t grad_stride, void* stream);

/* ---------------------------------------------------- SwiGLU with dropout
 *
 * out[m, c] = silu(x[m, I + c]) x[m, c] keep(m, c) / (1 - p) for the rows m
 * below *num_rows (NULL: all max_rows); the others get zeros with zero_rest,
 * else stay as they are. p = threshold / 65536 (0: no dropout), and keep(m, c)
 * is 1 where the 16 random bits of the element are at least threshold. These
 * are the c % 8th of the eight 16-bit halves (low one first) of Philox4x32-10
 * (Salmon, Moraes, Dror, Shaw, SC 2011) with the counter (c / 8, m, 0, 0) and
 * the 64-bit seed as key, low word first. The seed is *seed_ptr (on the
 * device), or `seed` if seed_ptr is NULL. fp32 inside, rounded once. */
typedef struct mi_layer_swiglu_args {
    const void* x;            /* [max_rows, 2 I] */
    const void* grad;         /* backward: [max_rows, I] */
    void* out;                /* [max_rows, I]; backward: dx [max_rows, 2 I] */
    const int32_t* num_rows;  /* one number, or NULL */
    const uint64_t* seed_ptr; /* or NULL */
    uint64_t seed;
    int64_t max_rows;
    int64_t I;
    int64_t x_stride;
    int64_t grad_stride;
    int64_t out_stride;
    int32_t dtype;            /* of x, grad and out */
    int32_t threshold;        /* 0 .. 65535 */
    int32_t zero_rest;
    int32_t reserved;
} mi_layer_swiglu_args;
int mi_layer_swiglu(const mi_layer_swiglu_args* args, void* stream);
/* out = the gradient of x for `grad`, the gradient of the result. */
int mi_layer_swiglu_backward(const mi_layer_swiglu_args* args, void* stream);

/* ------------------------------------------------------- 4-bit weights
 *
 * Weights q in -8 .. 7 of E experts (0: one dense matrix) with N output
 * channels of K values, in two's complement, laid out in tiles of 16 channels
 * x 128 values, 1024 bytes each: 64 pieces of 16 bytes, of which piece 16 g + r
 * holds what channel r has of the values 32 s + 8 g .. 32 s + 8 g + 7 for s = 0
 * .. 3, a 32-bit word each (what lane 16 g + r of a wave multiplies, as one
 * load). Of the eight values of a word the even ones are its low four nibbles,
 * the odd ones its high four. Channels past N and values past K are 0. Tiles go
 * by k inside a row of tiles, those by n: ceil(N / 16) * ceil(K / 128) * 1024
 * bytes an expert. Scales [E, ceil(K / group_size), Np] in rows of Np = 16
 * ceil(N / 16), zeros past N.
 */
#define MI_LAYER_INT4_TILE_N 16
#define MI_LAYER_INT4_TILE_K 128
#define MI_LAYER_INT4_MIN_GROUP 32 /* group sizes are powers of two from here */

/* packed from q int8 [E, N, K] (values clamped to -8 .. 7), and scale_out in
 * rows of Np from scale [E, N, ceil(K / group_size)] of scale_dtype. */
int mi_layer_pack_int4(const int8_t* q, int64_t q_expert_stride, int64_t q_stride, const void* scale,
                       int32_t scale_dtype, int64_t num_experts, int64_t N, int64_t K,
                       int32_t group_size, uint8_t* packed, void* scale_out, void* stream);

/* packed and scale_out (fp32) from w [E, N, K]: scale = max(amax, 1e-10) / 7
 * of each group, q = w / scale rounded to nearest even. A group with a NaN or
 * an infinity has a scale that is not finite. */
int mi_layer_quantize_int4(int32_t dtype, const void* w, int64_t w_expert_stride, int64_t w_stride,
                           int64_t num_experts, int64_t N, int64_t K, int32_t group_size,
                           uint8_t* packed, float* scale_out, void* stream);

/* out[m, n] = sum over groups g of scale[g, n] (sum over k in g of x[m, k]
 * q[n, k]) + bias[n]: sums in fp32, rounded once. Dense with num_experts 0;
 * else row m has the weights of the expert e with expert_offsets[e] <= m <
 * expert_offsets[e + 1] (entries are clamped to 0 .. rows), and is row
 * row_ids[m] of x (row m if row_ids is NULL; an id that is no row gives NaN).
 * Rows that no expert has are zeroed with zero_rest, else left as they are. */
typedef struct mi_layer_int4_args {
    const void* x;                 /* [x_rows, K], bf16 or f16 */
    const uint8_t* w;              /* packed, 16-byte aligned */
    const void* scale;             /* fp32, or of x's type; 16-byte aligned */
    const void* bias;              /* [N], dense only, or NULL */
    void* out;                     /* [rows, N] */
    const int32_t* expert_offsets; /* [E + 1] */
    const int32_t* row_ids;        /* [rows] */
    int64_t x_rows;
    int64_t rows;
    int64_t N;
    int64_t K;
    int64_t x_stride;
    int64_t out_stride;
    int32_t group_size;
    int32_t num_experts;
    int32_t x_dtype;
    int32_t scale_dtype;
    int32_t bias_dtype;
    int32_t out_dtype;
    int32_t zero_rest;
    int32_t reserved;
    void* workspace;
    size_t workspace_bytes;
} mi_layer_int4_args;
/* A workspace is needed where rows of x do not start at multiples of 16 bytes
 * or K is no multiple of 8 (aligned: 0): x is copied to such rows. */
size_t mi_layer_int4_workspace_size(int64_t x_rows, int64_t K, int32_t aligned);
int mi_layer_int4_matmul(const mi_layer_int4_args* args, void* stream);

/* Message of the calling thread's last failed call. */
const char* mi_layer_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* MI_LAYER_H_ */
