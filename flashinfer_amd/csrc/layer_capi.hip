// extern "C" boundary of the layer's operators (include/mi_layer.h): every
// argument is checked before the first launch.
#include <stdarg.h>
#include <stdio.h>

#include "layer_common.hpp"

using namespace miexp;

namespace {

thread_local char g_last_error[512];

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
    va_end(ap);
    return code;
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p % a) == 0; }
bool float_type(int32_t d) { return d == MI_LAYER_BF16 || d == MI_LAYER_F32 || d == MI_LAYER_F16; }
size_t size_of(int32_t d) { return d == MI_LAYER_F32 ? 4 : 2; }

int hip_status(const char* who, hipError_t e) {
    if (e == hipSuccess) return MI_LAYER_OK;
    return fail(MI_LAYER_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
}

int check_workspace(const char* who, const void* workspace, size_t bytes, size_t need) {
    if (need && (!workspace || bytes < need))
        return fail(MI_LAYER_ERR_WORKSPACE, "%s: workspace has %zu bytes, needs %zu", who,
                    workspace ? bytes : (size_t)0, need);
    if (need && !aligned(workspace, 256)) return fail(MI_LAYER_ERR_INVALID, "%s: misaligned workspace", who);
    return MI_LAYER_OK;
}

// Sizes of the balance loss, those the workspace goes by among them.
bool balance_sizes(int64_t T, int64_t S, int32_t E) {
    return T >= 0 && T <= INT32_MAX && S >= 1 && S <= (1 << 20) && E >= 1 && E <= MI_LAYER_MAX_EXPERTS;
}

int check_balance(const char* who, const mi_layer_balance_args& a, bool backward) {
    if (!float_type(a.dtype)) return fail(MI_LAYER_ERR_INVALID, "%s: unknown dtype %d", who, a.dtype);
    if (a.score != MI_LAYER_SCORE_SOFTMAX && a.score != MI_LAYER_SCORE_SIGMOID)
        return fail(MI_LAYER_ERR_INVALID, "%s: unknown score %d", who, a.score);
    if (a.num_experts < 1 || a.num_experts > MI_LAYER_MAX_EXPERTS)
        return fail(MI_LAYER_ERR_INVALID, "%s: num_experts %d out of range 1..%d", who, a.num_experts,
                    MI_LAYER_MAX_EXPERTS);
    if (!backward && (a.top_k < 1 || a.top_k > MI_LAYER_MAX_TOP_K))
        return fail(MI_LAYER_ERR_INVALID, "%s: top_k %d out of range 1..%d", who, a.top_k, MI_LAYER_MAX_TOP_K);
    if (!balance_sizes(a.num_tokens, a.num_seqs, a.num_experts))
        return fail(MI_LAYER_ERR_INVALID, "%s: num_tokens %lld or num_seqs %lld out of range", who,
                    (long long)a.num_tokens, (long long)a.num_seqs);
    if (!a.seq_offsets && a.num_seqs != 1)
        return fail(MI_LAYER_ERR_INVALID, "%s: num_seqs %lld without seq_offsets", who, (long long)a.num_seqs);
    if (a.logits_stride < 0) return fail(MI_LAYER_ERR_INVALID, "%s: bad stride", who);
    if (!a.weights || (a.num_tokens > 0 && !a.logits)) return fail(MI_LAYER_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(a.logits, size_of(a.dtype)) || !aligned(a.seq_offsets, 4) || !aligned(a.weights, 4))
        return fail(MI_LAYER_ERR_INVALID, "%s: misaligned pointer", who);
    return MI_LAYER_OK;
}

int check_swiglu(const char* who, const mi_layer_swiglu_args& a, bool backward) {
    if (!float_type(a.dtype)) return fail(MI_LAYER_ERR_INVALID, "%s: unknown dtype %d", who, a.dtype);
    if (a.max_rows < 0 || a.max_rows > INT32_MAX)
        return fail(MI_LAYER_ERR_INVALID, "%s: %lld rows out of range", who, (long long)a.max_rows);
    // units of a row and 2048 columns, in 32 bits with room for the grid's step
    if (a.I < 1 || a.I > INT32_MAX / 8 || (a.max_rows + 1) * ((a.I + 2047) / 2048) > INT32_MAX)
        return fail(MI_LAYER_ERR_INVALID, "%s: row length %lld out of range", who, (long long)a.I);
    if (a.threshold < 0 || a.threshold > 65535)
        return fail(MI_LAYER_ERR_INVALID, "%s: threshold %d out of range 0..65535", who, a.threshold);
    if (a.x_stride < 0 || a.grad_stride < 0 || a.out_stride < (backward ? 2 : 1) * a.I)
        return fail(MI_LAYER_ERR_INVALID, "%s: bad stride", who);
    if (a.max_rows == 0) return MI_LAYER_OK;
    if (!a.x || !a.out || (backward && !a.grad)) return fail(MI_LAYER_ERR_INVALID, "%s: NULL pointer argument", who);
    const size_t size = size_of(a.dtype);
    if (!aligned(a.x, size) || !aligned(a.out, size) || (backward && !aligned(a.grad, size)) ||
        !aligned(a.num_rows, 4) || !aligned(a.seed_ptr, 8))
        return fail(MI_LAYER_ERR_INVALID, "%s: misaligned pointer", who);
    return MI_LAYER_OK;
}

// Sizes of 4-bit weights: N and K to 2^24, groups a power of two.
int check_int4(const char* who, int64_t E, int64_t N, int64_t K, int32_t group) {
    if (E < 0 || E > MI_LAYER_MAX_EXPERTS)
        return fail(MI_LAYER_ERR_INVALID, "%s: num_experts %lld out of range 0..%d", who, (long long)E,
                    MI_LAYER_MAX_EXPERTS);
    if (N < 0 || N > 1 << 24 || K < 1 || K > 1 << 24)
        return fail(MI_LAYER_ERR_INVALID, "%s: N %lld or K %lld out of range", who, (long long)N, (long long)K);
    if (group < MI_LAYER_INT4_MIN_GROUP || (group & (group - 1)) != 0)
        return fail(MI_LAYER_ERR_INVALID, "%s: group_size %d is no power of two from %d", who, group,
                    MI_LAYER_INT4_MIN_GROUP);
    return MI_LAYER_OK;
}

}  // namespace

extern "C" {

const char* mi_layer_last_error(void) { return g_last_error; }

size_t mi_layer_balance_workspace_size(int64_t num_tokens, int64_t num_seqs, int32_t num_experts) {
    return balance_sizes(num_tokens, num_seqs, num_experts) ? balance_workspace(num_tokens, num_seqs, num_experts) : 0;
}

int mi_layer_balance(const mi_layer_balance_args* args, void* stream) {
    const char* who = "mi_layer_balance";
    g_last_error[0] = 0;
    if (!args) return fail(MI_LAYER_ERR_INVALID, "%s: args is NULL", who);
    if (int rc = check_balance(who, *args, false)) return rc;
    if (args->num_tokens * args->top_k > INT32_MAX)  // counts have 32 bits
        return fail(MI_LAYER_ERR_INVALID, "%s: num_tokens %lld x top_k %d out of range", who,
                    (long long)args->num_tokens, args->top_k);
    if (!args->loss || !args->counts || (args->num_tokens > 0 && !args->topk_ids))
        return fail(MI_LAYER_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(args->loss, 4) || !aligned(args->counts, 4) || !aligned(args->topk_ids, 4))
        return fail(MI_LAYER_ERR_INVALID, "%s: misaligned pointer", who);
    if (int rc = check_workspace(who, args->workspace, args->workspace_bytes,
                                 balance_workspace(args->num_tokens, args->num_seqs, args->num_experts)))
        return rc;
    return hip_status(who, launch_balance(*args, (hipStream_t)stream));
}

int mi_layer_balance_backward(const mi_layer_balance_args* args, const float* grad_loss, void* grad_logits,
                              int64_t grad_stride, void* stream) {
    const char* who = "mi_layer_balance_backward";
    g_last_error[0] = 0;
    if (!args) return fail(MI_LAYER_ERR_INVALID, "%s: args is NULL", who);
    if (int rc = check_balance(who, *args, true)) return rc;
    if (grad_stride < args->num_experts) return fail(MI_LAYER_ERR_INVALID, "%s: bad stride", who);
    if (args->num_tokens == 0) return MI_LAYER_OK;
    if (!grad_loss || !grad_logits) return fail(MI_LAYER_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(grad_loss, 4) || !aligned(grad_logits, size_of(args->dtype)))
        return fail(MI_LAYER_ERR_INVALID, "%s: misaligned pointer", who);
    return hip_status(who, launch_balance_backward(*args, grad_loss, grad_logits, grad_stride, (hipStream_t)stream));
}

int mi_layer_swiglu(const mi_layer_swiglu_args* args, void* stream) {
    const char* who = "mi_layer_swiglu";
    g_last_error[0] = 0;
    if (!args) return fail(MI_LAYER_ERR_INVALID, "%s: args is NULL", who);
    if (int rc = check_swiglu(who, *args, false)) return rc;
    if (args->max_rows == 0) return MI_LAYER_OK;
    return hip_status(who, launch_swiglu(*args, false, (hipStream_t)stream));
}

int mi_layer_swiglu_backward(const mi_layer_swiglu_args* args, void* stream) {
    const char* who = "mi_layer_swiglu_backward";
    g_last_error[0] = 0;
    if (!args) return fail(MI_LAYER_ERR_INVALID, "%s: args is NULL", who);
    if (int rc = check_swiglu(who, *args, true)) return rc;
    if (args->max_rows == 0) return MI_LAYER_OK;
    return hip_status(who, launch_swiglu(*args, true, (hipStream_t)stream));
}

int mi_layer_pack_int4(const int8_t* q, int64_t q_expert_stride, int64_t q_stride, const void* scale,
                       int32_t scale_dtype, int64_t num_experts, int64_t N, int64_t K, int32_t group_size,
                       uint8_t* packed, void* scale_out, void* stream) {
    const char* who = "mi_layer_pack_int4";
    g_last_error[0] = 0;
    if (!float_type(scale_dtype)) return fail(MI_LAYER_ERR_INVALID, "%s: unknown dtype %d", who, scale_dtype);
    if (int rc = check_int4(who, num_experts, N, K, group_size)) return rc;
    if (q_expert_stride < 0 || q_stride < 0) return fail(MI_LAYER_ERR_INVALID, "%s: bad stride", who);
    if (N == 0) return MI_LAYER_OK;
    if (!q || !scale || !packed || !scale_out) return fail(MI_LAYER_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(scale, size_of(scale_dtype)) || !aligned(packed, 16) || !aligned(scale_out, 16))
        return fail(MI_LAYER_ERR_INVALID, "%s: misaligned pointer", who);
    return hip_status(who, launch_pack_int4(q, q_expert_stride, q_stride, scale, scale_dtype,
                                            num_experts ? num_experts : 1, N, K, group_size, packed, scale_out,
                                            (hipStream_t)stream));
}

int mi_layer_quantize_int4(int32_t dtype, const void* w, int64_t w_expert_stride, int64_t w_stride,
                           int64_t num_experts, int64_t N, int64_t K, int32_t group_size, uint8_t* packed,
                           float* scale_out, void* stream) {
    const char* who = "mi_layer_quantize_int4";
    g_last_error[0] = 0;
    if (!float_type(dtype)) return fail(MI_LAYER_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
    if (int rc = check_int4(who, num_experts, N, K, group_size)) return rc;
    if (w_expert_stride < 0 || w_stride < 0) return fail(MI_LAYER_ERR_INVALID, "%s: bad stride", who);
    if (N == 0) return MI_LAYER_OK;
    if (!w || !packed || !scale_out) return fail(MI_LAYER_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(w, size_of(dtype)) || !aligned(packed, 16) || !aligned(scale_out, 16))
        return fail(MI_LAYER_ERR_INVALID, "%s: misaligned pointer", who);
    return hip_status(who, launch_quantize_int4(dtype, w, w_expert_stride, w_stride, num_experts ? num_experts : 1, N,
                                                K, group_size, packed, scale_out, (hipStream_t)stream));
}

size_t mi_layer_int4_workspace_size(int64_t x_rows, int64_t K, int32_t is_aligned) {
    if (is_aligned || x_rows <= 0 || x_rows > INT32_MAX || K < 1 || K > 1 << 24) return 0;
    return (size_t)x_rows * (size_t)((K + 7) / 8 * 8) * 2;
}

int mi_layer_int4_matmul(const mi_layer_int4_args* args, void* stream) {
    const char* who = "mi_layer_int4_matmul";
    g_last_error[0] = 0;
    if (!args) return fail(MI_LAYER_ERR_INVALID, "%s: args is NULL", who);
    const mi_layer_int4_args& a = *args;
    if ((a.x_dtype != MI_LAYER_BF16 && a.x_dtype != MI_LAYER_F16) || !float_type(a.out_dtype) ||
        (a.bias && !float_type(a.bias_dtype)) || (a.scale_dtype != MI_LAYER_F32 && a.scale_dtype != a.x_dtype))
        return fail(MI_LAYER_ERR_INVALID, "%s: dtypes not supported (x of 16 bits, scales of fp32 or x's type)", who);
    if (int rc = check_int4(who, a.num_experts, a.N, a.K, a.group_size)) return rc;
    if (a.rows < 0 || a.rows > INT32_MAX || a.x_rows < 0 || a.x_rows > INT32_MAX)
        return fail(MI_LAYER_ERR_INVALID, "%s: size out of range", who);
    if (a.num_experts == 0 && (a.row_ids || a.expert_offsets))
        return fail(MI_LAYER_ERR_INVALID, "%s: row_ids and expert_offsets belong to grouped products", who);
    if (a.num_experts > 0 && a.bias) return fail(MI_LAYER_ERR_INVALID, "%s: grouped products take no bias", who);
    if (!a.row_ids && a.rows != a.x_rows)
        return fail(MI_LAYER_ERR_INVALID, "%s: rows (%lld) must equal x_rows (%lld) without row_ids", who,
                    (long long)a.rows, (long long)a.x_rows);
    if (a.x_stride < 0 || a.out_stride < a.N) return fail(MI_LAYER_ERR_INVALID, "%s: bad stride", who);
    // tiles are counted in 32 bits
    if (((a.rows + 15) / 16 + a.num_experts) * ((a.N + 15) / 16) > INT32_MAX)
        return fail(MI_LAYER_ERR_INVALID, "%s: %lld x %lld outputs are too many for one call", who, (long long)a.rows,
                    (long long)a.N);
    if (a.rows == 0 || a.N == 0) return MI_LAYER_OK;
    if (a.x_rows == 0) return fail(MI_LAYER_ERR_INVALID, "%s: x has no rows for row_ids", who);
    if (!a.x || !a.w || !a.scale || !a.out || (a.num_experts && !a.expert_offsets))
        return fail(MI_LAYER_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(a.x, 2) || !aligned(a.w, 16) || !aligned(a.scale, 16) || !aligned(a.out, size_of(a.out_dtype)) ||
        !aligned(a.bias, a.bias ? size_of(a.bias_dtype) : 1) || !aligned(a.expert_offsets, 4) ||
        !aligned(a.row_ids, 4))
        return fail(MI_LAYER_ERR_INVALID, "%s: misaligned pointer", who);
    if (int rc = check_workspace(who, a.workspace, a.workspace_bytes,
                                 mi_layer_int4_workspace_size(a.x_rows, a.K, int4_aligned(a))))
        return rc;
    return hip_status(who, launch_int4_matmul(a, (hipStream_t)stream));
}

}  // extern "C"
