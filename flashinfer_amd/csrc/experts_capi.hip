// extern "C" boundary of the expert operators (include/mi_experts.h): every
// argument is checked before the first launch.
#include <stdarg.h>
#include <stdio.h>

#include "experts_common.hpp"

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
bool float_type(int32_t d) { return d == MI_EXPERTS_BF16 || d == MI_EXPERTS_F32 || d == MI_EXPERTS_F16; }
size_t size_of(int32_t d) { return d == MI_EXPERTS_F32 ? 4 : 2; }

// Rows of the row-moving kernels: at most 2^15 chunks of 256 units.
constexpr int64_t MAX_ROW_BYTES = 1 << 23;

int hip_status(const char* who, hipError_t e) {
    if (e == hipSuccess) return MI_EXPERTS_OK;
    return fail(MI_EXPERTS_ERR_HIP, "%s: launch failed: %s", who, hipGetErrorString(e));
}

// Sizes shared by the operators that go by token and slot.
int check_slots(const char* who, int64_t T, int32_t k) {
    if (k < 1 || k > MI_EXPERTS_MAX_TOP_K)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: top_k %d out of range 1..%d", who, k, MI_EXPERTS_MAX_TOP_K);
    if (T < 0 || T > MI_EXPERTS_MAX_SLOTS / k)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: num_tokens %lld out of range (at most %d slots)", who,
                    (long long)T, MI_EXPERTS_MAX_SLOTS);
    return MI_EXPERTS_OK;
}

int check_row(const char* who, int64_t row_len, int64_t size) {
    if (row_len < 1 || row_len > MAX_ROW_BYTES / size)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: row length %lld out of range (rows of 1 to %lld bytes)", who,
                    (long long)row_len, (long long)MAX_ROW_BYTES);
    return MI_EXPERTS_OK;
}

}  // namespace

extern "C" {

const char* mi_experts_last_error(void) { return g_last_error; }

size_t mi_experts_sort_workspace_size(int64_t num_slots, int32_t num_experts) {
    if (num_slots <= 0 || num_slots > MI_EXPERTS_MAX_SLOTS || num_experts < 1) return 0;
    return (size_t)sort_chunks(num_slots) * ((size_t)num_experts + 1) * sizeof(int32_t);
}

int mi_experts_sort(const int32_t* topk_ids, int64_t num_tokens, int32_t top_k, int32_t num_experts,
                    int64_t expert_offset, int32_t* expert_offsets, int32_t* token_of_row,
                    int32_t* row_of_slot, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "mi_experts_sort";
    g_last_error[0] = 0;
    if (int rc = check_slots(who, num_tokens, top_k)) return rc;
    if (num_experts < 1 || num_experts > MI_EXPERTS_MAX_EXPERTS)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: num_experts %d out of range 1..%d", who, num_experts,
                    MI_EXPERTS_MAX_EXPERTS);
    if (!expert_offsets || (num_tokens > 0 && (!topk_ids || !token_of_row || !row_of_slot)))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(topk_ids, 4) || !aligned(expert_offsets, 4) || !aligned(token_of_row, 4) ||
        !aligned(row_of_slot, 4))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: misaligned pointer", who);
    const size_t need = mi_experts_sort_workspace_size(num_tokens * top_k, num_experts);
    if (need && (!workspace || workspace_bytes < need))
        return fail(MI_EXPERTS_ERR_WORKSPACE, "%s: workspace has %zu bytes, needs %zu", who,
                    workspace ? workspace_bytes : (size_t)0, need);
    if (need && !aligned(workspace, 4))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: misaligned workspace", who);
    // beyond int32 ids and expert counts an offset selects no expert
    const int64_t most = (int64_t)1 << 40;
    const int64_t off = expert_offset > most ? most : expert_offset < -most ? -most : expert_offset;
    return hip_status(who, launch_sort(topk_ids, num_tokens, top_k, num_experts, off, expert_offsets,
                                       token_of_row, row_of_slot, (int32_t*)workspace, (hipStream_t)stream));
}

int mi_experts_permute(const void* x, int64_t x_stride, int64_t num_tokens, int32_t top_k,
                       int64_t row_bytes, const int32_t* row_of_slot, const int32_t* num_rows,
                       void* rows, int64_t rows_stride, int32_t zero_rest, void* stream) {
    const char* who = "mi_experts_permute";
    g_last_error[0] = 0;
    if (int rc = check_slots(who, num_tokens, top_k)) return rc;
    if (int rc = check_row(who, row_bytes, 1)) return rc;
    if (x_stride < 0 || rows_stride < row_bytes)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: bad stride", who);
    if (num_tokens == 0) return MI_EXPERTS_OK;
    if (!x || !row_of_slot || !num_rows || !rows)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(row_of_slot, 4) || !aligned(num_rows, 4))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: misaligned pointer", who);
    return hip_status(who, launch_permute(x, x_stride, num_tokens, top_k, row_bytes, row_of_slot, num_rows,
                                          rows, rows_stride, zero_rest != 0, (hipStream_t)stream));
}

int mi_experts_unpermute(int32_t dtype, const void* rows, int64_t rows_stride, int64_t num_tokens,
                         int32_t top_k, int64_t row_len, const int32_t* row_of_slot,
                         const int32_t* num_rows, const float* weights, void* out,
                         int64_t out_stride, void* stream) {
    const char* who = "mi_experts_unpermute";
    g_last_error[0] = 0;
    if (!float_type(dtype)) return fail(MI_EXPERTS_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
    if (int rc = check_slots(who, num_tokens, top_k)) return rc;
    if (int rc = check_row(who, row_len, (int64_t)size_of(dtype))) return rc;
    if (rows_stride < 0 || out_stride < row_len) return fail(MI_EXPERTS_ERR_INVALID, "%s: bad stride", who);
    if (num_tokens == 0) return MI_EXPERTS_OK;
    if (!rows || !row_of_slot || !num_rows || !out)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(rows, size_of(dtype)) || !aligned(out, size_of(dtype)) || !aligned(row_of_slot, 4) ||
        !aligned(num_rows, 4) || !aligned(weights, 4))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: misaligned pointer", who);
    return hip_status(who, launch_unpermute(dtype, rows, rows_stride, num_tokens, top_k, row_len,
                                            row_of_slot, num_rows, weights, out, out_stride,
                                            (hipStream_t)stream));
}

int mi_experts_unpermute_backward(int32_t dtype, const void* grad, int64_t grad_stride,
                                  const void* rows, int64_t rows_stride, int64_t num_tokens,
                                  int32_t top_k, int64_t row_len, const int32_t* row_of_slot,
                                  const int32_t* num_rows, const float* weights, void* grad_rows,
                                  int64_t grad_rows_stride, int32_t zero_rest, float* grad_weights,
                                  void* stream) {
    const char* who = "mi_experts_unpermute_backward";
    g_last_error[0] = 0;
    if (!float_type(dtype)) return fail(MI_EXPERTS_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
    if (int rc = check_slots(who, num_tokens, top_k)) return rc;
    if (int rc = check_row(who, row_len, (int64_t)size_of(dtype))) return rc;
    if (grad_stride < 0 || (grad_weights && rows_stride < 0) || (grad_rows && grad_rows_stride < row_len))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: bad stride", who);
    if (num_tokens == 0 || (!grad_rows && !grad_weights)) return MI_EXPERTS_OK;
    if (!grad || !row_of_slot || !num_rows || (grad_weights && !rows))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(grad, size_of(dtype)) || !aligned(rows, size_of(dtype)) || !aligned(grad_rows, size_of(dtype)) ||
        !aligned(row_of_slot, 4) || !aligned(num_rows, 4) || !aligned(weights, 4) || !aligned(grad_weights, 4))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: misaligned pointer", who);
    return hip_status(who, launch_unpermute_backward(dtype, grad, grad_stride, rows, rows_stride, num_tokens,
                                                     top_k, row_len, row_of_slot, num_rows, weights,
                                                     grad_rows, grad_rows_stride, zero_rest != 0,
                                                     grad_weights, (hipStream_t)stream));
}

int mi_experts_quantize_int8(int32_t dtype, const void* x, int64_t x_stride, int64_t num_rows_max,
                             int64_t row_len, int32_t swiglu, const int32_t* num_rows,
                             int32_t zero_rest, int8_t* q, int64_t q_stride, float* scale,
                             void* stream) {
    const char* who = "mi_experts_quantize_int8";
    g_last_error[0] = 0;
    if (!float_type(dtype)) return fail(MI_EXPERTS_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
    if (num_rows_max < 0 || num_rows_max > INT32_MAX)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: %lld rows out of range", who, (long long)num_rows_max);
    if (row_len < 1 || row_len > INT32_MAX / 8)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: row length %lld out of range", who, (long long)row_len);
    if (x_stride < 0 || q_stride < row_len) return fail(MI_EXPERTS_ERR_INVALID, "%s: bad stride", who);
    if (num_rows_max == 0) return MI_EXPERTS_OK;
    if (!x || !q || !scale) return fail(MI_EXPERTS_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(x, size_of(dtype)) || !aligned(scale, 4) || !aligned(num_rows, 4))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: misaligned pointer", who);
    return hip_status(who, launch_quantize(dtype, x, x_stride, num_rows_max, row_len, swiglu != 0, num_rows,
                                           zero_rest != 0, q, q_stride, scale, (hipStream_t)stream));
}

size_t mi_experts_int8_workspace_size(int64_t rows, int64_t N, int64_t K, int32_t num_experts) {
    if (rows <= 0 || N <= 0 || K <= 0 || num_experts < 0) return 0;
    return int8_workspace(rows, N, K, num_experts);
}

int mi_experts_int8_matmul(const mi_experts_int8_args* args, void* stream) {
    const char* who = "mi_experts_int8_matmul";
    g_last_error[0] = 0;
    if (!args) return fail(MI_EXPERTS_ERR_INVALID, "%s: args is NULL", who);
    const mi_experts_int8_args& a = *args;
    if (!float_type(a.out_dtype) || (a.bias && !float_type(a.bias_dtype)))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: unknown dtype", who);
    if (a.num_experts < 0 || a.num_experts > MI_EXPERTS_MAX_EXPERTS)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: num_experts %d out of range 0..%d", who, a.num_experts,
                    MI_EXPERTS_MAX_EXPERTS);
    if (a.K < 1 || a.K > MI_EXPERTS_MAX_K)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: K %lld out of range 1..%d", who, (long long)a.K,
                    MI_EXPERTS_MAX_K);
    if (a.rows < 0 || a.rows > INT32_MAX || a.a_rows < 0 || a.a_rows > INT32_MAX || a.N < 0 ||
        a.N > INT32_MAX / 2)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: size out of range", who);
    if (a.num_experts == 0 && (a.row_ids || a.expert_offsets))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: row_ids and expert_offsets belong to grouped products", who);
    if (a.num_experts > 0 && a.bias)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: grouped products take no bias", who);
    if (!a.row_ids && a.rows != a.a_rows)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: rows (%lld) must equal a_rows (%lld) without row_ids", who,
                    (long long)a.rows, (long long)a.a_rows);
    if (a.a_stride < 0 || a.b_stride < 0 || a.b_expert_stride < 0 || a.out_stride < a.N)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: bad stride", who);
    // a launch holds fewer than 2^32 threads
    if (((a.rows + 63) / 64 + a.num_experts) * ((a.N + 63) / 64) >= (int64_t)1 << 24)
        return fail(MI_EXPERTS_ERR_INVALID, "%s: %lld x %lld outputs are too many for one call", who,
                    (long long)a.rows, (long long)a.N);
    if (a.rows == 0 || a.N == 0) return MI_EXPERTS_OK;
    if (a.a_rows == 0) return fail(MI_EXPERTS_ERR_INVALID, "%s: a has no rows for row_ids", who);
    if (!a.a || !a.a_scale || !a.b || !a.b_scale || !a.out || (a.num_experts && !a.expert_offsets))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: NULL pointer argument", who);
    if (!aligned(a.a_scale, 4) || !aligned(a.b_scale, 4) || !aligned(a.out, size_of(a.out_dtype)) ||
        !aligned(a.bias, a.bias ? size_of(a.bias_dtype) : 1) || !aligned(a.expert_offsets, 4) ||
        !aligned(a.row_ids, 4))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: misaligned pointer", who);
    const size_t need = int8_workspace(a.rows, a.N, a.K, a.num_experts);
    if (need && (!a.workspace || a.workspace_bytes < need))
        return fail(MI_EXPERTS_ERR_WORKSPACE, "%s: workspace has %zu bytes, needs %zu", who,
                    a.workspace ? a.workspace_bytes : (size_t)0, need);
    if (need && !aligned(a.workspace, 256))
        return fail(MI_EXPERTS_ERR_INVALID, "%s: misaligned workspace", who);
    return hip_status(who, launch_int8_matmul(a, (hipStream_t)stream));
}

}  // extern "C"
