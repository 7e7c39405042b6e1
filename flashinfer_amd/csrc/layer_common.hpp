// Shared by the operators of libmi_layer.so (include/mi_layer.h): launchers.
// Element types, vector loads and stores are those of the expert operators.
#pragma once

#include "../../include/mi_layer.h"
#include "experts_common.hpp"

namespace miexp {

static_assert(MI_LAYER_BF16 == MI_EXPERTS_BF16 && MI_LAYER_F32 == MI_EXPERTS_F32 && MI_LAYER_F16 == MI_EXPERTS_F16,
              "one set of element types");

size_t balance_workspace(int64_t T, int64_t S, int E);
hipError_t launch_balance(const mi_layer_balance_args& a, hipStream_t s);
hipError_t launch_balance_backward(const mi_layer_balance_args& a, const float* grad_loss, void* grad,
                                   int64_t grad_stride, hipStream_t s);
hipError_t launch_swiglu(const mi_layer_swiglu_args& a, bool backward, hipStream_t s);
hipError_t launch_pack_int4(const int8_t* q, int64_t q_expert_stride, int64_t q_stride, const void* scale,
                            int scale_dtype, int64_t E, int64_t N, int64_t K, int group, uint8_t* packed,
                            void* scale_out, hipStream_t s);
hipError_t launch_quantize_int4(int dtype, const void* w, int64_t w_expert_stride, int64_t w_stride, int64_t E,
                                int64_t N, int64_t K, int group, uint8_t* packed, float* scale_out, hipStream_t s);
bool int4_aligned(const mi_layer_int4_args& a);
hipError_t launch_int4_matmul(const mi_layer_int4_args& a, hipStream_t s);

}  // namespace miexp
