// Shared by the torch sides of the operators (_mi_experts, _mi_layer): checks of
// tensors, destinations, streams.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/grad_mode.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/mi_experts.h"

namespace mitorch {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// The current stream of a device, which is made current while this lives.
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t)
        : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

inline void expect_type(const Tensor& t, const char* name, at::ScalarType want) {
    TORCH_CHECK_TYPE(t.scalar_type() == want, name, " must have dtype ", want, ", got ", t.scalar_type());
}

inline int float_dtype(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return MI_EXPERTS_BF16;
        case at::kHalf: return MI_EXPERTS_F16;
        case at::kFloat: return MI_EXPERTS_F32;
        default:
            TORCH_CHECK_TYPE(false, name, " must have dtype bfloat16, float16 or float32, got ", t.scalar_type());
    }
}

inline int out_dtype_of(at::ScalarType t) {
    TORCH_CHECK_TYPE(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat,
                     "out_dtype must be bfloat16, float16 or float32, got ", t);
    return t == at::kBFloat16 ? MI_EXPERTS_BF16 : t == at::kHalf ? MI_EXPERTS_F16 : MI_EXPERTS_F32;
}

inline void expect_shape(const Tensor& t, const char* name, at::IntArrayRef want) {
    TORCH_CHECK_VALUE(t.sizes() == want, name, " must have shape ", want, ", got ", t.sizes());
}

inline void expect_dim(const Tensor& t, const char* name, int64_t dim) {
    TORCH_CHECK_VALUE(t.dim() == dim, name, " must have ", dim, " dimensions, got shape ", t.sizes());
}

inline void expect_gpu(const Tensor& t, const char* name) {
    TORCH_CHECK_VALUE(t.is_cuda(), name, " must be on a ROCm GPU (device type 'cuda'), got ", t.device(),
                      "; there is no CPU path");
}

inline void expect_device(const Tensor& t, const char* name, const Tensor& like) {
    TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", expected ", like.device());
}

// Kernels read memory as it is: a view whose sign torch changes only when it is
// read (the imaginary part of a conjugate) is copied.
inline Tensor dense(const Tensor& t) { return t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous(); }

// Rows of consecutive elements at any distance: as it is, or copied.
inline Tensor rows_of(const Tensor& t) {
    if (t.is_neg()) return t.resolve_neg().contiguous();
    const bool ok = t.stride(-1) == 1 || t.size(-1) <= 1;
    return ok && (t.dim() < 2 || t.stride(-2) >= 0) ? t : t.contiguous();
}
// Distance of rows; that of a tensor with one row is of no account (torch may report any).
inline int64_t row_stride(const Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// A destination: right type, shape and device, rows of consecutive elements
// that do not overlap, and no part of an autograd graph.
inline void expect_out(const Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape, const Tensor& like) {
    expect_type(t, name, type);
    expect_shape(t, name, shape);
    expect_device(t, name, like);
    TORCH_CHECK_VALUE(!t.is_neg(), name, " must not be a negated view");
    TORCH_CHECK_VALUE(t.numel() == 0 || t.dim() != 2 ||
                          ((t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1))),
                      name, " must have rows of consecutive elements that do not overlap, got strides ", t.strides());
    TORCH_CHECK_VALUE(t.dim() != 1 || t.is_contiguous(), name, " must be contiguous");
}

// Bytes a tensor's elements lie in.
inline std::pair<const char*, const char*> extent(const Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    const char* p = static_cast<const char*>(t.const_data_ptr());
    return {p, p + (last + 1) * (int64_t)t.element_size()};
}

// Rows of `width` bytes, `pitch` apart; a vector at a distance is a column.
struct Rows {
    const char* first;
    int64_t width, pitch, rows;
};
inline std::optional<Rows> as_rows(const Tensor& t) {
    if (t.dim() < 1 || t.dim() > 2) return std::nullopt;
    const bool column = t.dim() == 1 && t.stride(0) != 1;
    if (t.dim() == 2 && t.size(1) > 1 && t.stride(1) != 1) return std::nullopt;
    const int64_t size = (int64_t)t.element_size();
    return Rows{static_cast<const char*>(t.const_data_ptr()), (column ? 1 : t.size(-1)) * size, t.stride(0) * size,
                t.dim() == 2 || column ? t.size(0) : 1};
}

// Whether two tensors whose extents overlap are columns of one buffer that lie
// side by side.
inline bool side_by_side(const Tensor& x, const Tensor& y) {
    auto a = as_rows(x), b = as_rows(y);
    if (!a || !b) return false;
    if (a->rows == 1) std::swap(a, b);  // one row lies beside rows of any pitch
    if (a->pitch <= 0 || (b->rows > 1 && b->pitch != a->pitch)) return false;
    const int64_t at = ((b->first - a->first) % a->pitch + a->pitch) % a->pitch;
    return at >= a->width && at + b->width <= a->pitch;
}

// A destination shares no memory with what is read: rows are written while
// others are read. Columns of one buffer may be both.
inline void expect_apart(const Tensor& out, const char* name, std::initializer_list<const Tensor*> inputs) {
    if (out.numel() == 0) return;
    const auto o = extent(out);
    for (const Tensor* t : inputs) {
        if (!t->defined() || t->numel() == 0) continue;
        const auto i = extent(*t);
        if (i.second <= o.first || o.second <= i.first) continue;
        TORCH_CHECK_VALUE(side_by_side(out, *t), name, " shares memory with a tensor that the call reads");
    }
}

// Writes through a pointer are in-place changes to autograd, too.
inline void written(const Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }

inline void no_grad_out(const char* what, bool needs, const OptTensor& out) {
    TORCH_CHECK_VALUE(!(out && out->defined() && (needs || (at::GradMode::is_enabled() && out->requires_grad()))),
                      what, "(): out= takes no part in autograd; call it without out, or under torch.no_grad()");
}

// A tangent of forward-mode differentiation. It comes without requires_grad
// and is there under torch.no_grad(), too.
inline bool has_tangent(const Tensor& t) {
    return t.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined();
}

// The results carry no tangents: inputs whose tangent would be lost, and
// destinations that would keep a wrong one, are refused.
inline void expect_no_tangent(const char* what, std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        TORCH_CHECK_VALUE(!has_tangent(*t), what,
                          "() has no forward-mode derivative and got a tensor with a tangent: detach it");
}

// An optional tensor, undefined if there is none.
inline const Tensor& or_none(const OptTensor& t) {
    static const Tensor none;
    return t ? *t : none;
}

// Some operators have no gradient: one that would be lost is refused.
inline void expect_no_grad(const char* what, std::initializer_list<const Tensor*> inputs) {
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor* t : inputs)
        TORCH_CHECK_VALUE(!t->defined() || !t->requires_grad(), what,
                          "() has no gradient and got a tensor that requires one: detach it, or call it under "
                          "torch.no_grad()");
}

}  // namespace mitorch
