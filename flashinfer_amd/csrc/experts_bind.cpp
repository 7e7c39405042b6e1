// Torch side of the expert operators (_mi_experts): the checks of tensors,
// allocation of results, streams and autograd of sort_experts, permute,
// unpermute, quantize_int8 and the int8 products, in front of
// libmi_experts.so. Done in C++ because a decode call's kernels take a few
// microseconds, less than the same checks take from Python.
//
// Errors are Python's: TypeError for a wrong type of tensor, ValueError for a
// wrong shape, device or value, RuntimeError with the library's message for
// what the library refuses.
//
// Built with g++ against torch's headers (no device code here).
#include "torch_common.hpp"

namespace py = pybind11;

namespace {

using namespace mitorch;

void check(int rc) {
    TORCH_CHECK(rc == MI_EXPERTS_OK, "mi_experts error ", rc, ": ", mi_experts_last_error());
}

// ---------------------------------------------------------------- sorting

py::tuple sort_experts(const Tensor& topk_ids, int64_t num_experts, int64_t expert_offset) {
    expect_dim(topk_ids, "topk_ids", 2);
    expect_type(topk_ids, "topk_ids", at::kInt);
    expect_gpu(topk_ids, "topk_ids");
    const int64_t T = topk_ids.size(0), k = topk_ids.size(1);
    TORCH_CHECK_VALUE(k >= 1 && k <= MI_EXPERTS_MAX_TOP_K, "topk_ids must have 1 to ", MI_EXPERTS_MAX_TOP_K,
                      " experts per token, got ", k);
    TORCH_CHECK_VALUE(num_experts >= 1 && num_experts <= MI_EXPERTS_MAX_EXPERTS, "num_experts must be 1 to ",
                      MI_EXPERTS_MAX_EXPERTS, ", got ", num_experts);
    TORCH_CHECK_VALUE(T <= MI_EXPERTS_MAX_SLOTS / k, "topk_ids: ", T, " x ", k, " slots, at most ",
                      MI_EXPERTS_MAX_SLOTS, " in one call");
    On on(topk_ids);
    const Tensor ids = topk_ids.contiguous();
    const auto opt = topk_ids.options().requires_grad(false);
    Tensor offsets = at::empty({num_experts + 1}, opt), token = at::empty({T * k}, opt), row = at::empty({T, k}, opt);
    const size_t need = mi_experts_sort_workspace_size(T * k, (int32_t)num_experts);
    Tensor ws;
    if (need) ws = at::empty({(int64_t)need}, opt.dtype(at::kByte));
    check(mi_experts_sort(ids.const_data_ptr<int32_t>(), T, (int32_t)k, (int32_t)num_experts, expert_offset,
                          offsets.mutable_data_ptr<int32_t>(), token.mutable_data_ptr<int32_t>(),
                          row.mutable_data_ptr<int32_t>(), need ? ws.data_ptr() : nullptr, need, on.stream));
    return py::make_tuple(offsets, token, row);
}

// The tables of a plan, as permute and unpermute read them.
struct Plan {
    Tensor row_of_slot;  // [T, k] contiguous
    Tensor offsets;      // [E+1] contiguous
    int64_t T, k;
    const int32_t* rows() const { return row_of_slot.const_data_ptr<int32_t>(); }
    const int32_t* count() const { return offsets.const_data_ptr<int32_t>() + offsets.size(0) - 1; }
};

Plan plan_of(const Tensor& offsets, const Tensor& row_of_slot, const Tensor& like) {
    expect_dim(offsets, "plan.expert_offsets", 1);
    expect_dim(row_of_slot, "plan.row_of_slot", 2);
    expect_type(offsets, "plan.expert_offsets", at::kInt);
    expect_type(row_of_slot, "plan.row_of_slot", at::kInt);
    TORCH_CHECK_VALUE(offsets.size(0) >= 2, "plan.expert_offsets must have an entry for each expert and the end");
    expect_device(offsets, "plan.expert_offsets", like);
    expect_device(row_of_slot, "plan.row_of_slot", like);
    return Plan{row_of_slot.contiguous(), offsets.contiguous(), row_of_slot.size(0), row_of_slot.size(1)};
}

// --------------------------------------------------------------- permute

void permute_into(const Tensor& x, const Plan& p, const Tensor& rows, bool zero_rest) {
    if (rows.numel() == 0) return;
    On on(x);
    const Tensor in = rows_of(x);
    const int64_t size = (int64_t)in.element_size();
    check(mi_experts_permute(in.const_data_ptr(), row_stride(in) * size, p.T, (int32_t)p.k, in.size(1) * size,
                             p.rows(), p.count(), rows.mutable_data_ptr(), row_stride(rows) * size, zero_rest,
                             on.stream));
}

Tensor unpermute_new(const Tensor& rows, const Plan& p, const Tensor& weights) {
    On on(rows);
    Tensor out = at::empty({p.T, rows.size(1)}, rows.options().requires_grad(false));
    if (out.numel() == 0) return out;
    const Tensor in = rows_of(rows);
    check(mi_experts_unpermute(float_dtype(in, "rows"), in.const_data_ptr(), row_stride(in), p.T, (int32_t)p.k,
                               in.size(1), p.rows(), p.count(),
                               weights.defined() ? weights.const_data_ptr<float>() : nullptr,
                               out.mutable_data_ptr(), row_stride(out), on.stream));
    return out;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct PermuteFn : torch::autograd::Function<PermuteFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& offsets, const Tensor& row_of_slot) {
        const Plan p = plan_of(offsets, row_of_slot, x);
        ctx->save_for_backward({p.offsets, p.row_of_slot});
        c10::DeviceGuard guard(x.device());
        Tensor rows = at::empty({p.T * p.k, x.size(1)}, x.options().requires_grad(false));
        permute_into(x, p, rows, true);
        return rows;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "permute() has no second derivative (create_graph=True)");
        TORCH_CHECK(!has_tangent(grads[0]), "permute() has no second derivative (a gradient with a tangent)");
        const auto saved = ctx->get_saved_variables();
        const Plan p = plan_of(saved[0], saved[1], grads[0]);
        return {unpermute_new(grads[0], p, Tensor()), Tensor(), Tensor()};
    }
};

Tensor permute(const Tensor& hidden, const Tensor& offsets, const Tensor& row_of_slot, const OptTensor& out) {
    expect_dim(hidden, "hidden", 2);
    expect_no_tangent("permute", {&hidden, &or_none(out)});
    expect_gpu(hidden, "hidden");
    const Plan p = plan_of(offsets, row_of_slot, hidden);
    TORCH_CHECK_VALUE(hidden.size(0) == p.T, "hidden has ", hidden.size(0), " tokens, the plan ", p.T);
    TORCH_CHECK_VALUE(hidden.size(1) >= 1, "hidden must have at least one column");
    TORCH_CHECK_TYPE(!hidden.is_complex() && !hidden.is_quantized(), "hidden has an unsupported dtype ", hidden.scalar_type());
    const bool needs = at::GradMode::is_enabled() && hidden.requires_grad();
    no_grad_out("permute", needs, out);
    if (out && out->defined()) {
        expect_out(*out, "out", hidden.scalar_type(), {p.T * p.k, hidden.size(1)}, hidden);
        expect_apart(*out, "out", {&hidden, &p.row_of_slot, &p.offsets});
        written(*out);
        permute_into(hidden, p, *out, false);
        return *out;
    }
    if (needs) {
        float_dtype(hidden, "hidden that requires a gradient");
        return PermuteFn::apply(hidden, p.offsets, p.row_of_slot);
    }
    c10::DeviceGuard guard(hidden.device());
    Tensor rows = at::empty({p.T * p.k, hidden.size(1)}, hidden.options().requires_grad(false));
    permute_into(hidden, p, rows, true);
    return rows;
}

// -------------------------------------------------------------- unpermute

struct UnpermuteFn : torch::autograd::Function<UnpermuteFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& offsets, const Tensor& row_of_slot,
                          const OptTensor& weights) {
        const Plan p = plan_of(offsets, row_of_slot, rows);
        const Tensor w = weights ? dense(*weights) : Tensor();
        // rows are read again for the gradient of the weights alone
        const bool keep = weights && weights->requires_grad();
        ctx->save_for_backward({p.offsets, p.row_of_slot, w, keep ? rows : Tensor()});
        return unpermute_new(rows, p, w);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "unpermute() has no second derivative (create_graph=True)");
        TORCH_CHECK(!has_tangent(grads[0]), "unpermute() has no second derivative (a gradient with a tangent)");
        const auto saved = ctx->get_saved_variables();
        On on(grads[0]);
        const Tensor g = rows_of(grads[0]);
        const Plan p = plan_of(saved[0], saved[1], g);
        const Tensor w = saved[2], rows = saved[3].defined() ? rows_of(saved[3]) : saved[3];
        const bool need_rows = ctx->needs_input_grad(0), need_w = w.defined() && ctx->needs_input_grad(3);
        Tensor dr, dw;
        if (need_rows) dr = at::empty({p.T * p.k, g.size(1)}, g.options());
        if (need_w) dw = at::empty(w.sizes(), w.options().requires_grad(false));
        if (p.T > 0)
            check(mi_experts_unpermute_backward(
                float_dtype(g, "grad"), g.const_data_ptr(), row_stride(g), need_w ? rows.const_data_ptr() : nullptr,
                need_w ? row_stride(rows) : 0, p.T, (int32_t)p.k, g.size(1), p.rows(), p.count(),
                w.defined() ? w.const_data_ptr<float>() : nullptr, need_rows ? dr.mutable_data_ptr() : nullptr,
                need_rows ? row_stride(dr) : 0, 1, need_w ? dw.mutable_data_ptr<float>() : nullptr, on.stream));
        return {dr, Tensor(), Tensor(), dw};
    }
};

Tensor unpermute(const Tensor& rows, const Tensor& offsets, const Tensor& row_of_slot, const OptTensor& weights,
                 const OptTensor& out) {
    expect_dim(rows, "rows", 2);
    expect_no_tangent("unpermute", {&rows, &or_none(weights), &or_none(out)});
    expect_gpu(rows, "rows");
    const int dtype = float_dtype(rows, "rows");
    const Plan p = plan_of(offsets, row_of_slot, rows);
    TORCH_CHECK_VALUE(rows.size(0) == p.T * p.k, "rows must have a row for each of the plan's ", p.T * p.k,
                      " slots, got ", rows.size(0));
    TORCH_CHECK_VALUE(rows.size(1) >= 1, "rows must have at least one column");
    Tensor w;
    if (weights && weights->defined()) {
        w = *weights;
        expect_type(w, "weights", at::kFloat);
        expect_shape(w, "weights", {p.T, p.k});
        expect_device(w, "weights", rows);
    }
    const bool needs = at::GradMode::is_enabled() && (rows.requires_grad() || (w.defined() && w.requires_grad()));
    no_grad_out("unpermute", needs, out);
    if (out && out->defined()) {
        expect_out(*out, "out", rows.scalar_type(), {p.T, rows.size(1)}, rows);
        expect_apart(*out, "out", {&rows, &w, &p.row_of_slot, &p.offsets});
        written(*out);
        if (out->numel() == 0) return *out;
        On on(rows);
        const Tensor in = rows_of(rows), wc = w.defined() ? dense(w) : w;
        check(mi_experts_unpermute(dtype, in.const_data_ptr(), row_stride(in), p.T, (int32_t)p.k, in.size(1), p.rows(),
                                   p.count(), wc.defined() ? wc.const_data_ptr<float>() : nullptr,
                                   out->mutable_data_ptr(), row_stride(*out), on.stream));
        return *out;
    }
    if (needs) return UnpermuteFn::apply(rows, p.offsets, p.row_of_slot, w.defined() ? OptTensor(w) : std::nullopt);
    return unpermute_new(rows, p, w.defined() ? dense(w) : w);
}

// ------------------------------------------------------------- int8 rows

py::tuple quantize(const Tensor& x, bool swiglu, const OptTensor& num_rows, const OptTensor& q_out,
                   const OptTensor& scale_out) {
    expect_dim(x, "x", 2);
    const int dtype = float_dtype(x, "x");
    expect_no_tangent(swiglu ? "swiglu_quantize_int8" : "quantize_int8", {&x, &or_none(scale_out)});
    expect_gpu(x, "x");
    const int64_t M = x.size(0), C = x.size(1);
    TORCH_CHECK_VALUE(!swiglu || C % 2 == 0, "x must have 2 I columns, got ", C);
    const int64_t K = swiglu ? C / 2 : C;
    TORCH_CHECK_VALUE(K >= 1, "x must have at least one column");
    if (num_rows && num_rows->defined()) {
        expect_type(*num_rows, "num_rows", at::kInt);
        TORCH_CHECK_VALUE(num_rows->numel() == 1, "num_rows must hold one number, got shape ", num_rows->sizes());
        expect_device(*num_rows, "num_rows", x);
    }
    expect_no_grad(swiglu ? "swiglu_quantize_int8" : "quantize_int8", {&x});
    if (scale_out) expect_no_grad(swiglu ? "swiglu_quantize_int8" : "quantize_int8", {&*scale_out});
    On on(x);
    const bool given_q = q_out && q_out->defined(), given_s = scale_out && scale_out->defined();
    const Tensor none, &count = num_rows ? *num_rows : none;
    if (given_q) {
        expect_out(*q_out, "q", at::kChar, {M, K}, x);
        expect_apart(*q_out, "q", {&x, &count});
        written(*q_out);
    }
    if (given_s) {
        expect_out(*scale_out, "scale", at::kFloat, {M}, x);
        expect_apart(*scale_out, "scale", {&x, &count, given_q ? &*q_out : &none});
        written(*scale_out);
    }
    const auto opt = x.options().requires_grad(false);
    const bool cut = num_rows && num_rows->defined();
    // rows past num_rows: the kernel's to clear if both buffers are new
    const bool zero_rest = cut && !given_q && !given_s;
    auto fresh = [&](at::IntArrayRef shape, at::ScalarType t) {
        return cut && !zero_rest ? at::zeros(shape, opt.dtype(t)) : at::empty(shape, opt.dtype(t));
    };
    Tensor q = given_q ? *q_out : fresh({M, K}, at::kChar);
    Tensor scale = given_s ? *scale_out : fresh({M}, at::kFloat);
    if (M > 0) {
        const Tensor in = rows_of(x);
        check(mi_experts_quantize_int8(dtype, in.const_data_ptr(), row_stride(in), M, K, swiglu,
                                       cut ? num_rows->const_data_ptr<int32_t>() : nullptr, zero_rest,
                                       q.mutable_data_ptr<int8_t>(), row_stride(q), scale.mutable_data_ptr<float>(),
                                       on.stream));
    }
    return py::make_tuple(q, scale);
}

// ---------------------------------------------------------- int8 products

Tensor int8_call(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, const OptTensor& bias,
                 const Tensor* offsets, const OptTensor& row_ids, at::ScalarType out_type, const OptTensor& out_opt) {
    const bool grouped = offsets != nullptr;
    expect_dim(a, "a", 2);
    expect_dim(b, "b", grouped ? 3 : 2);
    expect_type(a, "a", at::kChar);
    expect_type(b, "b", at::kChar);
    expect_type(a_scale, "a_scale", at::kFloat);
    expect_type(b_scale, "b_scale", at::kFloat);
    expect_no_tangent(grouped ? "int8_grouped_matmul" : "int8_matmul",
                      {&a_scale, &b_scale, &or_none(bias), &or_none(out_opt)});
    expect_gpu(a, "a");
    const int64_t M = a.size(0), K = a.size(1), E = grouped ? b.size(0) : 0, N = b.size(-2);
    TORCH_CHECK_VALUE(b.size(-1) == K, "b must have ", K, " columns as a has, got shape ", b.sizes());
    TORCH_CHECK_VALUE(K >= 1 && K <= MI_EXPERTS_MAX_K, "a and b must have 1 to ", MI_EXPERTS_MAX_K,
                      " columns (the sums are exact in 32 bits), got ", K);
    expect_shape(a_scale, "a_scale", {M});
    if (grouped)
        expect_shape(b_scale, "b_scale", {E, N});
    else
        expect_shape(b_scale, "b_scale", {N});
    expect_device(a_scale, "a_scale", a);
    expect_device(b, "b", a);
    expect_device(b_scale, "b_scale", a);
    mi_experts_int8_args c{};
    Tensor ids, offs, bias_c;
    int64_t rows = M;
    if (grouped) {
        TORCH_CHECK_VALUE(E >= 1 && E <= MI_EXPERTS_MAX_EXPERTS, "b must hold 1 to ", MI_EXPERTS_MAX_EXPERTS,
                          " experts, got ", E);
        expect_type(*offsets, "expert_offsets", at::kInt);
        expect_shape(*offsets, "expert_offsets", {E + 1});
        expect_device(*offsets, "expert_offsets", a);
        if (row_ids && row_ids->defined()) {
            expect_type(*row_ids, "row_ids", at::kInt);
            expect_dim(*row_ids, "row_ids", 1);
            expect_device(*row_ids, "row_ids", a);
            rows = row_ids->size(0);
        }
    }
    if (bias && bias->defined()) {
        TORCH_CHECK_TYPE(bias->scalar_type() == at::kFloat || bias->scalar_type() == at::kBFloat16 ||
                             bias->scalar_type() == at::kHalf,
                         "bias must have dtype float32, bfloat16 or float16, got ", bias->scalar_type());
        expect_shape(*bias, "bias", {N});
        expect_device(*bias, "bias", a);
    }
    const bool given = out_opt && out_opt->defined();
    expect_no_grad(grouped ? "int8_grouped_matmul" : "int8_matmul", {&a_scale, &b_scale});
    if (bias) expect_no_grad("int8_matmul", {&*bias});
    if (given) expect_no_grad(grouped ? "int8_grouped_matmul" : "int8_matmul", {&*out_opt});
    if (given) out_type = out_opt->scalar_type();
    c.out_dtype = out_dtype_of(out_type);
    TORCH_CHECK_VALUE(M > 0 || rows == 0, "a has no rows, row_ids ", rows);
    if (given) {
        const Tensor none;
        expect_out(*out_opt, "out", out_type, {rows, N}, a);
        expect_apart(*out_opt, "out", {&a, &a_scale, &b, &b_scale, bias ? &*bias : &none,
                                       offsets ? offsets : &none, row_ids ? &*row_ids : &none});
        written(*out_opt);
    }
    On on(a);
    const auto opt = a.options().requires_grad(false).dtype(out_type);
    Tensor out = given ? *out_opt : at::empty({rows, N}, opt);
    if (out.numel() == 0) return out;
    const Tensor ac = rows_of(a), as = dense(a_scale), bs = dense(b_scale);
    const Tensor bc = rows_of(b);
    c.a = ac.const_data_ptr<int8_t>();
    c.a_scale = as.const_data_ptr<float>();
    c.b = bc.const_data_ptr<int8_t>();
    c.b_scale = bs.const_data_ptr<float>();
    if (bias && bias->defined()) {
        bias_c = dense(*bias);
        c.bias = bias_c.const_data_ptr();
        c.bias_dtype = out_dtype_of(bias_c.scalar_type());
    }
    c.out = out.mutable_data_ptr();
    if (grouped) {
        offs = offsets->contiguous();
        c.expert_offsets = offs.const_data_ptr<int32_t>();
        if (row_ids && row_ids->defined()) {
            ids = row_ids->contiguous();
            c.row_ids = ids.const_data_ptr<int32_t>();
        }
    }
    c.a_rows = M;
    c.rows = rows;
    c.N = N;
    c.K = K;
    c.a_stride = row_stride(ac);
    c.b_stride = N <= 1 ? K : bc.stride(-2);
    c.b_expert_stride = grouped && E > 1 ? bc.stride(0) : 0;
    c.out_stride = row_stride(out);
    c.num_experts = (int32_t)E;
    c.zero_rest = grouped && !given;
    const size_t need = mi_experts_int8_workspace_size(rows, N, K, (int32_t)E);
    Tensor ws;
    if (need) {
        ws = at::empty({(int64_t)need}, opt.dtype(at::kByte));
        c.workspace = ws.data_ptr();
        c.workspace_bytes = need;
    }
    check(mi_experts_int8_matmul(&c, on.stream));
    return out;
}

Tensor int8_matmul(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale,
                   const OptTensor& bias, at::ScalarType out_dtype, const OptTensor& out) {
    return int8_call(a, a_scale, b, b_scale, bias, nullptr, std::nullopt, out_dtype, out);
}

Tensor int8_grouped_matmul(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale,
                           const Tensor& expert_offsets, const OptTensor& row_ids, at::ScalarType out_dtype,
                           const OptTensor& out) {
    return int8_call(a, a_scale, b, b_scale, std::nullopt, &expert_offsets, row_ids, out_dtype, out);
}

}  // namespace

PYBIND11_MODULE(_mi_experts, m) {
    m.doc() = "Torch side of the expert operators (flashinfer_amd.experts, flashinfer_amd.int8)";
    m.def("sort_experts", &sort_experts);
    m.def("permute", &permute);
    m.def("unpermute", &unpermute);
    m.def("quantize", &quantize);
    m.def("int8_matmul", &int8_matmul);
    m.def("int8_grouped_matmul", &int8_grouped_matmul);
}
