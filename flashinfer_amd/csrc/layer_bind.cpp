// The torch side of the layer's operators (flashinfer_amd.layer,
// flashinfer_amd.int4): checks of the tensors, allocation of results and
// workspaces, the current stream, and the gradients of the balance loss and of
// swiglu, over the C ABI of include/mi_layer.h.
//
// Built with g++ against torch's headers (no device code here).
#include "../../include/mi_layer.h"
#include "torch_common.hpp"

namespace py = pybind11;

namespace {

using namespace mitorch;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

static_assert(MI_LAYER_BF16 == MI_EXPERTS_BF16 && MI_LAYER_F32 == MI_EXPERTS_F32 && MI_LAYER_F16 == MI_EXPERTS_F16,
              "one set of element types");

void check(int rc) { TORCH_CHECK(rc == MI_LAYER_OK, "mi_layer error ", rc, ": ", mi_layer_last_error()); }

const int32_t* ints_or_null(const Tensor& t) { return t.defined() ? t.const_data_ptr<int32_t>() : nullptr; }

Tensor dense_or_none(const OptTensor& t) { return t && t->defined() ? dense(*t) : Tensor(); }

// ------------------------------------------------------------ balance loss

// What the forward and the backward pass both read.
mi_layer_balance_args balance_args(const Tensor& logits, const Tensor& offsets, const Tensor& mask,
                                   const Tensor& weights, int64_t score) {
    mi_layer_balance_args a{};
    a.logits = logits.const_data_ptr();
    a.seq_offsets = ints_or_null(offsets);
    a.mask = mask.defined() ? reinterpret_cast<const uint8_t*>(mask.const_data_ptr<bool>()) : nullptr;
    a.weights = weights.mutable_data_ptr<float>();
    a.num_tokens = logits.size(0);
    a.num_seqs = offsets.defined() ? offsets.size(0) - 1 : 1;
    a.logits_stride = row_stride(logits);
    a.num_experts = (int32_t)logits.size(1);
    a.dtype = float_dtype(logits, "logits");
    a.score = (int32_t)score;
    return a;
}

// loss, counts, weights
std::array<Tensor, 3> balance_forward(const Tensor& logits, const Tensor& ids, const Tensor& offsets,
                                      const Tensor& mask, int64_t score) {
    On on(logits);
    const auto opt = logits.options().requires_grad(false);
    const int64_t E = logits.size(1);
    Tensor loss = at::empty({}, opt.dtype(at::kFloat));
    auto shape = [&](at::ScalarType t) {
        return offsets.defined() ? at::empty({offsets.size(0) - 1, E}, opt.dtype(t)) : at::empty({E}, opt.dtype(t));
    };
    Tensor counts = shape(at::kInt), weights = shape(at::kFloat);
    const Tensor in = rows_of(logits);
    mi_layer_balance_args a = balance_args(in, offsets, mask, weights, score);
    a.topk_ids = ids.const_data_ptr<int32_t>();
    a.loss = loss.mutable_data_ptr<float>();
    a.counts = counts.mutable_data_ptr<int32_t>();
    a.top_k = (int32_t)ids.size(1);
    a.workspace_bytes = mi_layer_balance_workspace_size(a.num_tokens, a.num_seqs, a.num_experts);
    Tensor ws = at::empty({(int64_t)a.workspace_bytes}, opt.dtype(at::kByte));
    a.workspace = ws.data_ptr();
    check(mi_layer_balance(&a, on.stream));
    return {loss, counts, weights};
}

struct BalanceFn : torch::autograd::Function<BalanceFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& ids,
                                 const OptTensor& offsets, const OptTensor& mask, int64_t score) {
        const auto [loss, counts, weights] =
            balance_forward(logits, ids, or_none(offsets), or_none(mask), score);
        ctx->save_for_backward({logits, or_none(offsets), or_none(mask), weights});
        ctx->saved_data["score"] = score;
        ctx->mark_non_differentiable({counts});
        return {loss, counts};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "balance_loss() has no second derivative (create_graph=True)");
        TORCH_CHECK(!has_tangent(grads[0]), "balance_loss() has no second derivative (a gradient with a tangent)");
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &weights = saved[3];
        On on(logits);
        const Tensor in = rows_of(logits), g = dense(grads[0]);
        Tensor out = at::empty(logits.sizes(), logits.options().requires_grad(false));
        const mi_layer_balance_args a =
            balance_args(in, saved[1], saved[2], weights, ctx->saved_data["score"].toInt());
        check(mi_layer_balance_backward(&a, g.const_data_ptr<float>(), out.mutable_data_ptr(), row_stride(out),
                                        on.stream));
        return {out, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

py::tuple balance_loss(const Tensor& logits, const Tensor& topk_ids, const OptTensor& seq_offsets,
                       const OptTensor& mask, int64_t score) {
    expect_dim(logits, "logits", 2);
    expect_dim(topk_ids, "topk_ids", 2);
    float_dtype(logits, "logits");
    expect_type(topk_ids, "topk_ids", at::kInt);
    expect_no_tangent("balance_loss", {&logits});
    expect_gpu(logits, "logits");
    const int64_t T = logits.size(0), E = logits.size(1), k = topk_ids.size(1);
    TORCH_CHECK_VALUE(E >= 1 && E <= MI_LAYER_MAX_EXPERTS, "logits must have 1 to ", MI_LAYER_MAX_EXPERTS,
                      " experts, got ", E);
    TORCH_CHECK_VALUE(topk_ids.size(0) == T, "topk_ids has ", topk_ids.size(0), " tokens, logits ", T);
    TORCH_CHECK_VALUE(k >= 1 && k <= MI_LAYER_MAX_TOP_K, "topk_ids must have 1 to ", MI_LAYER_MAX_TOP_K,
                      " experts per token, got ", k);
    expect_device(topk_ids, "topk_ids", logits);
    OptTensor offsets, kept;
    if (seq_offsets && seq_offsets->defined()) {
        expect_type(*seq_offsets, "seq_offsets", at::kInt);
        expect_dim(*seq_offsets, "seq_offsets", 1);
        TORCH_CHECK_VALUE(seq_offsets->size(0) >= 2, "seq_offsets must have an entry for each sequence and the end");
        expect_device(*seq_offsets, "seq_offsets", logits);
        offsets = seq_offsets->contiguous();
    }
    if (mask && mask->defined()) {
        expect_type(*mask, "mask", at::kBool);
        expect_shape(*mask, "mask", {T});
        expect_device(*mask, "mask", logits);
        kept = mask->contiguous();
    }
    const Tensor ids = topk_ids.contiguous();
    if (at::GradMode::is_enabled() && logits.requires_grad()) {
        const variable_list out = BalanceFn::apply(logits, ids, offsets, kept, score);
        return py::make_tuple(out[0], out[1]);
    }
    const auto out = balance_forward(logits, ids, or_none(offsets), or_none(kept), score);
    return py::make_tuple(out[0], out[1]);
}

// ------------------------------------------------------------------ swiglu

struct Dropout {
    int64_t threshold, seed;
    Tensor seed_ptr;  // undefined: seed
};

void swiglu_run(const Tensor& x, const Tensor& grad, const Tensor& num_rows, const Dropout& d, const Tensor& out,
                bool zero_rest) {
    if (out.numel() == 0) return;
    On on(x);
    const Tensor in = rows_of(x), g = grad.defined() ? rows_of(grad) : grad;
    mi_layer_swiglu_args a{};
    a.x = in.const_data_ptr();
    a.out = out.mutable_data_ptr();
    a.num_rows = ints_or_null(num_rows);
    a.seed = (uint64_t)d.seed;
    a.seed_ptr = d.seed_ptr.defined() ? reinterpret_cast<const uint64_t*>(d.seed_ptr.const_data_ptr<int64_t>()) : nullptr;
    a.max_rows = in.size(0);
    a.I = in.size(1) / 2;
    a.x_stride = row_stride(in);
    a.out_stride = row_stride(out);
    a.dtype = float_dtype(in, "x");
    a.threshold = (int32_t)d.threshold;
    a.zero_rest = zero_rest;
    if (g.defined()) {
        a.grad = g.const_data_ptr();
        a.grad_stride = row_stride(g);
        check(mi_layer_swiglu_backward(&a, on.stream));
    } else {
        check(mi_layer_swiglu(&a, on.stream));
    }
}

Tensor swiglu_new(const Tensor& x, const Tensor& num_rows, const Dropout& d) {
    c10::DeviceGuard guard(x.device());
    Tensor out = at::empty({x.size(0), x.size(1) / 2}, x.options().requires_grad(false));
    swiglu_run(x, Tensor(), num_rows, d, out, true);
    return out;
}

struct SwigluFn : torch::autograd::Function<SwigluFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& num_rows, int64_t threshold,
                          int64_t seed, const OptTensor& seed_ptr) {
        const Dropout d{threshold, seed, or_none(seed_ptr)};
        ctx->save_for_backward({x, or_none(num_rows), d.seed_ptr});
        ctx->saved_data["threshold"] = threshold;
        ctx->saved_data["seed"] = seed;
        return swiglu_new(x, or_none(num_rows), d);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "swiglu() has no second derivative (create_graph=True)");
        TORCH_CHECK(!has_tangent(grads[0]), "swiglu() has no second derivative (a gradient with a tangent)");
        const auto saved = ctx->get_saved_variables();
        const Tensor& x = saved[0];
        const Dropout d{ctx->saved_data["threshold"].toInt(), ctx->saved_data["seed"].toInt(), saved[2]};
        c10::DeviceGuard guard(x.device());
        Tensor dx = at::empty(x.sizes(), x.options().requires_grad(false));
        swiglu_run(x, grads[0], saved[1], d, dx, true);
        return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor swiglu(const Tensor& x, int64_t threshold, int64_t seed, const OptTensor& seed_ptr, const OptTensor& num_rows,
              const OptTensor& out) {
    expect_dim(x, "x", 2);
    float_dtype(x, "x");
    expect_no_tangent("swiglu", {&x, &or_none(out)});
    expect_gpu(x, "x");
    const int64_t M = x.size(0), C = x.size(1);
    TORCH_CHECK_VALUE(C >= 2 && C % 2 == 0, "x must have 2 I columns, got ", C);
    Dropout d{threshold, seed, Tensor()};
    Tensor count;
    if (num_rows && num_rows->defined()) {
        expect_type(*num_rows, "num_rows", at::kInt);
        TORCH_CHECK_VALUE(num_rows->numel() == 1, "num_rows must hold one number, got shape ", num_rows->sizes());
        expect_device(*num_rows, "num_rows", x);
        count = *num_rows;
    }
    if (threshold && seed_ptr && seed_ptr->defined()) {
        expect_type(*seed_ptr, "seed", at::kLong);
        TORCH_CHECK_VALUE(seed_ptr->numel() == 1, "seed must hold one number, got shape ", seed_ptr->sizes());
        expect_device(*seed_ptr, "seed", x);
        d.seed_ptr = *seed_ptr;
    }
    const bool needs = at::GradMode::is_enabled() && x.requires_grad();
    no_grad_out("swiglu", needs, out);
    if (out && out->defined()) {
        expect_out(*out, "out", x.scalar_type(), {M, C / 2}, x);
        expect_apart(*out, "out", {&x, &count, &d.seed_ptr});
        written(*out);
        swiglu_run(x, Tensor(), count, d, *out, false);
        return *out;
    }
    if (needs)
        return SwigluFn::apply(x, count.defined() ? OptTensor(count) : std::nullopt, threshold, seed,
                               d.seed_ptr.defined() ? OptTensor(d.seed_ptr) : std::nullopt);
    return swiglu_new(x, count, d);
}

// ------------------------------------------------------------ 4-bit weights

// Sizes of the weights of E experts (0: dense), and the checks they share.
struct Int4Sizes {
    int64_t E, N, K, nt, kt, groups;
    Int4Sizes(int64_t E, int64_t N, int64_t K, int64_t group)
        : E(E), N(N), K(K), nt((N + MI_LAYER_INT4_TILE_N - 1) / MI_LAYER_INT4_TILE_N),
          kt((K + MI_LAYER_INT4_TILE_K - 1) / MI_LAYER_INT4_TILE_K) {
        TORCH_CHECK_VALUE(group >= MI_LAYER_INT4_MIN_GROUP && group <= 1 << 24 && (group & (group - 1)) == 0,
                          "group_size must be a power of two from ", MI_LAYER_INT4_MIN_GROUP, " to 2^24, got ", group);
        TORCH_CHECK_VALUE(E >= 0 && E <= MI_LAYER_MAX_EXPERTS, "weights must have 1 to ", MI_LAYER_MAX_EXPERTS,
                          " experts, got ", E);
        TORCH_CHECK_VALUE(N >= 1 && N <= 1 << 24 && K >= 1 && K <= 1 << 24,
                          "weights must have 1 to 2^24 channels and columns, got ", N, " x ", K);
        groups = (K + group - 1) / group;
    }
    std::vector<int64_t> with(std::initializer_list<int64_t> rest) const {
        std::vector<int64_t> s;
        if (E) s.push_back(E);
        s.insert(s.end(), rest);
        return s;
    }
    std::vector<int64_t> packed() const { return with({nt, kt, MI_LAYER_INT4_TILE_N * MI_LAYER_INT4_TILE_K / 2}); }
    std::vector<int64_t> scale() const { return with({groups, nt * MI_LAYER_INT4_TILE_N}); }
};

Int4Sizes sizes_of(const Tensor& w, const char* name, int64_t group) {
    TORCH_CHECK_VALUE(w.dim() == 2 || w.dim() == 3, name, " must have shape [N, K] or [E, N, K], got ", w.sizes());
    TORCH_CHECK_VALUE(w.dim() == 2 || w.size(0) >= 1, name, " must have an expert at least");
    return Int4Sizes(w.dim() == 3 ? w.size(0) : 0, w.size(-2), w.size(-1), group);
}

int64_t expert_stride(const Tensor& w) { return w.dim() == 3 && w.size(0) > 1 ? w.stride(0) : 0; }
int64_t channel_stride(const Tensor& w) { return w.size(-2) > 1 ? w.stride(-2) : 0; }
// Rows of consecutive values at any distances, those of experts too.
Tensor weights_of(const Tensor& w) {
    const Tensor r = rows_of(w);
    return r.dim() == 3 && r.stride(0) < 0 ? r.contiguous() : r;
}

py::tuple pack_int4(const Tensor& q, const Tensor& scale, int64_t group) {
    expect_type(q, "q", at::kChar);
    const int dtype = float_dtype(scale, "scale");
    const Int4Sizes z = sizes_of(q, "q", group);
    expect_no_tangent("pack_int4", {&scale});
    expect_gpu(q, "q");
    expect_shape(scale, "scale", z.with({z.N, z.groups}));
    expect_device(scale, "scale", q);
    expect_no_grad("pack_int4", {&scale});
    On on(q);
    const Tensor in = weights_of(q), s = dense(scale);
    Tensor packed = at::empty(z.packed(), q.options().dtype(at::kByte));
    Tensor laid = at::empty(z.scale(), s.options().requires_grad(false));
    check(mi_layer_pack_int4(in.const_data_ptr<int8_t>(), expert_stride(in), channel_stride(in), s.const_data_ptr(),
                             dtype, z.E, z.N, z.K, (int32_t)group, packed.mutable_data_ptr<uint8_t>(),
                             laid.mutable_data_ptr(), on.stream));
    return py::make_tuple(packed, laid);
}

py::tuple quantize_int4(const Tensor& w, int64_t group) {
    const int dtype = float_dtype(w, "w");
    const Int4Sizes z = sizes_of(w, "w", group);
    expect_no_tangent("quantize_int4", {&w});
    expect_gpu(w, "w");
    expect_no_grad("quantize_int4", {&w});
    On on(w);
    const Tensor in = weights_of(w);
    const auto opt = w.options().requires_grad(false);
    Tensor packed = at::empty(z.packed(), opt.dtype(at::kByte)), scale = at::empty(z.scale(), opt.dtype(at::kFloat));
    check(mi_layer_quantize_int4(dtype, in.const_data_ptr(), expert_stride(in), channel_stride(in), z.E, z.N, z.K,
                                 (int32_t)group, packed.mutable_data_ptr<uint8_t>(), scale.mutable_data_ptr<float>(),
                                 on.stream));
    return py::make_tuple(packed, scale);
}

// packed, scale, N, K, group_size as flashinfer_amd.int4.Int4Weights holds them.
Tensor int4_matmul(const char* what, const Tensor& x, const Tensor& packed, const Tensor& scale, int64_t N, int64_t K,
                   int64_t group, const OptTensor& bias, const OptTensor& offsets, const OptTensor& row_ids,
                   std::optional<at::ScalarType> out_type, const OptTensor& out_opt) {
    const bool grouped = offsets && offsets->defined(), given = out_opt && out_opt->defined();
    expect_dim(x, "x", 2);
    TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
                     "x must have dtype bfloat16 or float16, got ", x.scalar_type());
    expect_type(packed, "w.packed", at::kByte);
    TORCH_CHECK_TYPE(scale.scalar_type() == at::kFloat || scale.scalar_type() == x.scalar_type(),
                     "w.scale must have dtype float32 or that of x, got ", scale.scalar_type());
    expect_dim(packed, "w.packed", grouped ? 4 : 3);
    const Int4Sizes z(grouped ? packed.size(0) : 0, N, K, group);
    TORCH_CHECK_VALUE(!grouped || z.E >= 1, "w must hold 1 expert at least");
    expect_shape(packed, "w.packed", z.packed());
    expect_shape(scale, "w.scale", z.scale());
    TORCH_CHECK_VALUE(packed.is_contiguous() && scale.is_contiguous() && !scale.is_neg(), "w must be contiguous");
    const Tensor& b = or_none(bias);
    expect_no_tangent(what, {&x, &scale, &b, &or_none(out_opt)});
    expect_gpu(x, "x");
    TORCH_CHECK_VALUE(x.size(1) == K, "x must have ", K, " columns as w has, got shape ", x.sizes());
    expect_device(packed, "w.packed", x);
    expect_device(scale, "w.scale", x);
    int64_t rows = x.size(0);
    Tensor offs, ids;
    if (grouped) {
        expect_type(*offsets, "expert_offsets", at::kInt);
        expect_shape(*offsets, "expert_offsets", {z.E + 1});
        expect_device(*offsets, "expert_offsets", x);
        offs = offsets->contiguous();
        if (row_ids && row_ids->defined()) {
            expect_type(*row_ids, "row_ids", at::kInt);
            expect_dim(*row_ids, "row_ids", 1);
            expect_device(*row_ids, "row_ids", x);
            ids = row_ids->contiguous();
            rows = ids.size(0);
        }
    }
    if (b.defined()) {
        float_dtype(b, "bias");
        expect_shape(b, "bias", {N});
        expect_device(b, "bias", x);
    }
    expect_no_grad(what, {&x, &scale, &b, &or_none(out_opt)});
    const at::ScalarType type = given ? out_opt->scalar_type() : out_type ? *out_type : x.scalar_type();
    mi_layer_int4_args a{};
    a.out_dtype = out_dtype_of(type);
    TORCH_CHECK_VALUE(x.size(0) > 0 || rows == 0, "x has no rows, row_ids ", rows);
    if (given) {
        expect_out(*out_opt, "out", type, {rows, N}, x);
        expect_apart(*out_opt, "out", {&x, &packed, &scale, &b, &or_none(offsets), &or_none(row_ids)});
        written(*out_opt);
    }
    On on(x);
    const auto opt = x.options().requires_grad(false);
    Tensor out = given ? *out_opt : at::empty({rows, N}, opt.dtype(type));
    if (out.numel() == 0) return out;
    const Tensor in = rows_of(x), bc = b.defined() ? dense(b) : b;
    a.x = in.const_data_ptr();
    a.w = packed.const_data_ptr<uint8_t>();
    a.scale = scale.const_data_ptr();
    if (bc.defined()) {
        a.bias = bc.const_data_ptr();
        a.bias_dtype = float_dtype(bc, "bias");
    }
    a.out = out.mutable_data_ptr();
    a.expert_offsets = ints_or_null(offs);
    a.row_ids = ints_or_null(ids);
    a.x_rows = in.size(0);
    a.rows = rows;
    a.N = N;
    a.K = K;
    a.x_stride = row_stride(in);
    a.out_stride = row_stride(out);
    a.group_size = (int32_t)group;
    a.num_experts = (int32_t)z.E;
    a.x_dtype = float_dtype(in, "x");
    a.scale_dtype = float_dtype(scale, "w.scale");
    a.zero_rest = grouped && !given;
    const bool aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_stride % 8 == 0 && K % 8 == 0;
    a.workspace_bytes = mi_layer_int4_workspace_size(a.x_rows, K, aligned);
    Tensor ws;
    if (a.workspace_bytes) {
        ws = at::empty({(int64_t)a.workspace_bytes}, opt.dtype(at::kByte));
        a.workspace = ws.data_ptr();
    }
    check(mi_layer_int4_matmul(&a, on.stream));
    return out;
}

}  // namespace

PYBIND11_MODULE(_mi_layer, m) {
    m.doc() = "Torch side of the layer's operators (flashinfer_amd.layer, flashinfer_amd.int4)";
    m.def("balance_loss", &balance_loss);
    m.def("swiglu", &swiglu);
    m.def("pack_int4", &pack_int4);
    m.def("quantize_int4", &quantize_int4);
    m.def("int4_matmul", &int4_matmul);
}
