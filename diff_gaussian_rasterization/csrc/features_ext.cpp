// features_ext.cpp -- the learned-feature operators as autograd nodes over the C ABI (include/e3dgs_hip.h): embedding, layer
// norm, distillation.  Bound by event_3dgs_amd.features and event_3dgs_amd.losses, which hold the documentation; this file
// checks the arguments, lays tensors out where the ABI needs it, allocates the results on the tensors' device and launches
// on the current stream of that device.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <cmath>
#include <stdexcept>
#include <string>
#include <tuple>

#include "e3dgs_hip.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Guard = c10::hip::HIPGuardMasqueradingAsCUDA;      // (torch-ROCm tensors say "cuda")

void check(int rc, const char* what) {
    if (rc != 0) throw std::runtime_error(std::string(what) + " failed (code " + std::to_string(rc) + "): " + e3dgs_last_error());
}
void* stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

int dtype_of(const Tensor& t, const char* name) {
    if (t.scalar_type() == torch::kFloat32) return E3DGS_F32;
    if (t.scalar_type() == torch::kFloat16) return E3DGS_F16;
    TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be float32, float16 or bfloat16");
    return E3DGS_BF16;
}
int index_bytes_of(const Tensor& t) {
    TORCH_CHECK(t.scalar_type() == torch::kInt32 || t.scalar_type() == torch::kInt64, "index must be int32 or int64");
    return t.scalar_type() == torch::kInt64 ? 8 : 4;
}
void on_gpu(const Tensor& t, const char* name) { TORCH_CHECK(t.is_cuda(), name, " must be a CUDA/HIP tensor (this op has no CPU path)"); }
void same_device(const Tensor& t, const Tensor& with, const char* name) {
    on_gpu(t, name);
    TORCH_CHECK(t.device() == with.device(), name, " is on ", t.device(), ", the operator runs on ", with.device());
}
// a second derivative would silently be zero: refuse the graph of the gradient
void once(const char* who) {
    TORCH_CHECK(!at::GradMode::is_enabled(), who, " is differentiable once only (create_graph is not supported)");
}
// ... and so would a forward-mode derivative, which needs no requires_grad
void no_tangent(const char* who, std::initializer_list<Tensor> inputs) {
    for (const Tensor& t : inputs)
        TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), who, " has no forward-mode derivative (its inputs must not be dual tensors)");
}
char* bytes(const Tensor& t) { return reinterpret_cast<char*>(t.data_ptr()); }
Tensor scratch_of(size_t n, const Tensor& like) { return torch::empty({(int64_t)n}, like.options().dtype(torch::kByte)); }

struct Rows {                                     // a tensor as rows of `n` entries, the entry dimension anywhere
    Tensor t;                                     // keeps the memory
    size_t row_stride, entry_stride;
};
// Without a copy when the other dimensions run through memory in one stride; by a copy with the entries last otherwise.
// (No tensor views: each would cost a small call a microsecond.)
Rows rows_of(const Tensor& t, int64_t dim) {
    const auto sizes = t.sizes(), strides = t.strides();
    int64_t stride = sizes[dim], next = -1;       // of the rows (any for a single one); what the next outer dimension's has to be
    bool one = true;
    for (int64_t d = t.dim() - 1; d >= 0; --d) {
        if (d == dim || sizes[d] == 1) continue;
        if (next < 0) stride = strides[d];
        else one = one && strides[d] == next;
        next = strides[d] * sizes[d];
    }
    if (one) return {t, (size_t)stride, (size_t)(sizes[dim] == 1 ? 1 : strides[dim])};
    const int64_t n = sizes[dim];
    return {t.movedim(dim, -1).contiguous(), (size_t)n, 1};
}

// ... with the values of a row next to each other
Rows rows_of(const Tensor& t) {
    Rows r = rows_of(t, t.dim() - 1);
    if (r.entry_stride != 1) r = {t.contiguous(), (size_t)t.size(-1), 1};
    return r;
}

// ------------------------------------------------------------------------------------------------ embedding
Tensor embedding_forward(const Tensor& index, const Tensor& table, double scale) {
    const Guard guard(table.device());
    std::vector<int64_t> shape = index.sizes().vec();
    shape.push_back(table.size(1));
    Tensor out = torch::empty(shape, table.options());
    const Tensor idx = index.contiguous();
    const Rows tab = rows_of(table);
    check(e3dgs_embedding_forward((size_t)idx.numel(), (size_t)table.size(0), (size_t)table.size(1), idx.data_ptr(),
                                  index_bytes_of(idx), tab.t.data_ptr(), tab.row_stride, dtype_of(table, "table"),
                                  (float)scale, out.data_ptr(), stream()),
          "e3dgs_embedding_forward");
    return out;
}

struct EmbeddingFunction : public torch::autograd::Function<EmbeddingFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& index, const Tensor& table, double scale) {
        ctx->save_for_backward({index});
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        return embedding_forward(index, table, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("embedding");
        const auto saved = ctx->get_saved_variables();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        no_tangent("embedding", {grads[0]});
        const Guard guard(grads[0].device());
        const int64_t rows = ctx->saved_data["rows"].toInt();
        const Tensor index = saved[0].contiguous();
        const Rows g = rows_of(grads[0]);
        const int64_t dim = g.t.size(-1), n = index.numel();
        Tensor d = torch::empty({rows, dim}, g.t.options());
        Tensor scratch = scratch_of(e3dgs_embedding_backward_scratch_bytes((size_t)n, (size_t)rows, (size_t)dim), g.t);
        check(e3dgs_embedding_backward((size_t)n, (size_t)rows, (size_t)dim, index.data_ptr(), index_bytes_of(index),
                                       g.t.data_ptr(), g.row_stride, dtype_of(g.t, "grad"),
                                       (float)ctx->saved_data["scale"].toDouble(), d.data_ptr(), bytes(scratch), stream()),
              "e3dgs_embedding_backward");
        return {Tensor(), d, Tensor()};
    }
};

Tensor embedding(const Tensor& index, const Tensor& table, double scale) {
    on_gpu(table, "table");
    same_device(index, table, "index");
    TORCH_CHECK(table.dim() == 2 && table.size(1) >= 1, "table must have dimensions (rows, dim)");
    TORCH_CHECK(table.size(1) <= E3DGS_FEATURE_MAX_DIM, "at most ", E3DGS_FEATURE_MAX_DIM, " values to a row");
    TORCH_CHECK(index.numel() < 0x7FFFFFFF && table.size(0) < 0x7FFFFFFF, "embedding takes fewer than 2^31 - 1 indices and rows");
    TORCH_CHECK(std::isfinite((float)scale), "scale must be finite (in float32)");
    dtype_of(table, "table");
    index_bytes_of(index);
    no_tangent("embedding", {table});
    if (!(at::GradMode::is_enabled() && table.requires_grad())) return embedding_forward(index, table, scale);
    return EmbeddingFunction::apply(index, table, scale);
}

// ------------------------------------------------------------------------------------------------ layer norm
std::tuple<Tensor, Tensor> layer_norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, bool stats) {
    const Guard guard(x.device());
    const Rows r = rows_of(x);
    const int64_t dim = x.size(-1), rows = x.numel() / dim;
    Tensor out = torch::empty(x.sizes(), x.options());
    Tensor st = stats ? torch::empty({2, rows}, x.options().dtype(torch::kFloat32)) : Tensor();
    const Tensor w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
    const int affine = w.defined() ? dtype_of(w, "weight") : b.defined() ? dtype_of(b, "bias") : E3DGS_F32;
    check(e3dgs_layer_norm_forward((size_t)rows, (size_t)dim, r.t.data_ptr(), r.row_stride, dtype_of(x, "x"),
                                   w.defined() ? w.data_ptr() : nullptr, b.defined() ? b.data_ptr() : nullptr, affine,
                                   (float)eps, out.data_ptr(), stats ? st.data_ptr<float>() : nullptr,
                                   stats ? st.data_ptr<float>() + rows : nullptr, stream()),
          "e3dgs_layer_norm_forward");
    return std::make_tuple(out, st);
}

struct LayerNormFunction : public torch::autograd::Function<LayerNormFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& weight_,
                          const c10::optional<Tensor>& bias_, double eps) {
        const Tensor weight = weight_ ? *weight_ : Tensor(), bias = bias_ ? *bias_ : Tensor();
        auto r = layer_norm_forward(x, weight, bias, eps, true);
        ctx->save_for_backward({x, weight, std::get<1>(r)});
        ctx->saved_data["bias"] = bias.defined();
        ctx->saved_data["affine"] = (int64_t)(weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type());
        return std::get<0>(r);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("layer_norm");
        const auto saved = ctx->get_saved_variables();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        no_tangent("layer_norm", {grads[0]});
        const Tensor &x = saved[0], &weight = saved[1], &st = saved[2];
        const Guard guard(x.device());
        const Rows r = rows_of(x), g = rows_of(grads[0]);
        const int64_t dim = x.size(-1), rows = x.numel() / dim;
        const Tensor w = weight.defined() ? weight.contiguous() : weight;
        const auto affine = x.options().dtype((c10::ScalarType)ctx->saved_data["affine"].toInt());
        // (what this call of the backward pass asks for; the inputs are numbered without those that are None)
        const size_t bias_input = weight.defined() ? 2 : 1;
        Tensor dx = ctx->needs_input_grad(0) ? torch::empty(x.sizes(), x.options()) : Tensor();
        Tensor dw = weight.defined() && ctx->needs_input_grad(1) ? torch::empty({dim}, affine) : Tensor();
        Tensor db = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(bias_input) ? torch::empty({dim}, affine) : Tensor();
        Tensor scratch;
        if (dw.defined() || db.defined()) scratch = scratch_of(e3dgs_layer_norm_backward_scratch_bytes((size_t)rows, (size_t)dim), x);
        const auto kind = affine.dtype().toScalarType();
        check(e3dgs_layer_norm_backward((size_t)rows, (size_t)dim, g.t.data_ptr(), g.row_stride, r.t.data_ptr(), r.row_stride,
                                        dtype_of(x, "x"), w.defined() ? w.data_ptr() : nullptr,
                                        kind == torch::kFloat32 ? E3DGS_F32 : kind == torch::kFloat16 ? E3DGS_F16 : E3DGS_BF16,
                                        st.data_ptr<float>(), st.data_ptr<float>() + rows, dx.defined() ? dx.data_ptr() : nullptr,
                                        dw.defined() ? dw.data_ptr() : nullptr, db.defined() ? db.data_ptr() : nullptr,
                                        scratch.defined() ? bytes(scratch) : nullptr, stream()),
              "e3dgs_layer_norm_backward");
        return {dx, dw, db, Tensor()};
    }
};

Tensor layer_norm(const Tensor& x, const c10::optional<Tensor>& weight_, const c10::optional<Tensor>& bias_, double eps) {
    const Tensor weight = weight_ ? *weight_ : Tensor(), bias = bias_ ? *bias_ : Tensor();
    on_gpu(x, "x");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "x must have at least one value to a row");
    TORCH_CHECK(x.size(-1) <= E3DGS_FEATURE_MAX_DIM, "at most ", E3DGS_FEATURE_MAX_DIM, " values to a row");
    TORCH_CHECK(std::isfinite((float)eps) && eps >= 0.0, "eps must be finite (in float32) and not negative");
    dtype_of(x, "x");
    bool grad = x.requires_grad();
    for (const auto& p : {std::make_pair(&weight, "weight"), std::make_pair(&bias, "bias")}) {
        if (!p.first->defined()) continue;
        same_device(*p.first, x, p.second);
        dtype_of(*p.first, p.second);
        TORCH_CHECK(p.first->dim() == 1 && p.first->size(0) == x.size(-1), p.second, " must have dimensions (", x.size(-1), ",)");
        grad = grad || p.first->requires_grad();
    }
    TORCH_CHECK(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), "weight and bias must have one type");
    no_tangent("layer_norm", {x, weight, bias});
    if (!(at::GradMode::is_enabled() && grad)) return std::get<0>(layer_norm_forward(x, weight, bias, eps, false));
    return LayerNormFunction::apply(x, weight_, bias_, eps);
}

// ------------------------------------------------------------------------------------------------ distillation
// The scores as (rows, classes) in one of the two layouts of the ABI, and the labels with whatever strides they have.
struct Scores {
    Rows logits, teacher, index;
    std::vector<int64_t> shape;                   // of the logits
    int64_t class_dim;
    size_t rows, classes, k;
    bool planes;
};

Scores scores_of(const Tensor& logits, const Tensor& teacher, const Tensor& index, int64_t class_dim) {
    Scores s;
    s.class_dim = class_dim;
    s.shape = logits.sizes().vec();
    s.classes = (size_t)logits.size(class_dim);
    s.rows = (size_t)logits.numel() / s.classes;
    s.k = (size_t)teacher.size(class_dim);
    s.logits = rows_of(logits, class_dim);
    s.teacher = rows_of(teacher, class_dim);
    s.index = rows_of(index, class_dim);
    s.planes = s.rows > 1 && s.logits.entry_stride != 1 && s.logits.row_stride == 1 && s.classes <= E3DGS_DISTILL_MAX_PLANES &&
               s.k <= E3DGS_DISTILL_MAX_PLANES;
    if (!s.planes && s.logits.entry_stride != 1) s.logits = {logits.movedim(class_dim, -1).contiguous(), s.classes, 1};
    return s;
}

// The gradient in the layout of the scores, and in their shape.
Tensor empty_grad(const Scores& s) {
    const auto opt = s.logits.t.options();
    const int64_t last = (int64_t)s.shape.size() - 1;
    if (s.class_dim == (s.planes ? 0 : last)) return torch::empty(s.shape, opt);
    std::vector<int64_t> shape = s.shape;         // classes first (planes) or last in memory, back to their place in the shape
    const int64_t to = s.planes ? 0 : last;
    shape.erase(shape.begin() + s.class_dim);
    shape.insert(shape.begin() + to, (int64_t)s.classes);
    return torch::empty(shape, opt).movedim(to, s.class_dim);
}
size_t grad_row(const Scores& s) { return s.planes ? 1 : s.classes; }
size_t grad_class(const Scores& s) { return s.planes ? s.rows : 1; }

// value (0-dim, or one per row) and what the backward call needs; fills `grad` (of empty_grad) if it is defined
std::tuple<Tensor, Tensor> distill_forward(const Scores& s, double temperature, int64_t reduction, const Tensor& grad) {
    const auto opt = s.logits.t.options().dtype(torch::kFloat32);
    const size_t n_stats = (2 * s.rows + 1 + 1) / 2 * 2;                      // (the scratch behind it is 8-byte aligned)
    Tensor stats = torch::empty({(int64_t)(n_stats + (e3dgs_distill_scratch_bytes(s.rows) + 3) / 4)}, opt);
    Tensor loss = torch::empty({}, opt);
    Tensor row_loss;
    if (reduction == 0) {
        std::vector<int64_t> shape = s.shape;
        shape.erase(shape.begin() + s.class_dim);
        row_loss = torch::empty(shape, opt);
    }
    check(e3dgs_distill_forward(s.rows, s.classes, s.k, s.logits.t.data_ptr(), s.logits.row_stride, s.logits.entry_stride,
                                dtype_of(s.logits.t, "logits"), s.teacher.t.data_ptr(), s.teacher.row_stride,
                                s.teacher.entry_stride, dtype_of(s.teacher.t, "teacher_logits"), s.index.t.data_ptr(),
                                s.index.row_stride, s.index.entry_stride, index_bytes_of(s.index.t),
                                (float)temperature, (int)reduction, stats.data_ptr<float>(),
                                row_loss.defined() ? row_loss.data_ptr<float>() : nullptr, loss.data_ptr<float>(),
                                grad.defined() ? grad.data_ptr() : nullptr, grad_row(s), grad_class(s),
                                reinterpret_cast<char*>(stats.data_ptr<float>() + n_stats), stream()),
          "e3dgs_distill_forward");
    return std::make_tuple(reduction == 0 ? row_loss : loss, stats);
}

Tensor distill_backward(const Scores& s, double temperature, int64_t reduction, const Tensor& stats, const Tensor& d_loss) {
    Tensor grad = empty_grad(s);
    check(e3dgs_distill_backward(s.rows, s.classes, s.k, s.logits.t.data_ptr(), s.logits.row_stride, s.logits.entry_stride,
                                 dtype_of(s.logits.t, "logits"), s.teacher.t.data_ptr(), s.teacher.row_stride,
                                 s.teacher.entry_stride, dtype_of(s.teacher.t, "teacher_logits"), s.index.t.data_ptr(),
                                 s.index.row_stride, s.index.entry_stride, index_bytes_of(s.index.t),
                                 (float)temperature, (int)reduction, stats.data_ptr<float>(), d_loss.data_ptr<float>(), grad.data_ptr(), grad_row(s), grad_class(s), stream()),
          "e3dgs_distill_backward");
    return grad;
}

struct DistillFunction : public torch::autograd::Function<DistillFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher, const Tensor& index,
                          double temperature, int64_t reduction, int64_t class_dim) {
        const Guard guard(logits.device());
        auto r = distill_forward(scores_of(logits, teacher, index, class_dim), temperature, reduction, Tensor());
        ctx->save_for_backward({logits, teacher, index, std::get<1>(r)});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["reduction"] = reduction;
        ctx->saved_data["class_dim"] = class_dim;
        return std::get<0>(r);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once("distill_loss");
        const auto saved = ctx->get_saved_variables();
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
        no_tangent("distill_loss", {grads[0]});
        const Guard guard(saved[0].device());
        const Scores s = scores_of(saved[0], saved[1], saved[2], ctx->saved_data["class_dim"].toInt());
        const Tensor g = grads[0].to(torch::kFloat32).contiguous();
        Tensor d = distill_backward(s, ctx->saved_data["temperature"].toDouble(), ctx->saved_data["reduction"].toInt(), saved[3], g);
        return {d, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

int64_t distill_check(const Tensor& logits, const Tensor& teacher, const Tensor& index, double temperature, int64_t class_dim) {
    on_gpu(logits, "logits");
    same_device(teacher, logits, "teacher_logits");
    same_device(index, logits, "teacher_index");
    dtype_of(logits, "logits");
    dtype_of(teacher, "teacher_logits");
    index_bytes_of(index);
    TORCH_CHECK(logits.dim() >= 1 && class_dim >= -logits.dim() && class_dim < logits.dim(), "class_dim is not a dimension of logits");
    if (class_dim < 0) class_dim += logits.dim();
    TORCH_CHECK(teacher.sizes() == index.sizes(), "teacher_logits and teacher_index must have the same shape");
    TORCH_CHECK(teacher.dim() == logits.dim(), "teacher_logits must have as many dimensions as logits");
    for (int64_t d = 0; d < logits.dim(); ++d)
        TORCH_CHECK(d == class_dim || teacher.size(d) == logits.size(d), "teacher_logits and logits differ in dimension ", d);
    TORCH_CHECK(logits.size(class_dim) >= 1 && logits.size(class_dim) < 0x7FFFFFFF, "logits must have between 1 and 2^31 - 2 classes");
    TORCH_CHECK(logits.numel() / logits.size(class_dim) < 0x7FFFFFFF, "distill_loss takes fewer than 2^31 - 1 rows");
    TORCH_CHECK(teacher.size(class_dim) >= 1 && teacher.size(class_dim) <= E3DGS_DISTILL_MAX_K,
                "teacher_logits must list between 1 and ", E3DGS_DISTILL_MAX_K, " classes");
    TORCH_CHECK(std::isfinite(temperature) && temperature > 1e-6 && temperature < 1e6, "temperature must lie between 1e-6 and 1e6");
    TORCH_CHECK(!teacher.requires_grad() || !at::GradMode::is_enabled(), "teacher_logits takes no gradient: detach it");
    return class_dim;
}

Tensor distill(const Tensor& logits, const Tensor& teacher, const Tensor& index, double temperature, int64_t reduction, int64_t class_dim) {
    class_dim = distill_check(logits, teacher, index, temperature, class_dim);
    no_tangent("distill_loss", {logits, teacher});
    if (at::GradMode::is_enabled() && logits.requires_grad())
        return DistillFunction::apply(logits, teacher, index, temperature, reduction, class_dim);
    const Guard guard(logits.device());
    return std::get<0>(distill_forward(scores_of(logits, teacher, index, class_dim), temperature, reduction, Tensor()));
}

std::tuple<Tensor, Tensor> distill_raw(const Tensor& logits_, const Tensor& teacher, const Tensor& index, double temperature,
                                       int64_t reduction, int64_t class_dim) {
    const Tensor logits = logits_.detach();
    class_dim = distill_check(logits, teacher.detach(), index, temperature, class_dim);
    const Guard guard(logits.device());
    at::NoGradGuard no_grad;
    const Scores s = scores_of(logits, teacher, index, class_dim);
    const Tensor grad = empty_grad(s);
    auto r = distill_forward(s, temperature, reduction, grad);
    return std::make_tuple(std::get<0>(r), grad);
}

}  // namespace

void bind_features(pybind11::module& m) {
    const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
    m.def("embedding", &embedding, free);
    m.def("layer_norm", &layer_norm, free);
    m.def("distill", &distill, free);
    m.def("distill_raw", &distill_raw, free);
}
