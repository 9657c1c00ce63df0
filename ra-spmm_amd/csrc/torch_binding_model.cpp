// torch_binding_model.cpp — torch surface of the operators at a model's ends and between
// its layers: embedding lookup, layer norm, distillation.  Checks and output allocation;
// launches use the current torch stream.
#include <cmath>
#include <string>
#include <tuple>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include "torch_checks.hpp"

namespace {

Tensor workspace(int64_t bytes, const Tensor& like) { return torch::empty({bytes}, like.options().dtype(torch::kUInt8)); }

bool is_int64(const Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == torch::kInt64 || t.scalar_type() == torch::kInt32, name, " must be int32 or int64");
    return t.scalar_type() == torch::kInt64;
}

int64_t matrix_stride(const Tensor& t, const char* name) {
    TORCH_CHECK(t.dim() == 2, name, " must have two dimensions, has shape ", t.sizes());
    return row_stride(t, name);
}

// t itself where only its rows are strided, else a contiguous copy.
Tensor with_rows(const Tensor& t) {
    if (t.is_neg()) return t.resolve_neg().contiguous();
    int64_t run = 1;
    for (int64_t d = t.dim() - 1; d > 0; --d) {
        if (t.size(d) > 1 && t.stride(d) != run) return t.contiguous();
        run *= t.size(d);
    }
    return t.dim() == 0 || t.size(0) <= 1 || t.stride(0) >= run ? t : t.contiguous();
}

// ------------------------------------------------------------ embedding lookup
ra_embed_shape embed_shape(const Tensor& ids, int64_t rows, int64_t dim, const Tensor& values, double scale,
                           c10::optional<int64_t> padding) {
    TORCH_CHECK(ids.is_contiguous(), "ids must be contiguous");
    TORCH_CHECK(dim > 0 && dim < INT32_MAX, "the table must have rows of at least one element");
    ra_embed_shape s{};
    s.ids64 = is_int64(ids, "ids");
    s.count = ids.numel();
    s.rows = rows;
    s.dim = static_cast<int32_t>(dim);
    s.dtype = dtype_of(values, "the table and its gradients");
    s.has_padding = padding.has_value();
    s.padding = padding.value_or(0);
    s.scale = static_cast<float>(scale);
    return s;
}

Tensor run_embed(Tensor ids, Tensor table, double scale, c10::optional<int64_t> padding) {
    check_no_tangents({{table, "table"}});
    check_no_proxies("table");
    check_memory(table, "table");
    check_memory(ids, "ids");
    TORCH_CHECK(ids.is_cuda(), "ids must be a CUDA tensor");
    const auto dev = ids.device();
    check_on(table, "table", dev);
    const int64_t ld = matrix_stride(table, "table");
    ra_embed_shape s = embed_shape(ids, table.size(0), table.size(1), table, scale, padding);
    s.ld_table = ld;
    const c10::DeviceGuard guard(dev);
    auto size = ids.sizes().vec();
    size.push_back(table.size(1));
    auto out = torch::empty(size, table.options());
    check(ra_embed(&s, ids.data_ptr(), table.data_ptr(), out.data_ptr(), current_stream()), "embed");
    return out;
}

Tensor run_embed_backward(Tensor ids, Tensor grad, int64_t rows, double scale, c10::optional<int64_t> padding) {
    check_memory(ids, "ids");
    TORCH_CHECK(ids.is_cuda(), "ids must be a CUDA tensor");
    const auto dev = ids.device();
    check_on(grad, "grad", dev);
    const int64_t ld = matrix_stride(grad, "grad");
    TORCH_CHECK(grad.size(0) == ids.numel(), "grad has ", grad.size(0), " rows, ids ", ids.numel());
    ra_embed_shape s = embed_shape(ids, rows, grad.size(1), grad, scale, padding);
    s.ld_grad = ld;
    const c10::DeviceGuard guard(dev);
    auto out = torch::empty({rows, grad.size(1)}, grad.options());
    int64_t bytes = 0;
    check(ra_embed_workspace(&s, &bytes), "embed backward");
    auto work = workspace(bytes, grad);
    check(ra_embed_backward(&s, ids.data_ptr(), grad.data_ptr(), out.data_ptr(), work.data_ptr(), bytes, current_stream()),
          "embed backward");
    return out;
}

// ------------------------------------------------------------------- layer norm
ra_layer_norm_shape layer_norm_shape(const Tensor& x, double eps) {
    check_cuda(x, "x");
    ra_layer_norm_shape s{};
    s.ldx = matrix_stride(x, "x");
    TORCH_CHECK(x.size(1) > 0 && x.size(1) < INT32_MAX, "x has no columns");
    s.rows = x.size(0);
    s.dim = static_cast<int32_t>(x.size(1));
    s.dtype = dtype_of(x, "x");
    s.eps = static_cast<float>(eps);
    return s;
}

const float* vector_or_null(const OptTensor& t, const char* name, int64_t n, const torch::Device& dev) {
    return t.has_value() ? f32_vector(*t, name, n, dev) : nullptr;
}

// (y, x + residual or nothing, stats or nothing)
std::tuple<Tensor, OptTensor, OptTensor> run_layer_norm(Tensor x, OptTensor residual, OptTensor weight, OptTensor bias,
                                                        double eps, bool with_stats) {
    ra_layer_norm_shape s = layer_norm_shape(x, eps);
    const auto dev = x.device();
    if (residual.has_value()) {
        check_on(*residual, "residual", dev);
        TORCH_CHECK(residual->scalar_type() == x.scalar_type() && residual->sizes() == x.sizes(),
                    "residual must have x's dtype and shape");
        s.ldr = matrix_stride(*residual, "residual");
    }
    const float* const w = vector_or_null(weight, "weight", x.size(1), dev);
    const float* const b = vector_or_null(bias, "bias", x.size(1), dev);
    const c10::DeviceGuard guard(dev);
    auto y = torch::empty(x.sizes(), x.options());
    OptTensor sum, stats;
    if (residual.has_value()) sum = torch::empty(x.sizes(), x.options());
    if (with_stats) stats = torch::empty({x.size(0), 2}, x.options().dtype(torch::kFloat32));
    check(ra_layer_norm(&s, x.data_ptr(), residual.has_value() ? residual->data_ptr() : nullptr, w, b, y.data_ptr(),
                        sum.has_value() ? sum->data_ptr() : nullptr, with_stats ? stats->data_ptr<float>() : nullptr,
                        current_stream()),
          "layer_norm");
    return {y, sum, stats};
}

// (dx, dweight, dbias)
std::tuple<Tensor, OptTensor, OptTensor> run_layer_norm_backward(Tensor h, OptTensor weight, Tensor stats, Tensor grad_y,
                                                                 OptTensor grad_sum, bool weight_grad, bool bias_grad) {
    const ra_layer_norm_shape s = layer_norm_shape(h, 0.0);
    const auto dev = h.device();
    auto check_grad = [&](const Tensor& g, const char* name) {
        check_on(g, name, dev);
        TORCH_CHECK(g.scalar_type() == h.scalar_type() && g.is_contiguous() && g.sizes() == h.sizes(), name,
                    " must be contiguous, of the output's shape and dtype");
    };
    check_grad(grad_y, "grad_y");
    if (grad_sum.has_value()) check_grad(*grad_sum, "grad_sum");
    check_on(stats, "stats", dev);
    TORCH_CHECK(stats.scalar_type() == torch::kFloat32 && stats.is_contiguous() && stats.dim() == 2 &&
                    stats.size(0) == h.size(0) && stats.size(1) == 2,
                "stats must be what run_layer_norm returned for these inputs");
    const float* const w = vector_or_null(weight, "weight", h.size(1), dev);
    const c10::DeviceGuard guard(dev);
    auto dx = torch::empty(h.sizes(), h.options());
    OptTensor dw, db;
    const auto vector = h.options().dtype(torch::kFloat32);
    if (weight_grad) dw = torch::empty({h.size(1)}, vector);
    if (bias_grad) db = torch::empty({h.size(1)}, vector);
    int64_t bytes = 0;
    check(ra_layer_norm_workspace(&s, &bytes), "layer_norm backward");
    Tensor work;
    if (weight_grad || bias_grad) work = workspace(bytes, h);
    else bytes = 0;
    check(ra_layer_norm_backward(&s, h.data_ptr(), w, stats.data_ptr<float>(), grad_y.data_ptr(),
                                 grad_sum.has_value() ? grad_sum->data_ptr() : nullptr, dx.data_ptr(),
                                 weight_grad ? dw->data_ptr<float>() : nullptr, bias_grad ? db->data_ptr<float>() : nullptr,
                                 bytes ? work.data_ptr() : nullptr, bytes, current_stream()),
          "layer_norm backward");
    return {dx, dw, db};
}

// ----------------------------------------------------------------- distillation
struct DistillCall {
    ra_distill_shape shape{};
    const void* labels = nullptr;
};

DistillCall distill_call(const Tensor& logits, const Tensor& teacher, const Tensor& ids, double temperature,
                         const OptTensor& labels, double hard, const std::string& reduction) {
    check_cuda(logits, "logits");
    const auto dev = logits.device();
    check_on(teacher, "teacher", dev);
    check_on(ids, "ids", dev);
    DistillCall c;
    ra_distill_shape& s = c.shape;
    s.ld_logits = matrix_stride(logits, "logits");
    s.ld_teacher = matrix_stride(teacher, "teacher");
    s.ld_ids = matrix_stride(ids, "ids");
    TORCH_CHECK(logits.size(1) > 0 && logits.size(1) < INT32_MAX, "logits have no classes");
    TORCH_CHECK(teacher.size(0) == logits.size(0), "teacher has ", teacher.size(0), " rows, logits ", logits.size(0));
    TORCH_CHECK(ids.sizes() == teacher.sizes(), "ids and teacher must have one shape, have ", ids.sizes(), " and ", teacher.sizes());
    TORCH_CHECK(ids.size(1) < INT32_MAX, "too many kept entries");
    s.rows = logits.size(0);
    s.classes = static_cast<int32_t>(logits.size(1));
    s.kept = static_cast<int32_t>(ids.size(1));
    s.dtype = dtype_of(logits, "logits");
    s.teacher_dtype = dtype_of(teacher, "teacher");
    s.ids64 = is_int64(ids, "ids");
    if (labels.has_value()) {
        check_on(*labels, "labels", dev);
        s.labels64 = is_int64(*labels, "labels");
        TORCH_CHECK(labels->dim() == 1 && labels->size(0) == s.rows && labels->is_contiguous(),
                    "labels must be contiguous [rows], have shape ", labels->sizes());
        c.labels = labels->data_ptr();
    }
    TORCH_CHECK(labels.has_value() || hard == 0.0, "hard needs labels");
    if (reduction == "none") s.reduction = RA_REDUCE_NONE;
    else if (reduction == "mean") s.reduction = RA_REDUCE_MEAN;
    else if (reduction == "sum") s.reduction = RA_REDUCE_SUM;
    else TORCH_CHECK(false, "reduction must be 'none', 'mean' or 'sum', got '", reduction, "'");
    s.temperature = static_cast<float>(temperature);
    s.hard = static_cast<float>(hard);
    return c;
}

int64_t distill_stats_rows(const DistillCall& c) {
    int64_t bytes = 0;
    check(ra_distill_stats_bytes(&c.shape, &bytes), "distill_loss");
    return bytes / 16;
}

// (loss, stats or nothing, gradient or nothing)
std::tuple<Tensor, OptTensor, OptTensor> run_distill(Tensor logits, Tensor teacher, Tensor ids, double temperature,
                                                     OptTensor labels, double hard, std::string reduction, bool with_stats,
                                                     bool with_grad, OptTensor factor) {
    check_no_tracer("distill_loss");
    check_no_tangents({{logits, "logits"}, {teacher, "teacher"}});
    logits = with_rows(logits);
    teacher = with_rows(teacher);
    ids = with_rows(ids);
    if (labels.has_value()) labels = labels->contiguous();
    const DistillCall c = distill_call(logits, teacher, ids, temperature, labels, hard, reduction);
    if (factor.has_value()) factor = factor->reshape({-1});
    const float* const up = factor.has_value() ? f32_vector(*factor, "factor", 1, logits.device()) : nullptr;
    const c10::DeviceGuard guard(logits.device());
    const auto f32 = logits.options().dtype(torch::kFloat32);
    auto loss = c.shape.reduction == RA_REDUCE_NONE ? torch::empty({logits.size(0)}, f32) : torch::empty({}, f32);
    OptTensor stats, grad;
    if (with_stats) stats = torch::empty({distill_stats_rows(c), 4}, f32);
    if (with_grad) grad = torch::empty(logits.sizes(), logits.options());
    int64_t bytes = 0;
    check(ra_distill_workspace(&c.shape, &bytes), "distill_loss");
    auto work = workspace(bytes, logits);
    check(ra_distill_loss(&c.shape, logits.data_ptr(), teacher.data_ptr(), ids.data_ptr(), c.labels, up,
                          loss.data_ptr<float>(), with_stats ? stats->data_ptr<float>() : nullptr,
                          with_grad ? grad->data_ptr() : nullptr, work.data_ptr(), bytes, current_stream()),
          "distill_loss");
    return {loss, stats, grad};
}

Tensor run_distill_backward(Tensor logits, Tensor teacher, Tensor ids, double temperature, OptTensor labels, double hard,
                            std::string reduction, Tensor stats, Tensor grad_loss) {
    const DistillCall c = distill_call(logits, teacher, ids, temperature, labels, hard, reduction);
    check_on(stats, "stats", logits.device());
    TORCH_CHECK(stats.scalar_type() == torch::kFloat32 && stats.is_contiguous() && stats.dim() == 2 &&
                    stats.size(0) == distill_stats_rows(c) && stats.size(1) == 4,
                "stats must be what run_distill returned for these inputs");
    const int64_t n = c.shape.reduction == RA_REDUCE_NONE ? logits.size(0) : 1;
    grad_loss = grad_loss.reshape({-1});  // a copy of it has to live until the launch
    const float* const up = f32_vector(grad_loss, "grad_loss", n, logits.device());
    const c10::DeviceGuard guard(logits.device());
    auto grad = torch::empty(logits.sizes(), logits.options());
    check(ra_distill_backward(&c.shape, logits.data_ptr(), teacher.data_ptr(), ids.data_ptr(), c.labels,
                              stats.data_ptr<float>(), up, grad.data_ptr(), current_stream()),
          "distill_loss backward");
    return grad;
}

// --------------------------------------------------------------------- autograd
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
    if (!torch::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// Gradients that a second differentiation must not pass silently: as Python's
// once_differentiable, they raise where they are differentiated.
variable_list once(variable_list grads, const variable_list& inputs) {
    if (!torch::GradMode::is_enabled()) return grads;
    bool any = false;
    for (const Tensor& t : inputs) any = any || (t.defined() && t.requires_grad());
    if (!any) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int64_t>(grads.size()));
    for (Tensor& t : grads)
        if (t.defined()) t = t.detach().set_requires_grad(true);
    return (*error)(std::move(grads));
}

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor raw(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

struct EmbedNode : torch::autograd::Function<EmbedNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale,
                          c10::optional<int64_t> padding) {
        ctx->save_for_backward({ids});
        ctx->saved_data["rows"] = table.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding;
        return run_embed(ids, table, scale, padding);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor ids = ctx->get_saved_variables()[0];
        Tensor out;
        {
            const torch::NoGradGuard guard;
            const Tensor grad = with_rows(grads[0].reshape({ids.numel(), grads[0].size(-1)}));
            out = run_embed_backward(ids, grad, ctx->saved_data["rows"].toInt(), ctx->saved_data["scale"].toDouble(),
                                     ctx->saved_data["padding"].toOptional<int64_t>());
        }
        return once({Tensor(), out, Tensor(), Tensor()}, {grads[0]});
    }
};

Tensor embed(Tensor ids, Tensor table, double scale, c10::optional<int64_t> padding) {
    check_no_tracer("embed");
    ids = ids.contiguous();
    table = with_rows(table);
    return wants_grad({&table}) ? EmbedNode::apply(ids, table, scale, padding) : run_embed(ids, table, scale, padding);
}

// With a residual two outputs: y and the sum.
struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const OptTensor& weight,
                                 const OptTensor& bias, double eps) {
        auto [y, sum, stats] = run_layer_norm(x, residual, weight, bias, eps, true);
        // Without a residual the input itself is kept, else the sum, which the caller has anyway.
        ctx->save_for_backward({sum.has_value() ? *sum : x, raw(weight), *stats});
        ctx->saved_data["bias"] = bias.has_value();
        ctx->set_materialize_grads(false);
        if (sum.has_value()) return {y, *sum};
        return {y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &weight = saved[1];
        size_t given = 0;  // inputs that are not given are not counted
        const bool x_grad = ctx->needs_input_grad(given++), residual_grad = grads.size() > 1 && ctx->needs_input_grad(given++);
        const bool weight_grad = weight.defined() && ctx->needs_input_grad(given++);
        const bool bias_grad = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(given++);
        Tensor dx, dw, db, of_sum = grads.size() > 1 ? grads[1] : Tensor();
        {
            const torch::NoGradGuard guard;
            if (grads[0].defined()) {
                if (of_sum.defined()) of_sum = of_sum.contiguous();
                auto [x, w, b] = run_layer_norm_backward(h, opt(weight), saved[2], grads[0].contiguous(), opt(of_sum), weight_grad,
                                                         bias_grad);
                dx = x;
                dw = raw(w);
                db = raw(b);
            } else if (of_sum.defined()) {  // only the sum was used
                dx = of_sum;
                if (weight_grad) dw = torch::zeros_like(weight);
                if (bias_grad) db = torch::zeros({h.size(1)}, h.options().dtype(torch::kFloat32));
            }
        }
        return once({x_grad ? dx : Tensor(), residual_grad ? dx : Tensor(), dw, db, Tensor()},
                    {grads[0], grads.size() > 1 ? grads[1] : Tensor(), h, weight});
    }
};

// (y, x + residual or nothing) of matrices.
std::tuple<Tensor, OptTensor> layer_norm(Tensor x, OptTensor residual, OptTensor weight, OptTensor bias, double eps) {
    check_no_tracer("layer_norm");
    x = with_rows(x);
    if (residual.has_value()) residual = with_rows(*residual);
    const Tensor r = raw(residual), w = raw(weight), b = raw(bias);
    check_no_tangents({{x, "x"}, {r, "residual"}, {w, "weight"}, {b, "bias"}});
    if (wants_grad({&x, &r, &w, &b})) {
        const variable_list out = LayerNormNode::apply(x, residual, weight, bias, eps);
        return {out[0], out.size() > 1 ? OptTensor(out[1]) : OptTensor()};
    }
    auto [y, sum, stats] = run_layer_norm(x, residual, weight, bias, eps, false);
    return {y, sum};
}

struct DistillNode : torch::autograd::Function<DistillNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher, const Tensor& ids,
                          const OptTensor& labels, double temperature, double hard, std::string reduction) {
        auto [loss, stats, grad] = run_distill(logits, teacher, ids, temperature, labels, hard, reduction, true, false,
                                               OptTensor());
        ctx->save_for_backward({logits, teacher, ids, raw(labels), *stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["hard"] = hard;
        ctx->saved_data["reduction"] = reduction;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        Tensor out;
        {
            const torch::NoGradGuard guard;
            out = run_distill_backward(saved[0], saved[1], saved[2], ctx->saved_data["temperature"].toDouble(), opt(saved[3]),
                                       ctx->saved_data["hard"].toDouble(), ctx->saved_data["reduction"].toStringRef(), saved[4],
                                       grads[0].contiguous());
        }
        return once({out, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, {grads[0], saved[0]});
    }
};

Tensor distill_loss(Tensor logits, Tensor teacher, Tensor ids, double temperature, OptTensor labels, double hard,
                    std::string reduction) {
    if (!wants_grad({&logits}))
        return std::get<0>(run_distill(logits, teacher, ids, temperature, labels, hard, reduction, false, false, OptTensor()));
    logits = with_rows(logits);  // as they are kept for the backward pass
    teacher = with_rows(teacher);
    ids = with_rows(ids);
    if (labels.has_value()) labels = labels->contiguous();
    return DistillNode::apply(logits, teacher, ids, labels, temperature, hard, reduction);
}

}  // namespace

void bind_model_operators(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("embed", &embed, "scale * table[ids], differentiable in table", py::arg("ids"), py::arg("table"), py::arg("scale"),
          py::arg("padding"));
    m.def("layer_norm", &layer_norm, "Layer norm of a matrix's rows: (y, x + residual), differentiable", py::arg("x"),
          py::arg("residual"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
    m.def("distill_loss", &distill_loss, "Distillation loss, differentiable in logits", py::arg("logits"), py::arg("teacher"),
          py::arg("ids"), py::arg("temperature"), py::arg("labels"), py::arg("hard"), py::arg("reduction"));
    m.def("run_embed", &run_embed, "scale * table[ids]", py::arg("ids"), py::arg("table"), py::arg("scale"),
          py::arg("padding"));
    m.def("run_embed_backward", &run_embed_backward, "Gradient of run_embed's table, [rows, dim]", py::arg("ids"),
          py::arg("grad"), py::arg("rows"), py::arg("scale"), py::arg("padding"));
    m.def("run_layer_norm", &run_layer_norm, "Layer norm of a matrix's rows: (y, x + residual, stats)", py::arg("x"),
          py::arg("residual"), py::arg("weight"), py::arg("bias"), py::arg("eps"), py::arg("with_stats"));
    m.def("run_layer_norm_backward", &run_layer_norm_backward, "(dx, dweight, dbias) of run_layer_norm", py::arg("h"),
          py::arg("weight"), py::arg("stats"), py::arg("grad_y"), py::arg("grad_sum"), py::arg("weight_grad"),
          py::arg("bias_grad"));
    m.def("run_distill", &run_distill, "Distillation loss: (loss, stats, gradient of the logits)", py::arg("logits"),
          py::arg("teacher"), py::arg("ids"), py::arg("temperature"), py::arg("labels"), py::arg("hard"),
          py::arg("reduction"), py::arg("with_stats"), py::arg("with_grad"), py::arg("factor"));
    m.def("run_distill_backward", &run_distill_backward, "Gradient of the logits from run_distill's stats",
          py::arg("logits"), py::arg("teacher"), py::arg("ids"), py::arg("temperature"), py::arg("labels"), py::arg("hard"),
          py::arg("reduction"), py::arg("stats"), py::arg("grad_loss"));
}
