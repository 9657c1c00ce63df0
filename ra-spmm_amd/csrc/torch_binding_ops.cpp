// torch_binding_ops.cpp — torch surface of the operators around the SpMM: graph
// attention, head norms with rotation, 8-bit activations.  Checks, output
// allocation and plan ownership; launches use the current torch stream.
#include <torch/extension.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <memory>
#include <string>
#include <tuple>

#include "../../include/ra_spmm.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

ra_stream_t current_stream() {
    return reinterpret_cast<ra_stream_t>(c10::hip::getCurrentHIPStream().stream());
}

void check(ra_status s, const char* what) {
    TORCH_CHECK(s == RA_OK, what, " failed: ", ra_status_string(s), ": ", ra_last_error());
}

int dtype_of(const Tensor& t, const char* name) {
    if (t.scalar_type() == torch::kFloat32) return RA_DTYPE_F32;
    if (t.scalar_type() == torch::kFloat16) return RA_DTYPE_F16;
    if (t.scalar_type() == torch::kBFloat16) return RA_DTYPE_BF16;
    TORCH_CHECK(false, name, " must be float32, float16 or bfloat16");
    return -1;
}

void check_on(const Tensor& t, const char* name, const torch::Device& dev) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == dev, name, " must be on ", dev, ", is on ", t.device());
}

const float* f32_vector(const Tensor& t, const char* name, int64_t n, const torch::Device& dev) {
    check_on(t, name, dev);
    TORCH_CHECK(t.scalar_type() == torch::kFloat32, name, " must be float32");
    TORCH_CHECK(t.dim() == 1 && t.numel() == n, name, " must have shape [", n, "], has ", t.sizes());
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    return t.data_ptr<float>();
}

// Distance between the rows of t, whose other dimensions have to be contiguous.
int64_t row_stride(const Tensor& t, const char* name) {
    int64_t run = 1;
    for (int64_t d = t.dim() - 1; d > 0; --d) {
        TORCH_CHECK(t.size(d) <= 1 || t.stride(d) == run, name, " must be contiguous within its rows");
        run *= t.size(d);
    }
    if (t.size(0) <= 1) return run;
    TORCH_CHECK(t.stride(0) >= run, name, " must not have rows that overlap");
    return t.stride(0);
}

// ------------------------------------------------------------ graph attention
struct AttentionPlan {
    ra_attn_plan* plan = nullptr;
    ra_attn_info info{};
    Tensor rowptr, colind;  // the plan reads them at every run
    ~AttentionPlan() { ra_attn_plan_destroy(plan); }
};
using AttentionPlanPtr = std::shared_ptr<AttentionPlan>;

void check_lists(const Tensor& rowptr, const Tensor& colind) {
    TORCH_CHECK(rowptr.is_cuda() && colind.is_cuda(), "rowptr and colind must be CUDA tensors");
    TORCH_CHECK(rowptr.device() == colind.device(), "rowptr and colind must be on the same device");
    TORCH_CHECK(rowptr.scalar_type() == torch::kInt32 && colind.scalar_type() == torch::kInt32,
                "rowptr and colind must be int32");
    TORCH_CHECK(rowptr.dim() == 1 && rowptr.numel() >= 1 && rowptr.is_contiguous(),
                "rowptr must be 1-D with M+1 entries and contiguous");
    TORCH_CHECK(colind.dim() == 1 && colind.is_contiguous(), "colind must be 1-D and contiguous");
}

AttentionPlanPtr make_attention_plan(Tensor rowptr, Tensor colind, int64_t M, int64_t K, bool backward) {
    if (!rowptr.is_cuda() && !colind.is_cuda()) {  // a host CSR is uploaded, as the other plan builders do
        const torch::Device dev(torch::kCUDA, c10::hip::current_device());
        rowptr = rowptr.to(dev, torch::kInt32).contiguous();
        colind = colind.to(dev, torch::kInt32).contiguous();
    }
    check_lists(rowptr, colind);
    TORCH_CHECK(M >= 0 && K >= 0 && M < INT32_MAX && K < INT32_MAX, "M and K must be sizes of an int32 CSR");
    TORCH_CHECK(rowptr.numel() == M + 1, "rowptr has ", rowptr.numel(), " entries, M+1 = ", M + 1, " expected");
    const c10::DeviceGuard guard(rowptr.device());
    auto w = std::make_shared<AttentionPlan>();
    w->rowptr = rowptr;
    w->colind = colind;
    check(ra_attn_plan_create(rowptr.data_ptr<int32_t>(), colind.data_ptr<int32_t>(), static_cast<int32_t>(M),
                              static_cast<int32_t>(K), colind.numel(), backward, current_stream(), &w->plan),
          "make_attention_plan");
    check(ra_attn_plan_get_info(w->plan, &w->info), "attention plan info");
    return w;
}

// The lists may have been allocated on another stream than the one that reads them.
void use_on_current_stream(const AttentionPlan& w) {
    const auto st = c10::hip::getCurrentHIPStream(w.rowptr.device().index());
    c10::hip::HIPCachingAllocator::recordStream(w.rowptr.storage().data_ptr(), st);
    if (w.colind.numel()) c10::hip::HIPCachingAllocator::recordStream(w.colind.storage().data_ptr(), st);
}

struct AttentionCall {
    ra_attn_shape shape{};
    const float* lam = nullptr;
    const float* bias = nullptr;
};

AttentionCall attention_call(int64_t M, int64_t K, int64_t nnz, const torch::Device& dev, const Tensor& q,
                             const Tensor& k, const Tensor& v, const Tensor& lam, c10::optional<double> scale,
                             const OptTensor& bias) {
    check_on(q, "q", dev);
    check_on(k, "k", dev);
    check_on(v, "v", dev);
    TORCH_CHECK(q.dim() == 4 && q.size(2) == 2, "q must have shape [M, heads, 2, head_dim], has ", q.sizes());
    TORCH_CHECK(k.dim() == 4 && k.size(2) == 2, "k must have shape [K, kv_heads, 2, head_dim], has ", k.sizes());
    TORCH_CHECK(v.dim() == 3, "v must have shape [K, kv_heads, value_dim], has ", v.sizes());
    TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "q, k and v must have one dtype");
    TORCH_CHECK(q.size(0) == M, "q has ", q.size(0), " rows, the lists ", M);
    TORCH_CHECK(k.size(0) == K && v.size(0) == K, "k and v must have K = ", K, " rows, have ", k.size(0), " and ", v.size(0));
    TORCH_CHECK(k.size(3) == q.size(3), "q and k must have one head_dim");
    TORCH_CHECK(v.size(1) == k.size(1), "k and v must have the same heads");
    TORCH_CHECK(q.size(1) > 0 && k.size(1) > 0 && q.size(1) % k.size(1) == 0,
                "q's heads must be a positive multiple of k's");
    TORCH_CHECK(q.size(3) > 0 && v.size(2) > 0, "empty heads");
    AttentionCall c;
    c.shape.q_heads = static_cast<int32_t>(q.size(1));
    c.shape.kv_heads = static_cast<int32_t>(k.size(1));
    c.shape.head_dim = static_cast<int32_t>(q.size(3));
    c.shape.value_dim = static_cast<int32_t>(v.size(2));
    c.shape.dtype = dtype_of(q, "q, k and v");
    c.shape.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(3))));
    c.shape.ldq = row_stride(q, "q");
    c.shape.ldk = row_stride(k, "k");
    c.shape.ldv = row_stride(v, "v");
    c.lam = f32_vector(lam, "lam", q.size(1), dev);
    if (bias.has_value()) c.bias = f32_vector(*bias, "bias", nnz, dev);
    return c;
}

std::tuple<Tensor, Tensor> run_attention(const AttentionPlanPtr& w, const Tensor& q, const Tensor& k, const Tensor& v,
                                         const Tensor& lam, c10::optional<double> scale, const OptTensor& bias,
                                         bool with_stats) {
    TORCH_CHECK(w && w->plan, "Invalid attention plan");
    const auto dev = w->rowptr.device();
    const AttentionCall c = attention_call(w->info.M, w->info.K, w->info.nnz, dev, q, k, v, lam, scale, bias);
    const c10::DeviceGuard guard(dev);
    use_on_current_stream(*w);
    auto out = torch::empty({q.size(0), q.size(1), v.size(2)}, q.options());
    Tensor stats;
    if (with_stats) stats = torch::empty({q.size(0), q.size(1), 2, 2}, q.options().dtype(torch::kFloat32));
    check(ra_attn_plan_run(w->plan, &c.shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), c.lam, c.bias, out.data_ptr(),
                           with_stats ? stats.data_ptr<float>() : nullptr, current_stream()),
          "run_attention_plan");
    return {out, stats};
}

Tensor run_attention_plan(AttentionPlanPtr w, Tensor q, Tensor k, Tensor v, Tensor lam, c10::optional<double> scale,
                          OptTensor bias) {
    return std::get<0>(run_attention(w, q, k, v, lam, scale, bias, false));
}

std::tuple<Tensor, Tensor> run_attention_plan_train(AttentionPlanPtr w, Tensor q, Tensor k, Tensor v, Tensor lam,
                                                    c10::optional<double> scale, OptTensor bias) {
    return run_attention(w, q, k, v, lam, scale, bias, true);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> run_attention_plan_backward(AttentionPlanPtr w, Tensor q, Tensor k, Tensor v,
                                                                       Tensor lam, Tensor stats, Tensor grad_out,
                                                                       c10::optional<double> scale, OptTensor bias) {
    TORCH_CHECK(w && w->plan, "Invalid attention plan");
    TORCH_CHECK(w->info.backward, "the attention plan was made with backward=False");
    const auto dev = w->rowptr.device();
    const AttentionCall c = attention_call(w->info.M, w->info.K, w->info.nnz, dev, q, k, v, lam, scale, bias);
    check_on(stats, "stats", dev);
    check_on(grad_out, "grad_out", dev);
    TORCH_CHECK(stats.scalar_type() == torch::kFloat32 && stats.is_contiguous() && stats.dim() == 4 &&
                    stats.size(0) == q.size(0) && stats.size(1) == q.size(1) && stats.size(2) == 2 && stats.size(3) == 2,
                "stats must be what run_attention_plan_train returned for these inputs");
    TORCH_CHECK(grad_out.scalar_type() == q.scalar_type() && grad_out.is_contiguous() && grad_out.dim() == 3 &&
                    grad_out.size(0) == q.size(0) && grad_out.size(1) == q.size(1) && grad_out.size(2) == v.size(2),
                "grad_out must be contiguous, of q's dtype and of the output's shape");
    const c10::DeviceGuard guard(dev);
    use_on_current_stream(*w);
    auto dq = torch::empty(q.sizes(), q.options());
    auto dk = torch::empty(k.sizes(), k.options());
    auto dv = torch::empty(v.sizes(), v.options());
    auto dlam = torch::empty(lam.sizes(), lam.options());
    check(ra_attn_plan_run_backward(w->plan, &c.shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), c.lam, c.bias,
                                    stats.data_ptr<float>(), grad_out.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                                    dv.data_ptr(), dlam.data_ptr<float>(), current_stream()),
          "run_attention_plan_backward");
    return {dq, dk, dv, dlam};
}

Tensor diff_attention_csr(Tensor rowptr, Tensor colind, Tensor q, Tensor k, Tensor v, Tensor lam,
                          c10::optional<double> scale, OptTensor bias) {
    check_lists(rowptr, colind);
    const auto dev = rowptr.device();
    const int64_t M = rowptr.numel() - 1, nnz = colind.numel(), K = k.size(0);
    TORCH_CHECK(M < INT32_MAX && K < INT32_MAX && nnz <= INT32_MAX, "an int32 CSR holds at most 2^31 - 1 rows and edges");
    const AttentionCall c = attention_call(M, K, nnz, dev, q, k, v, lam, scale, bias);
    const c10::DeviceGuard guard(dev);
    auto out = torch::empty({q.size(0), q.size(1), v.size(2)}, q.options());
    int64_t bytes = 0;
    check(ra_attn_csr_workspace(&c.shape, static_cast<int32_t>(M), nnz, &bytes), "diff_attention_csr");
    auto work = torch::empty({bytes}, q.options().dtype(torch::kUInt8));
    check(ra_attn_csr(rowptr.data_ptr<int32_t>(), colind.data_ptr<int32_t>(), static_cast<int32_t>(M),
                      static_cast<int32_t>(K), nnz, &c.shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), c.lam, c.bias,
                      out.data_ptr(), work.data_ptr(), bytes, current_stream()),
          "diff_attention_csr");
    return out;
}

// ------------------------------------------------- head norms and rotation
// q and k: [rows, ..., head_dim]; the dimensions between are heads.
struct NormCall {
    ra_norm_shape shape{};
    const float *wq = nullptr, *wk = nullptr, *table = nullptr;
    const int32_t* positions = nullptr;
};

int64_t heads_of(const Tensor& t, const char* name) {
    TORCH_CHECK(t.dim() >= 2 && t.size(-1) > 0, name, " must have shape [rows, heads.., head_dim], has ", t.sizes());
    int64_t n = 1;
    for (int64_t d = 1; d + 1 < t.dim(); ++d) n *= t.size(d);
    TORCH_CHECK(n > 0, name, " has no heads");
    return n;
}

NormCall norm_call(const Tensor& q, const OptTensor& k, const Tensor& wq, const OptTensor& wk, const OptTensor& table,
                   const OptTensor& positions, double eps, const std::string& layout) {
    TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
    const auto dev = q.device();
    NormCall c;
    ra_norm_shape& s = c.shape;
    const int64_t hq = heads_of(q, "q"), hk = k.has_value() ? heads_of(*k, "k") : 0, D = q.size(-1);
    TORCH_CHECK(q.size(0) < INT32_MAX && hq < INT32_MAX && hk < INT32_MAX && D < INT32_MAX, "q or k is too large");
    s.rows = static_cast<int32_t>(q.size(0));
    s.q_heads = static_cast<int32_t>(hq);
    s.k_heads = static_cast<int32_t>(hk);
    s.head_dim = static_cast<int32_t>(D);
    s.dtype = dtype_of(q, "q and k");
    s.eps = static_cast<float>(eps);
    s.ldq = row_stride(q, "q");
    c.wq = f32_vector(wq, "wq", D, dev);
    TORCH_CHECK(k.has_value() == wk.has_value(), "k and wk go together");
    if (k.has_value()) {
        check_on(*k, "k", dev);
        TORCH_CHECK(k->scalar_type() == q.scalar_type(), "q and k must have one dtype");
        TORCH_CHECK(k->size(0) == q.size(0) && k->size(-1) == D, "q and k must have the same rows and head_dim");
        s.ldk = row_stride(*k, "k");
        c.wk = f32_vector(*wk, "wk", D, dev);
    }
    if (layout == "half") s.layout = RA_ROTATION_HALF;
    else if (layout == "interleaved") s.layout = RA_ROTATION_INTERLEAVED;
    else TORCH_CHECK(false, "layout must be 'half' or 'interleaved', got '", layout, "'");
    if (table.has_value()) {
        check_on(*table, "table", dev);
        TORCH_CHECK(table->scalar_type() == torch::kFloat32 && table->is_contiguous() && table->dim() == 3 && table->size(2) == 2,
                    "table must be contiguous float32 [positions, rot_dim / 2, 2], has ", table->sizes());
        TORCH_CHECK(2 * table->size(1) <= D, "the table's rot_dim ", 2 * table->size(1), " passes head_dim ", D);
        TORCH_CHECK(table->size(0) < INT32_MAX, "the table is too long");
        s.positions = static_cast<int32_t>(table->size(0));
        s.rot_dim = static_cast<int32_t>(2 * table->size(1));
        c.table = table->data_ptr<float>();
    }
    if (positions.has_value()) {
        check_on(*positions, "positions", dev);
        TORCH_CHECK(table.has_value(), "positions need a table");
        TORCH_CHECK(positions->scalar_type() == torch::kInt32 && positions->is_contiguous() && positions->dim() == 1 &&
                        positions->numel() == q.size(0),
                    "positions must be contiguous int32 [rows]");
        c.positions = positions->data_ptr<int32_t>();
    }
    return c;
}

std::tuple<Tensor, OptTensor> run_head_norm(Tensor q, OptTensor k, Tensor wq, OptTensor wk, OptTensor table,
                                            OptTensor positions, double eps, std::string layout) {
    const NormCall c = norm_call(q, k, wq, wk, table, positions, eps, layout);
    const c10::DeviceGuard guard(q.device());
    auto yq = torch::empty(q.sizes(), q.options());
    OptTensor yk;
    if (k.has_value()) yk = torch::empty(k->sizes(), k->options());
    check(ra_head_norm(&c.shape, q.data_ptr(), k.has_value() ? k->data_ptr() : nullptr, c.wq, c.wk, c.table, c.positions,
                       yq.data_ptr(), yk.has_value() ? yk->data_ptr() : nullptr, current_stream()),
          "head_norm_rotate");
    return {yq, yk};
}

std::tuple<Tensor, OptTensor, Tensor, OptTensor> run_head_norm_backward(Tensor q, OptTensor k, Tensor wq, OptTensor wk,
                                                                        OptTensor table, OptTensor positions, double eps,
                                                                        std::string layout, Tensor gq, OptTensor gk) {
    const NormCall c = norm_call(q, k, wq, wk, table, positions, eps, layout);
    auto check_grad = [&](const Tensor& g, const Tensor& x, const char* name) {
        check_on(g, name, q.device());
        TORCH_CHECK(g.scalar_type() == x.scalar_type() && g.is_contiguous() && g.sizes() == x.sizes(), name,
                    " must be contiguous, of the output's shape and dtype");
    };
    check_grad(gq, q, "grad_q");
    TORCH_CHECK(k.has_value() == gk.has_value(), "k and grad_k go together");
    if (k.has_value()) check_grad(*gk, *k, "grad_k");
    const c10::DeviceGuard guard(q.device());
    auto dq = torch::empty(q.sizes(), q.options());
    auto dwq = torch::empty(wq.sizes(), wq.options());
    OptTensor dk, dwk;
    if (k.has_value()) {
        dk = torch::empty(k->sizes(), k->options());
        dwk = torch::empty(wk->sizes(), wk->options());
    }
    int64_t bytes = 0;
    check(ra_head_norm_workspace(&c.shape, &bytes), "head_norm_rotate backward");
    auto work = torch::empty({bytes}, q.options().dtype(torch::kUInt8));
    check(ra_head_norm_backward(&c.shape, q.data_ptr(), k.has_value() ? k->data_ptr() : nullptr, c.wq, c.wk, c.table,
                                c.positions, gq.data_ptr(), gk.has_value() ? gk->data_ptr() : nullptr, dq.data_ptr(),
                                dk.has_value() ? dk->data_ptr() : nullptr, dwq.data_ptr<float>(),
                                dwk.has_value() ? dwk->data_ptr<float>() : nullptr, work.data_ptr(), bytes, current_stream()),
          "head_norm_rotate backward");
    return {dq, dk, dwq, dwk};
}

// ------------------------------------------------- activations kept in 8 bits
int64_t packed_width(int64_t cols) { return (cols + 31) / 32 * 32; }

Tensor empty_scales(const Tensor& x) {
    return torch::empty({packed_width(x.size(1)) / 32, (x.size(0) + 7) / 8 * 8}, x.options().dtype(torch::kUInt8));
}

int64_t check_matrix(const Tensor& x, const char* name) {
    TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(x.dim() == 2 && x.size(1) > 0 && x.size(1) < INT32_MAX - 64, name, " must be [rows, cols], has ", x.sizes());
    dtype_of(x, name);
    return row_stride(x, name);
}

void check_packed(const Tensor& codes, const Tensor& scales, int64_t cols) {
    TORCH_CHECK(codes.is_cuda() && scales.is_cuda() && codes.device() == scales.device(),
                "codes and scales must be CUDA tensors on the same device");
    TORCH_CHECK(codes.scalar_type() == torch::kUInt8 && codes.is_contiguous() && codes.dim() == 2 && cols > 0 &&
                    codes.size(1) == packed_width(cols),
                "codes must be contiguous uint8 [rows, cols rounded up to 32]");
    TORCH_CHECK(scales.scalar_type() == torch::kUInt8 && scales.is_contiguous() && scales.dim() == 2 &&
                    scales.size(0) == codes.size(1) / 32 && scales.size(1) == (codes.size(0) + 7) / 8 * 8,
                "scales must be contiguous uint8 [groups, rows rounded up to 8]");
}

std::tuple<Tensor, Tensor> pack8(Tensor x) {
    const int64_t ld = check_matrix(x, "x");
    const c10::DeviceGuard guard(x.device());
    const auto bytes = x.options().dtype(torch::kUInt8);
    auto codes = torch::empty({x.size(0), packed_width(x.size(1))}, bytes);
    auto scales = empty_scales(x);
    check(ra_pack8(x.data_ptr(), x.size(0), static_cast<int32_t>(x.size(1)), ld, dtype_of(x, "x"),
                   codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), current_stream()),
          "pack8");
    return {codes, scales};
}

std::tuple<Tensor, Tensor, Tensor> relu_pack8(Tensor x) {
    const int64_t ld = check_matrix(x, "x");
    const c10::DeviceGuard guard(x.device());
    const auto bytes = x.options().dtype(torch::kUInt8);
    auto y = torch::empty(x.sizes(), x.options());
    auto codes = torch::empty({x.size(0), packed_width(x.size(1))}, bytes);
    auto scales = empty_scales(x);
    check(ra_relu_pack8(x.data_ptr(), x.size(0), static_cast<int32_t>(x.size(1)), ld, dtype_of(x, "x"), y.data_ptr(),
                        codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), current_stream()),
          "relu_pack8");
    return {y, codes, scales};
}

Tensor unpack8(Tensor codes, Tensor scales, int64_t cols, bool is_signed, torch::ScalarType dtype) {
    check_packed(codes, scales, cols);
    TORCH_CHECK(dtype == torch::kFloat32 || dtype == torch::kFloat16 || dtype == torch::kBFloat16,
                "dtype must be float32, float16 or bfloat16");
    const c10::DeviceGuard guard(codes.device());
    auto out = torch::empty({codes.size(0), cols}, codes.options().dtype(dtype));
    check(ra_unpack8(codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), codes.size(0), static_cast<int32_t>(cols),
                     is_signed, dtype_of(out, "dtype"), out.data_ptr(), current_stream()),
          "unpack8");
    return out;
}

Tensor relu_grad8(Tensor grad, Tensor codes, Tensor scales, int64_t cols) {
    check_packed(codes, scales, cols);
    check_on(grad, "grad", codes.device());
    const int64_t ld = check_matrix(grad, "grad");
    TORCH_CHECK(grad.size(0) == codes.size(0) && grad.size(1) == cols, "grad must have the packed shape [", codes.size(0),
                ", ", cols, "], has ", grad.sizes());
    const c10::DeviceGuard guard(codes.device());
    auto out = torch::empty(grad.sizes(), grad.options());
    check(ra_relu_grad8(grad.data_ptr(), codes.data_ptr<uint8_t>(), grad.size(0), static_cast<int32_t>(cols), ld,
                        dtype_of(grad, "grad"), out.data_ptr(), current_stream()),
          "relu_grad8");
    return out;
}

Tensor weight_grad8(Tensor grad, Tensor codes, Tensor scales, int64_t cols, bool is_signed) {
    check_packed(codes, scales, cols);
    check_on(grad, "grad", codes.device());
    const int64_t ld = check_matrix(grad, "grad");
    TORCH_CHECK(grad.size(0) == codes.size(0), "grad has ", grad.size(0), " rows, the packed activation ", codes.size(0));
    const c10::DeviceGuard guard(codes.device());
    const auto O = static_cast<int32_t>(grad.size(1)), C = static_cast<int32_t>(cols);
    auto out = torch::empty({grad.size(1), cols}, grad.options().dtype(torch::kFloat32));
    int64_t bytes = 0;
    check(ra_weight_grad8_workspace(grad.size(0), O, C, &bytes), "weight_grad8");
    auto work = torch::empty({bytes}, codes.options());
    check(ra_weight_grad8(grad.data_ptr(), codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), grad.size(0), O, C, ld,
                          is_signed, dtype_of(grad, "grad"), out.data_ptr<float>(), work.data_ptr(), bytes, current_stream()),
          "weight_grad8");
    return out;
}

}  // namespace

void bind_operators(pybind11::module_& m) {
    namespace py = pybind11;
    py::class_<AttentionPlan, AttentionPlanPtr>(m, "RAAttentionPlan")
        .def_property_readonly("M", [](const AttentionPlan& w) { return w.info.M; })
        .def_property_readonly("K", [](const AttentionPlan& w) { return w.info.K; })
        .def_property_readonly("nnz", [](const AttentionPlan& w) { return w.info.nnz; })
        .def_property_readonly("backward", [](const AttentionPlan& w) { return w.info.backward != 0; })
        .def_property_readonly("num_items", [](const AttentionPlan& w) { return w.info.num_items; })
        .def_property_readonly("num_splits", [](const AttentionPlan& w) { return w.info.num_splits; })
        .def_property_readonly("num_items_t", [](const AttentionPlan& w) { return w.info.num_items_t; })
        .def_property_readonly("num_splits_t", [](const AttentionPlan& w) { return w.info.num_splits_t; })
        .def_property_readonly("plan_bytes", [](const AttentionPlan& w) { return w.info.plan_bytes; });
    m.def("make_attention_plan", &make_attention_plan,
          "Plan of differential attention over a graph's neighbour lists (built on the GPU; refers to rowptr and colind)",
          py::arg("rowptr"), py::arg("colind"), py::arg("M"), py::arg("K"), py::arg("backward") = true);
    m.def("run_attention_plan", &run_attention_plan, "Differential attention, inference (the result records no gradient)", py::arg("plan"), py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("lam"), py::arg("scale") = py::none(), py::arg("bias") = py::none());
    m.def("run_attention_plan_train", &run_attention_plan_train,
          "Differential attention: (out, stats), stats for run_attention_plan_backward", py::arg("plan"), py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("lam"), py::arg("scale") = py::none(), py::arg("bias") = py::none());
    m.def("run_attention_plan_backward", &run_attention_plan_backward, "(dq, dk, dv, dlam) of run_attention_plan_train",
          py::arg("plan"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("lam"), py::arg("stats"),
          py::arg("grad_out"), py::arg("scale") = py::none(), py::arg("bias") = py::none());
    m.def("diff_attention_csr", &diff_attention_csr,
          "Differential attention over lists that arrive with the call (no plan; rowptr and colind are not checked; the "
          "result records no gradient, unlike diff_attention's)",
          py::arg("rowptr"), py::arg("colind"), py::arg("q"), py::arg("k"), py::arg("v"), py::arg("lam"),
          py::arg("scale") = py::none(), py::arg("bias") = py::none());
    m.def("export_attention_plan",
          [](AttentionPlanPtr w, std::string name) {
              TORCH_CHECK(w && w->plan, "Invalid attention plan");
              int64_t n = 0;
              check(ra_attn_plan_export(w->plan, name.c_str(), nullptr, &n), "export_attention_plan");
              auto t = torch::empty({n}, torch::TensorOptions().dtype(torch::kInt32));
              check(ra_attn_plan_export(w->plan, name.c_str(), t.data_ptr<int32_t>(), &n), "export_attention_plan");
              return t;
          },
          "Copy a plan array to the host (items, splits, rowptr_t, row_t, edge_t, items_t, splits_t)", py::arg("plan"),
          py::arg("name"));

    m.def("run_head_norm", &run_head_norm, "RMS norm of every head and rotation: (q, k)", py::arg("q"), py::arg("k"),
          py::arg("wq"), py::arg("wk"), py::arg("table"), py::arg("positions"), py::arg("eps"), py::arg("layout"));
    m.def("run_head_norm_backward", &run_head_norm_backward, "(dq, dk, dwq, dwk) of run_head_norm", py::arg("q"),
          py::arg("k"), py::arg("wq"), py::arg("wk"), py::arg("table"), py::arg("positions"), py::arg("eps"),
          py::arg("layout"), py::arg("grad_q"), py::arg("grad_k"));

    m.def("pack8", &pack8, "(codes, scales) of a matrix in 8 bits", py::arg("x"));
    m.def("relu_pack8", &relu_pack8, "(relu(x), codes, scales)", py::arg("x"));
    m.def("unpack8",
          [](Tensor codes, Tensor scales, int64_t cols, bool is_signed, py::object dtype) {
              return unpack8(codes, scales, cols, is_signed, torch::python::detail::py_object_to_dtype(dtype));
          },
          "code * scale", py::arg("codes"), py::arg("scales"), py::arg("cols"), py::arg("signed"), py::arg("dtype"));
    m.def("relu_grad8", &relu_grad8, "grad where the unsigned code is positive", py::arg("grad"), py::arg("codes"),
          py::arg("scales"), py::arg("cols"));
    m.def("weight_grad8", &weight_grad8, "grad^T (code * scale), float32", py::arg("grad"), py::arg("codes"),
          py::arg("scales"), py::arg("cols"), py::arg("signed"));
}
