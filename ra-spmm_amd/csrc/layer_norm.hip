// layer_norm.hip — layer norm of every row, of x or of x + residual, and its backward
// pass.
//
//     h = x + residual;  n = (h - mean(h)) r,  r = rsqrt(mean((h - mean(h))^2) + eps)
//     y = n w + b
//     dx = r (w g - mean(w g) - n mean(w g n)) + grad_sum;  dw = sum g n,  db = sum g
//
// A workgroup takes a row; the variance is summed around the mean.  The sums of dw and
// db run over pieces of the rows, which a second launch adds in order.
#include <algorithm>
#include <type_traits>

#include "lanes.hpp"
#include "ra_internal.hpp"
#include "vector_run.hpp"

namespace ra {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 16384;
constexpr int kPieces = 256;       // pieces of the rows in the sums of dw and db
constexpr int64_t kMaxBlocks = 1 << 16;

struct LayerNormArgs {
    const void *x, *res, *gy, *gs;
    void *y, *sum;
    const float *w, *b;
    float* stats;
    float* part;  // [pieces][2][dim]
    int64_t rows, ldx, ldr;
    int32_t dim;
    float eps, count;  // dim as a float
};

template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_forward(const LayerNormArgs a) {
    __shared__ float part[2][kThreads / 64];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
        const T* const r = a.res ? static_cast<const T*>(a.res) + row * a.ldr : nullptr;
        auto value = [&](int d) { return r ? (float)(T)((float)x[d] + (float)r[d]) : (float)x[d]; };
        float s = 0.f;
        for (int d = threadIdx.x; d < a.dim; d += kThreads) s += value(d);
        const float mean = over_workgroup<Add>(s, part[0]) / a.count;
        s = 0.f;
        for (int d = threadIdx.x; d < a.dim; d += kThreads) {
            const float c = value(d) - mean;
            s = fmaf(c, c, s);
        }
        const float inv = rsqrtf(over_workgroup<Add>(s, part[1]) / a.count + a.eps);
        for (int d = threadIdx.x; d < a.dim; d += kThreads) {
            const float h = value(d);
            const float n = (h - mean) * inv;
            static_cast<T*>(a.y)[row * a.dim + d] = (T)fmaf(n, a.w ? a.w[d] : 1.f, a.b ? a.b[d] : 0.f);
            if (r) static_cast<T*>(a.sum)[row * a.dim + d] = (T)h;
        }
        if (a.stats && threadIdx.x == 0) {
            a.stats[2 * row] = mean;
            a.stats[2 * row + 1] = inv;
        }
        __syncthreads();
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_backward(const LayerNormArgs a) {
    __shared__ float part[2][kThreads / 64];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
        const T* const g = static_cast<const T*>(a.gy) + row * a.dim;
        const float mean = a.stats[2 * row], inv = a.stats[2 * row + 1];
        float s = 0.f, t = 0.f;
        for (int d = threadIdx.x; d < a.dim; d += kThreads) {
            const float wg = (a.w ? a.w[d] : 1.f) * (float)g[d], n = ((float)x[d] - mean) * inv;
            s += wg;
            t = fmaf(wg, n, t);
        }
        s = over_workgroup<Add>(s, part[0]) / a.count;
        t = over_workgroup<Add>(t, part[1]) / a.count;
        for (int d = threadIdx.x; d < a.dim; d += kThreads) {
            const float wg = (a.w ? a.w[d] : 1.f) * (float)g[d], n = ((float)x[d] - mean) * inv;
            float dx = inv * (wg - s - n * t);
            if (a.gs) dx += (float)static_cast<const T*>(a.gs)[row * a.dim + d];
            static_cast<T*>(a.y)[row * a.dim + d] = (T)dx;
        }
        __syncthreads();
    }
}

// dw and db over a piece of the rows: a thread per column.
template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_columns(const LayerNormArgs a) {
    const int d = blockIdx.y * kThreads + threadIdx.x;
    const int64_t per = (a.rows + kPieces - 1) / kPieces, first = blockIdx.x * per, end = min(a.rows, first + per);
    if (d >= a.dim) return;
    float dw = 0.f, db = 0.f;
    for (int64_t row = first; row < end; ++row) {
        const float g = (float)static_cast<const T*>(a.gy)[row * a.dim + d];
        const float n = ((float)static_cast<const T*>(a.x)[row * a.ldx + d] - a.stats[2 * row]) * a.stats[2 * row + 1];
        dw = fmaf(g, n, dw);
        db += g;
    }
    float* const to = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    to[d] = dw;
    to[a.dim + d] = db;
}

__global__ __launch_bounds__(kThreads) void layer_norm_weights(const float* __restrict__ part, int pieces, int dim,
                                                               float* dw, float* db) {
    const int d = blockIdx.x * kThreads + threadIdx.x;
    if (d >= 2 * dim) return;
    float s = 0.f;
    for (int p = 0; p < pieces; ++p) s += part[(int64_t)p * 2 * dim + d];
    float* const to = d < dim ? dw : db;
    if (to) to[d < dim ? d : d - dim] = s;
}

ra_status check(const ra_layer_norm_shape* s) {
    if (!s) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: shape is NULL");
    if (s->dtype != RA_DTYPE_F32 && s->dtype != RA_DTYPE_F16 && s->dtype != RA_DTYPE_BF16)
        return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: unknown dtype");
    if (s->rows < 0 || s->dim < 1) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: bad sizes");
    if (s->dim > kMaxDim) return fail(RA_ERR_UNSUPPORTED, "layer norm: dim is at most 16384");
    if (s->rows > INT32_MAX) return fail(RA_ERR_UNSUPPORTED, "layer norm: too many rows (2^31 - 1 at most)");
    if (s->rows > 1 && s->ldx < s->dim) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: rows overlap (ldx is too small)");
    return RA_OK;
}

template <typename F>
void by_type(int32_t dtype, F f) {
    if (dtype == RA_DTYPE_F32) f(float());
    else if (dtype == RA_DTYPE_F16) f(f16_t());
    else f(bf16_t());
}

}  // namespace
}  // namespace ra

using ra::fail;

extern "C" {

ra_status ra_layer_norm(const ra_layer_norm_shape* s, const void* d_x, const void* d_residual, const float* d_weight,
                        const float* d_bias, void* d_y, void* d_sum, float* d_stats, ra_stream_t stream) {
    RA_TRY(ra::check(s));
    if (s->rows == 0) return RA_OK;
    if (!d_x || !d_y) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: NULL tensor");
    if ((d_residual == nullptr) != (d_sum == nullptr))
        return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: a residual and the sum go together");
    if (d_residual && s->rows > 1 && s->ldr < s->dim)
        return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: rows overlap (ldr is too small)");
    ra::LayerNormArgs a{};
    a.x = d_x;
    a.res = d_residual;
    a.w = d_weight;
    a.b = d_bias;
    a.y = d_y;
    a.sum = d_sum;
    a.stats = d_stats;
    a.rows = s->rows;
    a.ldx = s->ldx;
    a.ldr = s->ldr;
    a.dim = s->dim;
    a.eps = s->eps;
    a.count = static_cast<float>(s->dim);
    const int blocks = static_cast<int>(std::min(s->rows, ra::kMaxBlocks));
    ra::by_type(s->dtype, [&](auto t) {
        ra::layer_norm_forward<decltype(t)><<<blocks, ra::kThreads, 0, reinterpret_cast<hipStream_t>(stream)>>>(a);
    });
    RA_LAUNCH_CHECK("layer_norm");
    return RA_OK;
}

ra_status ra_layer_norm_workspace(const ra_layer_norm_shape* s, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: bytes is NULL");
    RA_TRY(ra::check(s));
    *bytes = s->rows == 0 ? 0 : (int64_t)ra::kPieces * 2 * s->dim * (int64_t)sizeof(float);
    return RA_OK;
}

ra_status ra_layer_norm_backward(const ra_layer_norm_shape* s, const void* d_h, const float* d_weight,
                                 const float* d_stats, const void* d_grad_y, const void* d_grad_sum, void* d_dx,
                                 float* d_dweight, float* d_dbias, void* d_workspace, int64_t bytes,
                                 ra_stream_t stream) {
    int64_t need = 0;
    RA_TRY(ra_layer_norm_workspace(s, &need));
    if (!d_dweight && !d_dbias) need = 0;
    if (s->rows > 0 && (!d_h || !d_stats || !d_grad_y || !d_dx))
        return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: NULL tensor");
    if (bytes < need || (need && !d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: the workspace is too small");
    if (need && !ra::aligned16(d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: the workspace must be 16-byte aligned");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    ra::LayerNormArgs a{};
    a.x = d_h;
    a.gy = d_grad_y;
    a.gs = d_grad_sum;
    a.w = d_weight;
    a.y = d_dx;
    a.stats = const_cast<float*>(d_stats);
    a.part = static_cast<float*>(d_workspace);
    a.rows = s->rows;
    a.ldx = s->ldx;
    a.dim = s->dim;
    a.count = static_cast<float>(s->dim);
    const int pieces = s->rows ? ra::kPieces : 0;  // without rows the sums are empty
    if (s->rows) {
        const int blocks = static_cast<int>(std::min(s->rows, ra::kMaxBlocks));
        const dim3 columns(pieces, (s->dim + ra::kThreads - 1) / ra::kThreads);
        ra::by_type(s->dtype, [&](auto t) {
            ra::layer_norm_backward<decltype(t)><<<blocks, ra::kThreads, 0, st>>>(a);
            if (d_dweight || d_dbias) ra::layer_norm_columns<decltype(t)><<<columns, ra::kThreads, 0, st>>>(a);
        });
        RA_LAUNCH_CHECK("layer_norm backward");
    }
    if (d_dweight || d_dbias) {
        ra::layer_norm_weights<<<(2 * s->dim + ra::kThreads - 1) / ra::kThreads, ra::kThreads, 0, st>>>(
            a.part, pieces, s->dim, d_dweight, d_dbias);
        RA_LAUNCH_CHECK("layer_norm_weights");
    }
    return RA_OK;
}

}  // extern "C"
