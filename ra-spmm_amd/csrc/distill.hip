// distill.hip — loss of a student's logits against a teacher's largest ones and a label,
// and its gradient.
//
//     z = s / T;  p = softmax(t / T) over a row's kept entries;  q = softmax(z)
//     kl = sum_e p_e (log p_e - z[id_e] + lse(z));  ce = lse(s) - s[label]
//     loss = (1 - hard) T^2 kl + hard ce
//     d loss / d s_j = (1 - hard) T (q_j - P_j) + hard (softmax(s)_j - [j = label])
//
// with P_j the sum of p_e over the entries of class j.  The label is one more entry: what
// a class's entries take off its gradient is added up by the first of them, which writes
// the class again after the row was written without entries.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "lanes.hpp"
#include "ra_internal.hpp"
#include "vector_run.hpp"

namespace ra {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxKept = 1024;
constexpr int kParts = 1024;  // workgroups' parts of a reduced loss
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
    const void *logits, *teacher, *ids, *labels;
    const float* up;     // what the rows' gradients are multiplied with: one for all, or one each
    int64_t up_step;     // 0 or 1
    float up_scale;      // and this
    float* loss;         // [rows], or NULL
    double* part;        // [workgroups] sums of the rows' losses, or NULL
    float* stats;        // [rows][4]: maximum, sum of exponentials at T and at 1
    const float* kept_stats;
    void* grad;
    int64_t rows, ld, ldt, ldi;
    int32_t classes, kept, teacher_dtype;
    bool ids64, labels64;
    float inv_t;                // 1 / T
    double inv_t64;
    float soft, hard;           // (1 - hard) T^2 and hard
    float soft_grad;            // (1 - hard) T
};

__device__ __forceinline__ float teacher_at(const DistillArgs& a, int64_t at) {
    if (a.teacher_dtype == RA_DTYPE_F32) return static_cast<const float*>(a.teacher)[at];
    if (a.teacher_dtype == RA_DTYPE_F16) return (float)static_cast<const f16_t*>(a.teacher)[at];
    return (float)static_cast<const bf16_t*>(a.teacher)[at];
}
__device__ __forceinline__ int64_t id_at(const DistillArgs& a, int64_t at) {
    return a.ids64 ? static_cast<const int64_t*>(a.ids)[at] : (int64_t)static_cast<const int32_t*>(a.ids)[at];
}
// exp(x / T) for x <= 0 (or -inf), c = log2(e) / T
__device__ __forceinline__ float exp_of(float x, float c) { return __builtin_amdgcn_exp2f(x * c); }

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_rows(const DistillArgs a) {
    extern __shared__ char lds[];
    float* const amount = reinterpret_cast<float*>(lds);                      // [kept + 1]: taken off the gradient
    int32_t* const place = reinterpret_cast<int32_t*>(amount + a.kept + 1);   // its class, -1: none
    __shared__ float part[6][kThreads / 64];
    __shared__ double part64[kThreads / 64];
    const float c = kLog2e * a.inv_t;
    double total = 0.0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* const x = static_cast<const T*>(a.logits) + row * a.ld;
        // The teacher's entries.
        float top = -INFINITY;
        bool outside = false;
        for (int e = threadIdx.x; e < a.kept; e += kThreads) {
            const int64_t id = id_at(a, row * a.ldi + e);
            const float t = teacher_at(a, row * a.ldt + e);
            const bool used = id >= 0 && t != -INFINITY;
            outside |= used && id >= a.classes;
            place[e] = used && id < a.classes ? (int32_t)id : -1;
            amount[e] = t;
            if (used) top = t != t ? INFINITY : fmaxf(top, t);
        }
        top = over_workgroup<Max>(top, part[0]);
        const bool soft = a.soft > 0.f && top != -INFINITY;
        float sum = 0.f;
        for (int e = threadIdx.x; e < a.kept; e += kThreads)
            if (place[e] >= 0) sum += exp_of(amount[e] - top, c);
        sum = over_workgroup<Add>(outside ? NAN : sum, part[1]);
        // The label.
        int64_t label = -1;
        if (a.labels) label = a.labels64 ? static_cast<const int64_t*>(a.labels)[row] : (int64_t)static_cast<const int32_t*>(a.labels)[row];
        const bool hard = a.hard > 0.f && label >= 0;
        // The logits' sums of exponentials.
        float most = -FLT_MAX, at_t = 0.f, at_1 = 0.f;
        if (a.kept_stats) {
            most = a.kept_stats[4 * row];
            at_t = a.kept_stats[4 * row + 1];
            at_1 = a.kept_stats[4 * row + 2];
        } else if (soft || hard) {
            for (int j = threadIdx.x; j < a.classes; j += kThreads) most = fmaxf(most, (float)x[j]);
            most = over_workgroup<Max>(most, part[2]);
            for (int j = threadIdx.x; j < a.classes; j += kThreads) {
                at_t += exp_of((float)x[j] - most, c);
                at_1 += exp_of((float)x[j] - most, kLog2e);
            }
            at_t = over_workgroup<Add>(at_t, part[3]);
            at_1 = over_workgroup<Add>(at_1, part[4]);
        }
        if (a.stats && threadIdx.x == 0) {
            a.stats[4 * row] = most;
            a.stats[4 * row + 1] = at_t;
            a.stats[4 * row + 2] = at_1;
            a.stats[4 * row + 3] = 0.f;
        }
        if (a.loss || a.part) {
            double loss = 0.0;
            if (soft) {
                const double shift = log((double)at_t) - log((double)sum);
                for (int e = threadIdx.x; e < a.kept; e += kThreads) {
                    if (place[e] < 0) continue;
                    const float p = exp_of(amount[e] - top, c) / sum;
                    if (p != 0.f)
                        loss += (double)p * ((((double)amount[e] - top) - ((double)(float)x[place[e]] - most)) * a.inv_t64 + shift);
                }
                loss = sum_workgroup(loss, part64) * a.soft;
                if (sum != sum) loss = NAN;
                __syncthreads();
            }
            if (hard) loss += label < a.classes ? a.hard * (log((double)at_1) - ((double)(float)x[label] - most)) : NAN;
            if (a.loss && threadIdx.x == 0) a.loss[row] = (float)loss;
            total += loss;
        }
        if (a.grad) {
            const float up = (a.up ? a.up[row * a.up_step] : 1.f) * a.up_scale;
            const float soft_up = !soft ? 0.f : sum != sum ? NAN : a.soft_grad * up;
            const float hard_up = !hard ? 0.f : label < a.classes ? a.hard * up : NAN;
            const float ft = soft ? soft_up / at_t : 0.f, f1 = hard ? hard_up / at_1 : 0.f;
            auto without = [&](float s) {
                float g = 0.f;
                if (soft) g = ft * exp_of(s - most, c);
                if (hard) g += f1 * exp_of(s - most, kLog2e);
                return g;
            };
            __syncthreads();  // the loss has been read
            for (int e = threadIdx.x; e <= a.kept; e += kThreads) {
                if (e < a.kept) {
                    amount[e] = soft && place[e] >= 0 ? soft_up * (exp_of(amount[e] - top, c) / sum) : 0.f;
                    if (!soft) place[e] = -1;
                } else {
                    amount[e] = hard_up;
                    place[e] = hard && label < a.classes ? (int32_t)label : -1;
                }
            }
            T* const g = static_cast<T*>(a.grad) + row * a.classes;
            for (int j = threadIdx.x; j < a.classes; j += kThreads) g[j] = (T)without((float)x[j]);
            __threadfence_block();
            __syncthreads();
            for (int e = threadIdx.x; e <= a.kept; e += kThreads) {
                const int32_t j = place[e];
                if (j < 0) continue;
                float off = 0.f;
                bool first = true;
                for (int f = 0; f <= a.kept; ++f) {
                    if (place[f] != j) continue;
                    first &= f >= e;
                    off += amount[f];
                }
                if (first) g[j] = (T)(without((float)x[j]) - off);
            }
        }
        __syncthreads();
    }
    if (a.part && threadIdx.x == 0) a.part[blockIdx.x] = total;
}

// The workgroups' parts in order.
__global__ __launch_bounds__(kThreads) void distill_reduce(const double* __restrict__ part, int parts, double scale, float* loss) {
    __shared__ double sums[kThreads / 64];
    double s = 0.0;
    for (int p = threadIdx.x; p < parts; p += kThreads) s += part[p];
    s = sum_workgroup(s, sums);
    if (threadIdx.x == 0) *loss = (float)(s * scale);
}

// ------------------------------------------------------------ host side
bool known(int32_t dtype) { return dtype == RA_DTYPE_F32 || dtype == RA_DTYPE_F16 || dtype == RA_DTYPE_BF16; }

ra_status check(const ra_distill_shape* s) {
    if (!s) return fail(RA_ERR_INVALID_ARGUMENT, "distill: shape is NULL");
    if (!known(s->dtype) || !known(s->teacher_dtype)) return fail(RA_ERR_INVALID_ARGUMENT, "distill: unknown dtype");
    if (s->rows < 0 || s->classes < 1 || s->kept < 0) return fail(RA_ERR_INVALID_ARGUMENT, "distill: bad sizes");
    if (s->kept > kMaxKept) return fail(RA_ERR_UNSUPPORTED, "distill: at most 1024 kept entries");
    if (s->rows > INT32_MAX || s->classes > (1 << 30)) return fail(RA_ERR_UNSUPPORTED, "distill: too many rows or classes");
    if (s->reduction != RA_REDUCE_NONE && s->reduction != RA_REDUCE_MEAN && s->reduction != RA_REDUCE_SUM)
        return fail(RA_ERR_INVALID_ARGUMENT, "distill: unknown reduction");
    if (!(s->temperature >= 1e-3f && s->temperature <= 1e3f))
        return fail(RA_ERR_INVALID_ARGUMENT, "distill: temperature must be in 1e-3 .. 1e3");
    if (!(s->hard >= 0.f && s->hard <= 1.f)) return fail(RA_ERR_INVALID_ARGUMENT, "distill: hard must be in 0 .. 1");
    if (s->rows > 1 && (s->ld_logits < s->classes || s->ld_teacher < s->kept || s->ld_ids < s->kept))
        return fail(RA_ERR_INVALID_ARGUMENT, "distill: rows overlap (a leading dimension is too small)");
    return RA_OK;
}

ra_status check_tensors(const ra_distill_shape& s, const void* logits, const void* teacher, const void* ids,
                        const void* labels) {
    if (s.hard > 0.f && !labels) return fail(RA_ERR_INVALID_ARGUMENT, "distill: hard needs labels");
    if (s.rows && (!logits || (s.kept && (!teacher || !ids)))) return fail(RA_ERR_INVALID_ARGUMENT, "distill: NULL tensor");
    return RA_OK;
}

DistillArgs args_of(const ra_distill_shape& s, const void* logits, const void* teacher, const void* ids, const void* labels) {
    DistillArgs a{};
    a.logits = logits;
    a.teacher = teacher;
    a.ids = ids;
    a.labels = labels;
    a.up_scale = s.reduction == RA_REDUCE_MEAN && s.rows ? static_cast<float>(1.0 / static_cast<double>(s.rows)) : 1.f;
    a.rows = s.rows;
    a.ld = s.ld_logits;
    a.ldt = s.ld_teacher;
    a.ldi = s.ld_ids;
    a.classes = s.classes;
    a.kept = s.kept;
    a.teacher_dtype = s.teacher_dtype;
    a.ids64 = s.ids64 != 0;
    a.labels64 = s.labels64 != 0;
    a.inv_t64 = 1.0 / s.temperature;
    a.inv_t = static_cast<float>(a.inv_t64);
    a.soft = static_cast<float>((1.0 - s.hard) * s.temperature * s.temperature);
    a.hard = s.hard;
    a.soft_grad = static_cast<float>((1.0 - s.hard) * s.temperature);
    return a;
}

int blocks_of(const ra_distill_shape& s) { return static_cast<int>(std::min<int64_t>(s.rows, kParts)); }

void run(const ra_distill_shape& s, const DistillArgs& a, hipStream_t st) {
    const size_t lds = (size_t)(s.kept + 1) * 8;
    auto go = [&](auto t) { distill_rows<decltype(t)><<<blocks_of(s), kThreads, lds, st>>>(a); };
    if (s.dtype == RA_DTYPE_F32) go(float());
    else if (s.dtype == RA_DTYPE_F16) go(f16_t());
    else go(bf16_t());
}

}  // namespace
}  // namespace ra

using ra::fail;

extern "C" {

ra_status ra_distill_workspace(const ra_distill_shape* s, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "distill: bytes is NULL");
    RA_TRY(ra::check(s));
    *bytes = s->reduction == RA_REDUCE_NONE || s->rows == 0 ? 0 : (int64_t)ra::blocks_of(*s) * (int64_t)sizeof(double);
    return RA_OK;
}

ra_status ra_distill_loss(const ra_distill_shape* s, const void* d_logits, const void* d_teacher, const void* d_ids,
                          const void* d_labels, const float* d_factor, float* d_loss, float* d_stats, void* d_grad,
                          void* d_workspace, int64_t bytes, ra_stream_t stream) {
    int64_t need = 0;
    RA_TRY(ra_distill_workspace(s, &need));
    RA_TRY(ra::check_tensors(*s, d_logits, d_teacher, d_ids, d_labels));
    if (!d_loss && (s->rows || s->reduction != RA_REDUCE_NONE)) return fail(RA_ERR_INVALID_ARGUMENT, "distill: NULL loss");
    if (bytes < need || (need && !d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "distill: the workspace is too small");
    if (need && !ra::aligned16(d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "distill: the workspace must be 16-byte aligned");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    ra::DistillArgs a = ra::args_of(*s, d_logits, d_teacher, d_ids, d_labels);
    a.up = d_factor;
    a.stats = d_stats;
    a.grad = d_grad;
    if (s->reduction == RA_REDUCE_NONE) a.loss = d_loss;
    else a.part = static_cast<double*>(d_workspace);
    if (s->rows) {
        ra::run(*s, a, st);
        RA_LAUNCH_CHECK("distill");
    }
    if (s->reduction != RA_REDUCE_NONE) {  // the mean of no rows is NaN
        const double scale = s->reduction == RA_REDUCE_SUM ? 1.0 : s->rows ? 1.0 / static_cast<double>(s->rows) : NAN;
        ra::distill_reduce<<<1, ra::kThreads, 0, st>>>(a.part, s->rows ? ra::blocks_of(*s) : 0, scale, d_loss);
        RA_LAUNCH_CHECK("distill_reduce");
    }
    return RA_OK;
}

ra_status ra_distill_backward(const ra_distill_shape* s, const void* d_logits, const void* d_teacher, const void* d_ids,
                              const void* d_labels, const float* d_stats, const float* d_grad_loss, void* d_grad,
                              ra_stream_t stream) {
    RA_TRY(ra::check(s));
    RA_TRY(ra::check_tensors(*s, d_logits, d_teacher, d_ids, d_labels));
    if (s->rows == 0) return RA_OK;
    if (!d_stats || !d_grad_loss || !d_grad) return fail(RA_ERR_INVALID_ARGUMENT, "distill: NULL tensor");
    ra::DistillArgs a = ra::args_of(*s, d_logits, d_teacher, d_ids, d_labels);
    a.kept_stats = d_stats;
    a.up = d_grad_loss;
    a.up_step = s->reduction == RA_REDUCE_NONE;
    a.grad = d_grad;
    ra::run(*s, a, reinterpret_cast<hipStream_t>(stream));
    RA_LAUNCH_CHECK("distill backward");
    return RA_OK;
}

}  // extern "C"
