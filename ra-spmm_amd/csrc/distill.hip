// distill.hip — loss of a student's logits against a teacher's largest ones and a label,
// and its gradient.
//
//     z = s / T;  p = softmax(t / T) over a row's kept entries;  q = softmax(z)
//     kl = sum_e p_e (log p_e - z[id_e] + lse(z));  ce = lse(s) - s[label]
//     loss = (1 - hard) T^2 kl + hard ce
//     d loss / d s_j = (1 - hard) T (q_j - P_j) + hard (softmax(s)_j - [j = label])
//
// with P_j the sum of p_e over the entries of class j.  The label is one more entry: what a
// class's entries take off its gradient is added up by the first of them, which writes the class
// again after the row was written without entries.
//
// Bound by memory where rows are long (logits read, gradient written), by the vector unit and the
// loads' latency where they are short: an exponential is 4 operations' time, and the logarithms,
// divisions and entries come once a row.  So a row is held by as few lanes as the machine stays full
// with: a lane (up to 64 classes, 32,768 rows and more), a part of a wave (up to 1,024 classes), a
// wave, a workgroup, or, few rows of many classes, several workgroups.  The first two take the rows
// through LDS as one run of memory; the others read a row twice, once for its maximum and sums of
// exponentials together (scaled down where the maximum grows), once for the gradient, out of the
// caches.
//
// Measured: 2,048 x 100,003 in bf16, loss and gradient in one call, 208 us (0.82 GB, 3.9 TB/s; 126 us of it
// is the vector unit's time); 50,000 x 2,000 122 us (3.3 TB/s), 1e6 x 100 188 (2.1); 1e6 x 47 in fp32, loss
// and gradient 93 us each (44 us of it the vector unit's); 16 x 50,000 in fp16 5 us for the pieces, 9 for
// the loss and 9 for the gradient.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "lanes.hpp"
#include "overlap.hpp"
#include "ra_internal.hpp"
#include "vector_run.hpp"

namespace ra {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxKept = 1024;
constexpr int kMaxBlocks = 16384;      // workgroups, and so parts of a reduced loss
// Rows of up to 64 classes and 16 entries go by lanes from 32,768 rows on: of 47 classes in fp32,
// loss and gradient in one call, 16,384 rows take 14.3 us (by parts of waves 11.1), 32,768 15.1
// (14.9), 65,536 17.4 (23.4), 262,144 39 (60).
constexpr int kLaneClasses = 64;
constexpr int kLaneKept = 16;
constexpr int64_t kLaneRows = 32768;
constexpr int kMaxShort = 1024;        // classes of a row that a wave holds
constexpr int kStageBytes = 16384;     // rows of a workgroup at once, about
// A gradient past the last-level cache (256 MB) is written around the caches, which hold the row
// that is read again: 224 us, 211 (2,048 x 100,003 bf16).
constexpr int64_t kAroundBytes = int64_t(256) << 20;
constexpr int kAhead = 4;  // packets of a lane at once
constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
    const void *logits, *teacher, *ids, *labels;
    const float* up;     // what the rows' gradients are multiplied with: one for all, or one each
    int64_t up_step;     // 0 or 1
    float up_scale;      // and this
    float* loss;         // [rows], or NULL
    double* part;        // [workgroups] sums of the rows' losses, or NULL
    float* stats;        // of long rows, [rows][4]: maximum, sum of exponentials at T and at 1
    const float* kept_stats;
    float* piece_stats;  // [rows][pieces][4], where a row is cut
    void* grad;
    int64_t rows, ld, ldt, ldi;
    int32_t classes, kept, teacher_dtype;
    bool ids64, labels64;
    float inv_t;                // 1 / T
    float soft, hard;           // (1 - hard) T^2 and hard
    float soft_grad;            // (1 - hard) T
    int32_t stage_rows, lanes_shift;   // short rows: rows of a workgroup at once, lanes of a row
    bool whole;                 // rows lie one after the other on 16-byte addresses, the gradient's too
    int32_t pieces, piece;      // long rows: pieces of a row, classes of one
};

__device__ __forceinline__ float teacher_at(const DistillArgs& a, int64_t at) {
    if (a.teacher_dtype == RA_DTYPE_F32) return static_cast<const float*>(a.teacher)[at];
    if (a.teacher_dtype == RA_DTYPE_F16) return (float)static_cast<const f16_t*>(a.teacher)[at];
    return (float)static_cast<const bf16_t*>(a.teacher)[at];
}
__device__ __forceinline__ int64_t id_at(const DistillArgs& a, int64_t at) {
    return a.ids64 ? static_cast<const int64_t*>(a.ids)[at] : (int64_t)static_cast<const int32_t*>(a.ids)[at];
}
__device__ __forceinline__ int64_t label_at(const DistillArgs& a, int64_t row) {  // -1: none
    if (!a.labels) return -1;
    return a.labels64 ? static_cast<const int64_t*>(a.labels)[row] : (int64_t)static_cast<const int32_t*>(a.labels)[row];
}
// exp(x / T) for x <= 0 (or -inf), c = log2(e) / T
__device__ __forceinline__ float exp_of(float x, float c) { return __builtin_amdgcn_exp2f(x * c); }

// The lanes that share a row: a part of a wave, or the workgroup, whose waves exchange
// through LDS.
struct WaveTeam {
    int lane, lanes;
    template <typename Op>
    __device__ __forceinline__ float all(float x) { return over_lanes<Op>(x, lanes); }
    __device__ __forceinline__ float sum(float x) { return all<Add>(x); }
    __device__ __forceinline__ void sync() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }
};
struct WorkgroupTeam {
    int lane, lanes;
    float* lds;  // [2][16], in turn
    int turn = 0;
    template <typename Op>
    __device__ __forceinline__ float all(float x) {
        turn ^= 1;
        return over_workgroup<Op>(x, lds + 16 * turn);
    }
    __device__ __forceinline__ float sum(float x) { return all<Add>(x); }
    __device__ __forceinline__ void sync() { __syncthreads(); }
};

// A row's teacher entries and label: place[e] is the entry's class (-1: takes no part),
// amount[e] its logit; entry `kept` is the label.
struct Targets {
    float* amount;
    int32_t* place;
    float top, sum;
    int64_t label;
    bool soft, hard;
};

template <typename Team>
__device__ __forceinline__ void read_targets(const DistillArgs& a, int64_t row, Team& team, Targets& t) {
    float top = -INFINITY;
    bool outside = false;
    for (int e = team.lane; e < a.kept; e += team.lanes) {
        const int64_t id = id_at(a, row * a.ldi + e);
        const float x = teacher_at(a, row * a.ldt + e);
        const bool used = id >= 0 && x != -INFINITY;
        outside |= used && id >= a.classes;
        t.place[e] = used && id < a.classes ? (int32_t)id : -1;
        t.amount[e] = x;
        if (used) top = x != x ? INFINITY : fmaxf(top, x);
    }
    t.top = team.template all<Max>(top);
    t.soft = a.soft > 0.f && t.top != -INFINITY;
    float sum = 0.f;
    for (int e = team.lane; e < a.kept; e += team.lanes)
        if (t.place[e] >= 0) sum += exp_of(t.amount[e] - t.top, kLog2e * a.inv_t);
    t.sum = team.sum(outside ? NAN : sum);
    t.label = label_at(a, row);
    t.hard = a.hard > 0.f && t.label >= 0;
}

// The row's loss from its maximum and sums of exponentials; x(j): the logit of class j.
template <typename Team, typename X>
__device__ __forceinline__ float row_loss(const DistillArgs& a, Team& team, const Targets& t, float most, float at_t, float at_1, X x) {
    const float shift = logf(at_t) - logf(t.sum);
    float loss = 0.f;
    for (int e = team.lane; e < a.kept; e += team.lanes) {
        if (!t.soft || t.place[e] < 0) continue;
        const float p = exp_of(t.amount[e] - t.top, kLog2e * a.inv_t) / t.sum;
        if (p != 0.f) loss = fmaf(p, fmaf((t.amount[e] - t.top) - (x(t.place[e]) - most), a.inv_t, shift), loss);
    }
    loss = team.sum(loss) * a.soft;
    if (!t.soft) loss = 0.f;
    else if (t.sum != t.sum) loss = NAN;
    if (t.hard) loss += t.label < a.classes ? a.hard * (logf(at_1) - (x((int)t.label) - most)) : NAN;
    return loss;
}

// Factors of the row's gradient: it is soft exp((s - most) / T) + hard exp(s - most) without
// the entries, and amount[e] becomes what each entry takes off.
struct Factors {
    float soft, hard;
    // Of s - most.  A row without a part of the loss has its gradient 0 whatever its logits are.
    __device__ __forceinline__ float operator()(const DistillArgs& a, float d) const {
        float g = 0.f;
        if (soft != 0.f) g = soft * exp_of(d, kLog2e * a.inv_t);
        if (hard != 0.f) g = fmaf(hard, exp_of(d, kLog2e), g);
        return g;
    }
};
// The entries that there are: without `hard` labels are none.
__device__ __forceinline__ int entries_of(const DistillArgs& a) { return a.kept + (a.hard > 0.f); }
template <typename Team>
__device__ __forceinline__ Factors entry_amounts(const DistillArgs& a, int64_t row, Team& team, const Targets& t, float at_t,
                                                 float at_1) {
    const float up = (a.up ? a.up[row * a.up_step] : 1.f) * a.up_scale;
    const float soft_up = !t.soft ? 0.f : t.sum != t.sum ? NAN : a.soft_grad * up;
    const float hard_up = !t.hard ? 0.f : t.label < a.classes ? a.hard * up : NAN;
    for (int e = team.lane; e < entries_of(a); e += team.lanes) {
        if (e < a.kept) {
            t.amount[e] = t.soft && t.place[e] >= 0 ? soft_up * (exp_of(t.amount[e] - t.top, kLog2e * a.inv_t) / t.sum) : 0.f;
            if (!t.soft) t.place[e] = -1;
        } else {
            t.amount[e] = hard_up;
            t.place[e] = t.hard && t.label < a.classes ? (int32_t)t.label : -1;
        }
    }
    return {t.soft ? soft_up / at_t : 0.f, t.hard ? hard_up / at_1 : 0.f};
}
// What all of the first n entries of e's class take off; `first`: no earlier entry has it.
__device__ __forceinline__ float class_amount(const Targets& t, int n, int e, bool& first) {
    float off = 0.f;
    first = true;
    for (int f = 0; f < n; ++f) {
        if (t.place[f] != t.place[e]) continue;
        first &= f >= e;
        off += t.amount[f];
    }
    return off;
}

// ------------------------------------------------------------------ short rows
// Rows of up to 1,024 classes.  A workgroup takes stage_rows of them, one run of memory,
// through LDS: whole 16-byte packets whatever the number of classes is, where rows of 47
// elements would be read by single ones.  A row is held by 2^lanes_shift lanes, K elements
// each; its gradient takes its place in LDS and goes out the same way.
// SHIFT: lanes_shift, or -1 where it is only known at run time; HARD: labels count.  Both are
// constants because the choices they leave would stand at every element and every sum.
// Up to 10 classes a lane five workgroups fit a CU, with labels and up to eleven registers spilled (fp32: three)
// (769,230 x 65 in fp32 with labels 169 us, with four workgroups 195; in bf16 twice as many 279, 298).  With 16
// classes, labels and 16 bits up to four are spilled at four workgroups.
template <typename T, int K, int SHIFT, bool HARD>
__global__ __launch_bounds__(kThreads, K <= 10 ? 5 : 4) void distill_short(const DistillArgs args) {
    DistillArgs a = args;
    if constexpr (SHIFT >= 0) a.lanes_shift = SHIFT;
    if constexpr (!HARD) a.hard = 0.f;
    extern __shared__ __align__(16) char lds[];
    __shared__ double part64[kThreads / 64];
    constexpr int kPer = 16 / sizeof(T);
    const int lanes = 1 << a.lanes_shift, group = threadIdx.x >> a.lanes_shift, groups = kThreads >> a.lanes_shift;
    const int C = a.classes, entries = a.kept + 1;
    T* const stage = reinterpret_cast<T*>(lds);
    float* const arrays = reinterpret_cast<float*>(lds + (a.stage_rows * C * (int)sizeof(T) + 15) / 16 * 16);
    WaveTeam team{(int)threadIdx.x & (lanes - 1), lanes};
    Targets t{};
    t.amount = arrays + group * entries;
    t.place = reinterpret_cast<int32_t*>(arrays) + (groups + group) * entries;
    float* const value = arrays + (2 * groups + group) * entries;  // what an entry writes, and where (-1: another does)
    int32_t* const to = reinterpret_cast<int32_t*>(arrays) + (3 * groups + group) * entries;
    uint16_t* const owner = reinterpret_cast<uint16_t*>(arrays + 4 * groups * entries) + group * C;
    const float c = kLog2e * a.inv_t;
    // A lane's classes; groups begin at different ones, which keeps rows of 64 classes apart in LDS.
    // What is past the row is read at class 0 and written past the stage.
    int at[K];
    bool inside[K];
    T* const past = reinterpret_cast<T*>(owner - group * C + groups * C);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        at[k] = (k + group) % K * lanes + (int)team.lane;
        inside[k] = at[k] < C;
        at[k] = inside[k] ? at[k] : 0;
    }
    double total = 0.0;
    for (int64_t first = (int64_t)blockIdx.x * a.stage_rows; first < a.rows; first += (int64_t)gridDim.x * a.stage_rows) {
        const int rows = (int)min((int64_t)a.stage_rows, a.rows - first), n = rows * C;
        const T* const from = static_cast<const T*>(a.logits) + first * a.ld;
        const int packets = a.whole ? n / kPer : 0;
        for (int p0 = threadIdx.x; p0 < packets; p0 += kAhead * kThreads) {
            uint4 v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) v[u] = reinterpret_cast<const uint4*>(from)[min(p0 + u * kThreads, packets - 1)];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (p0 + u * kThreads < packets) reinterpret_cast<uint4*>(stage)[p0 + u * kThreads] = v[u];
        }
        if (a.whole) {
            const int i = packets * kPer + (int)threadIdx.x;
            if (i < n) stage[i] = from[i];
        } else {
            for (int r = threadIdx.x >> 6; r < rows; r += kThreads / 64)
                for (int j = threadIdx.x & 63; j < C; j += 64) stage[r * C + j] = from[r * a.ld + j];
        }
        __syncthreads();
        for (int r0 = 0; r0 < rows; r0 += groups) {
            const bool there = r0 + group < rows;
            const int r = there ? r0 + group : 0;  // lanes without a row go along with the first and keep nothing
            const int64_t row = first + r;
            T* const x = stage + r * C;
            auto logit = [&](int j) { return (float)x[j]; };
            read_targets(a, row, team, t);
            float v[K], most = -FLT_MAX, at_t = 0.f, at_1 = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const float value_at = (float)x[at[k]];
                v[k] = inside[k] ? value_at : -INFINITY;
                most = fmaxf(most, v[k]);
            }
            most = team.template all<Max>(most);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                v[k] -= most;
                const float e = exp_of(v[k], c);
                at_t += e;
                if constexpr (HARD) at_1 += exp_of(v[k], kLog2e);
                else v[k] = e;  // stays for the gradient
            }
            at_t = team.sum(at_t);
            if constexpr (HARD) at_1 = team.sum(at_1);
            if (a.loss || a.part) {
                const float loss = row_loss(a, team, t, most, at_t, at_1, logit);
                if (there && team.lane == 0) {
                    if (a.loss) a.loss[row] = loss;
                    total += loss;
                }
            }
            if (!a.grad) continue;
            const Factors f = entry_amounts(a, row, team, t, at_t, at_1);
            team.sync();
            // Whether a class has several entries: one of them is not its owner then.  The label is
            // often one of the teacher's classes: an entry of its class takes it along (1e6 x 100 in bf16
            // 227 us, 267 where that counted as twice); else it is an entry of its own.
            const int32_t label = HARD ? t.place[a.kept] : -1;
            if (HARD) {
                if (label >= 0) owner[label] = (uint16_t)a.kept;
                team.sync();
            }
            for (int e = team.lane; e < a.kept; e += lanes)
                if (t.place[e] >= 0) owner[t.place[e]] = (uint16_t)e;
            team.sync();
            bool twice = false;
            for (int e = team.lane; e < a.kept; e += lanes) twice |= t.place[e] >= 0 && owner[t.place[e]] != e;
            const bool any_twice = __any(twice);
            for (int e = team.lane; e < a.kept + HARD; e += lanes) {
                const int32_t j = t.place[e];
                bool first_of = true;
                float off = t.amount[e];
                if (HARD && e == a.kept) {
                    first_of = j >= 0 && owner[j] == e;
                } else {
                    if (any_twice && j >= 0) off = class_amount(t, a.kept, e, first_of);
                    if (HARD && j == label) off += t.amount[a.kept];
                }
                value[e] = j >= 0 ? f(a, logit(j) - most) - off : 0.f;
                to[e] = first_of && there ? j : -1;
            }
            team.sync();
            if (there) {
                const bool live = t.soft || t.hard;  // else 0 whatever the logits are
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const float g = HARD ? fmaf(f.hard, exp_of(v[k], kLog2e), f.soft * exp_of(v[k], c)) : f.soft * v[k];
                    *(inside[k] ? x + at[k] : past) = (T)(live ? g : 0.f);
                }
            }
            team.sync();
            for (int e = team.lane; e < a.kept + HARD; e += lanes)
                if (to[e] >= 0) x[to[e]] = (T)value[e];
        }
        __syncthreads();
        if (a.grad) {
            T* const out = static_cast<T*>(a.grad) + first * C;
            if (a.whole) {
                for (int i = threadIdx.x * kPer; i + kPer <= n; i += kThreads * kPer)
                    *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(stage + i);
                const int i = n / kPer * kPer + (int)threadIdx.x;
                if (i < n) out[i] = stage[i];
            } else {
                for (int i = threadIdx.x; i < n; i += kThreads) out[i] = stage[i];
            }
            __syncthreads();
        }
    }
    if (a.part) {
        total = sum_workgroup(total, part64);
        if (threadIdx.x == 0) a.part[blockIdx.x] = total;
    }
}

// ------------------------------------------------------- many rows of few classes
// A lane per row, 64 rows of up to 64 classes in LDS as floats, rows at an odd pitch: no
// sums between lanes, and the logarithms, divisions and entries of 64 rows at once.  The
// rows come and go as one run of memory, like those of distill_short, and so do the
// entries: read by their lanes, each load would touch 64 lines.  FLAT: the number of classes is
// odd, and so the pitch itself.
template <typename T, bool FLAT>
__global__ __launch_bounds__(64, FLAT ? 3 : 2) void distill_lanes(const DistillArgs a) {
    extern __shared__ __align__(16) float stage[];
    constexpr int kPer = 16 / sizeof(T), kPackets = kLaneClasses / kPer;
    typedef T vec __attribute__((ext_vector_type(kPer)));
    constexpr uint8_t kOutside = 254, kNone = 255;
    const int C = a.classes, pitch = FLAT ? C : C | 1, lane = threadIdx.x;
    const uint32_t magic = ((1u << 20) + C - 1) / C;  // i / C = i * magic >> 20 for i < 64 C <= 4096
    const int k = a.kept, entry_pitch = k | 1;
    const uint32_t entry_magic = k ? ((1u << 20) + k - 1) / k : 0;
    const float c = kLog2e * a.inv_t;
    float* const x = stage + lane * pitch;
    float* const amounts = stage + 64 * pitch;
    uint8_t* const places = reinterpret_cast<uint8_t*>(amounts + 64 * entry_pitch);  // class, kNone or kOutside
    const uint8_t* const place = places + lane * entry_pitch;
    float* const amount = amounts + lane * entry_pitch;  // logit, then exp((logit - top) / T)
    double total = 0.0;
    for (int64_t first = (int64_t)blockIdx.x * 64; first < a.rows; first += (int64_t)gridDim.x * 64) {
        const int rows = (int)min((int64_t)64, a.rows - first), n = rows * C;
        const T* const from = static_cast<const T*>(a.logits) + first * a.ld;
        const int packets = FLAT || a.whole ? n / kPer : 0;
        // All loads of the 64 rows before the first use: few waves fit a CU, so each keeps much in flight.
        vec v[kPackets];
#pragma unroll
        for (int u = 0; u < kPackets; ++u)
            if (u * 64 < packets) v[u] = *reinterpret_cast<const vec*>(from + min(u * 64 + lane, packets - 1) * kPer);
        const int64_t row = first + min(lane, rows - 1);
        const int64_t label = label_at(a, row);
        for (int u0 = 0; u0 < k; u0 += 8) {
            int64_t ids[8];
            float logits[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = min((u0 + u) * 64 + lane, rows * k - 1), r = (int)((uint32_t)i * entry_magic >> 20), e = i - r * k;
                ids[u] = id_at(a, (first + r) * a.ldi + e);
                logits[u] = teacher_at(a, (first + r) * a.ldt + e);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = min((u0 + u) * 64 + lane, rows * k - 1), r = (int)((uint32_t)i * entry_magic >> 20), e = i - r * k;
                places[r * entry_pitch + e] = ids[u] < 0 || logits[u] == -INFINITY ? kNone : ids[u] < C ? (uint8_t)ids[u] : kOutside;
                amounts[r * entry_pitch + e] = logits[u];
            }
        }
#pragma unroll
        for (int u = 0; u < kPackets; ++u) {
            const int p = u * 64 + lane;
            if (u * 64 < packets && p < packets) {
                if constexpr (FLAT) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e) stage[p * kPer + e] = (float)v[u][e];
                } else {
                    int r = (int)((uint32_t)(p * kPer) * magic >> 20), j = p * kPer - r * C;
#pragma unroll
                    for (int e = 0; e < kPer; ++e) {
                        stage[r * pitch + j] = (float)v[u][e];
                        const bool next = ++j == C;
                        r += next;
                        j = next ? 0 : j;
                    }
                }
            }
        }
        for (int i = packets * kPer + lane; i < n; i += 64) {
            const int r = (int)((uint32_t)i * magic >> 20), j = i - r * C;
            stage[r * pitch + j] = (float)from[r * a.ld + j];
        }
        __syncthreads();
        const bool there = lane < rows;  // the other lanes go along and keep nothing
        float most = -FLT_MAX;
#pragma unroll 8
        for (int j = 0; j < C; ++j) most = fmaxf(most, x[j]);
        float top = -INFINITY;
        bool outside = false;
        for (int e = 0; e < k; ++e) {
            outside |= place[e] == kOutside;
            if (place[e] != kNone) top = amount[e] != amount[e] ? INFINITY : fmaxf(top, amount[e]);
        }
        const bool soft = a.soft > 0.f && top != -INFINITY;
        float sum = outside ? NAN : 0.f, inner = 0.f;
        for (int e = 0; e < k; ++e) {
            const float t = amount[e];
            const float w = place[e] < C ? exp_of(t - top, c) : 0.f;
            sum += w;
            if (w != 0.f) inner = fmaf(w, (t - top) - (x[place[e]] - most), inner);
            amount[e] = w;
        }
        const bool hard = a.hard > 0.f && label >= 0, inside = label >= 0 && label < C;
        const float at_label = x[inside ? (int)label : 0] - most;
        float at_t = 0.f, at_1 = 0.f;
        if (a.hard > 0.f) {
#pragma unroll 8
            for (int j = 0; j < C; ++j) {
                const float v = x[j] - most;
                at_t += exp_of(v, c);
                at_1 += exp_of(v, kLog2e);
            }
        } else {  // one exponential an element: it stays for the gradient
#pragma unroll 8
            for (int j = 0; j < C; ++j) {
                const float e = exp_of(x[j] - most, c);
                at_t += e;
                x[j] = e;
            }
        }
        const float per_sum = 1.f / sum;
        if (a.loss || a.part) {
            float loss = 0.f;
            if (soft) loss = a.soft * fmaf(inner * per_sum, a.inv_t, logf(at_t) - logf(sum));
            if (hard) loss += inside ? a.hard * (logf(at_1) - at_label) : NAN;
            if (there) {
                if (a.loss) a.loss[row] = loss;
                total += loss;
            }
        }
        if (a.grad) {
            const float up = (a.up ? a.up[row * a.up_step] : 1.f) * a.up_scale;
            const float soft_up = !soft ? 0.f : sum != sum ? NAN : a.soft_grad * up;
            const float hard_up = !hard ? 0.f : inside ? a.hard * up : NAN;
            const float fs = soft ? soft_up / at_t : 0.f, fh = hard ? hard_up / at_1 : 0.f;
            if (a.hard > 0.f) {
#pragma unroll 8
                for (int j = 0; j < C; ++j) {
                    const float v = x[j] - most;
                    x[j] = fmaf(fh, exp_of(v, kLog2e), fs * exp_of(v, c));
                }
            } else {
#pragma unroll 8
                for (int j = 0; j < C; ++j) x[j] *= fs;
            }
            if (!soft && !hard)  // whatever the logits are
                for (int j = 0; j < C; ++j) x[j] = 0.f;
            if (soft)
                for (int e = 0; e < k; ++e)
                    if (place[e] < C) x[place[e]] -= soft_up * (amount[e] * per_sum);
            if (hard && inside) x[label] -= hard_up;
            __syncthreads();
            T* const to = static_cast<T*>(a.grad) + first * C;
#pragma unroll 2
            for (int p = lane; p < packets; p += 64) {
                vec out;
                if constexpr (FLAT) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e) out[e] = (T)stage[p * kPer + e];
                } else {
                    int r = (int)((uint32_t)(p * kPer) * magic >> 20), j = p * kPer - r * C;
#pragma unroll
                    for (int e = 0; e < kPer; ++e) {
                        out[e] = (T)stage[r * pitch + j];
                        if (++j == C) {
                            j = 0;
                            ++r;
                        }
                    }
                }
                *reinterpret_cast<vec*>(to + p * kPer) = out;
            }
            for (int i = packets * kPer + lane; i < n; i += 64) {
                const int r = (int)((uint32_t)i * magic >> 20), j = i - r * C;
                to[i] = (T)stage[r * pitch + j];
            }
        }
        __syncthreads();
    }
    if (a.part) {
        total = sum_lanes(total, 64);
        if (lane == 0) a.part[blockIdx.x] = total;
    }
}

// ------------------------------------------------------------------- long rows
// 16 bytes of a row; elements past the packets, at both ends, are taken one by one.
template <typename T>
struct Span {
    static constexpr int kPer = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(kPer)));
    int first, packets, end;  // [first, first + kPer * packets) lies on whole packets
    __device__ __forceinline__ Span(const T* x, int begin, int end_) : end(end_) {
        const int off = (int)((reinterpret_cast<uintptr_t>(x + begin) % 16) / sizeof(T));
        first = min(end, begin + (off ? kPer - off : 0));
        packets = (end - first) / kPer;
    }
};

// A team's maximum of a part of a row and the sums of its exponentials at T and at 1, in one
// pass: every lane scales its sums down when its maximum grows.
template <typename T, typename Team>
__device__ __forceinline__ void scan_part(const DistillArgs& a, Team& team, const T* x, int begin, int end, float& most, float& at_t,
                                          float& at_1) {
    using S = Span<T>;
    const float c = kLog2e * a.inv_t;
    const bool hard = a.hard > 0.f;
    most = -FLT_MAX;
    at_t = at_1 = 0.f;
    const S s(x, begin, end);
    auto add = [&](const float* v, int n) {
        float top = most;
        for (int i = 0; i < n; ++i) top = fmaxf(top, v[i]);
        const float down = most - top;
        at_t *= exp_of(down, c);
        for (int i = 0; i < n; ++i) at_t += exp_of(v[i] - top, c);
        if (hard) {
            at_1 *= exp_of(down, kLog2e);
            for (int i = 0; i < n; ++i) at_1 += exp_of(v[i] - top, kLog2e);
        }
        most = top;
    };
    for (int p = team.lane; p < s.packets; p += kAhead * team.lanes) {
        typename S::vec v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            v[u] = *reinterpret_cast<const typename S::vec*>(x + s.first + min(p + u * team.lanes, s.packets - 1) * S::kPer);
        float f[kAhead * S::kPer];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int e = 0; e < S::kPer; ++e) f[u * S::kPer + e] = p + u * team.lanes < s.packets ? (float)v[u][e] : -INFINITY;
        add(f, kAhead * S::kPer);
    }
    const int tail = s.first + s.packets * S::kPer;
    for (int j = begin + team.lane; j < s.first; j += team.lanes) {
        const float f = (float)x[j];
        add(&f, 1);
    }
    for (int j = tail + team.lane; j < end; j += team.lanes) {
        const float f = (float)x[j];
        add(&f, 1);
    }
    const float top = team.template all<Max>(most);
    at_t = team.sum(at_t * exp_of(most - top, c));
    if (hard) at_1 = team.sum(at_1 * exp_of(most - top, kLog2e));
    most = top;
}

// to[j] = f(x[j]) over a part of a row, in whole packets where both lie alike.
template <bool AROUND, typename T, typename Team, typename F>
__device__ __forceinline__ void write_part(const Team& team, const T* x, T* to, int begin, int end, F f) {
    using S = Span<T>;
    if ((reinterpret_cast<uintptr_t>(to) - reinterpret_cast<uintptr_t>(x)) % 16 != 0) {
        for (int j = begin + team.lane; j < end; j += team.lanes) to[j] = (T)f((float)x[j]);
        return;
    }
    const S s(x, begin, end);
    for (int p = team.lane; p < s.packets; p += kAhead * team.lanes) {
        typename S::vec v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            v[u] = *reinterpret_cast<const typename S::vec*>(x + s.first + min(p + u * team.lanes, s.packets - 1) * S::kPer);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (p + u * team.lanes >= s.packets) break;
#pragma unroll
            for (int e = 0; e < S::kPer; ++e) v[u][e] = (T)f((float)v[u][e]);
            auto* const at = reinterpret_cast<typename S::vec*>(to + s.first + (p + u * team.lanes) * S::kPer);
            if constexpr (AROUND) __builtin_nontemporal_store(v[u], at);
            else *at = v[u];
        }
    }
    for (int j = begin + team.lane; j < s.first; j += team.lanes) to[j] = (T)f((float)x[j]);
    for (int j = s.first + s.packets * S::kPer + team.lane; j < end; j += team.lanes) to[j] = (T)f((float)x[j]);
}

// Rows cut into pieces: each piece's maximum and sums.
template <typename T>
__global__ __launch_bounds__(512) void distill_pieces(const DistillArgs a) {
    __shared__ float lds[32];
    WorkgroupTeam team{(int)threadIdx.x, (int)blockDim.x, lds};
    for (int64_t work = blockIdx.x; work < a.rows * a.pieces; work += gridDim.x) {
        const int64_t row = work / a.pieces;
        const int begin = (int)(work - row * a.pieces) * a.piece, end = min(a.classes, begin + a.piece);
        float most, at_t, at_1;
        scan_part(a, team, static_cast<const T*>(a.logits) + row * a.ld, begin, end, most, at_t, at_1);
        if (threadIdx.x == 0) *reinterpret_cast<float4*>(a.piece_stats + 4 * work) = make_float4(most, at_t, at_1, 0.f);
        __syncthreads();
    }
}

// A team per row, or per piece of one where the gradient is wanted; the loss is formed by the
// first piece.  Teams are waves for the shorter rows, whose exchange needs no barrier, else
// workgroups.
template <typename T, bool AROUND, typename Team>
__global__ __launch_bounds__(512) void distill_long(const DistillArgs a) {
    constexpr bool kWave = std::is_same<Team, WaveTeam>::value;
    extern __shared__ float entries[];
    __shared__ float lds[32];
    __shared__ double part64[8];
    Team team{};
    const int unit = kWave ? threadIdx.x >> 6 : 0, units = kWave ? blockDim.x >> 6 : 1;
    team.lane = kWave ? threadIdx.x & 63 : threadIdx.x;
    team.lanes = kWave ? 64 : blockDim.x;
    if constexpr (!kWave) team.lds = lds;
    Targets t{};
    t.amount = entries + unit * 2 * (a.kept + 1);
    t.place = reinterpret_cast<int32_t*>(t.amount) + a.kept + 1;
    const int pieces = a.grad ? a.pieces : 1;
    double total = 0.0;
    for (int64_t work = (int64_t)blockIdx.x * units + unit; work < a.rows * pieces; work += (int64_t)gridDim.x * units) {
        const int64_t row = work / pieces;
        const int piece = (int)(work - row * pieces);
        const int begin = a.grad ? piece * a.piece : 0, end = a.grad ? min(a.classes, begin + a.piece) : a.classes;
        const T* const x = static_cast<const T*>(a.logits) + row * a.ld;
        auto logit = [&](int j) { return (float)x[j]; };
        read_targets(a, row, team, t);
        float most = -FLT_MAX, at_t = 0.f, at_1 = 0.f;
        if (a.kept_stats) {
            const float4 k = *reinterpret_cast<const float4*>(a.kept_stats + 4 * row);
            most = k.x;
            at_t = k.y;
            at_1 = k.z;
        } else if (a.piece_stats) {
            const float4* const from = reinterpret_cast<const float4*>(a.piece_stats) + row * a.pieces;
            for (int p = team.lane; p < a.pieces; p += team.lanes) most = fmaxf(most, from[p].x);
            most = team.template all<Max>(most);
            for (int p = team.lane; p < a.pieces; p += team.lanes) {
                at_t = fmaf(from[p].y, exp_of(from[p].x - most, kLog2e * a.inv_t), at_t);
                at_1 = fmaf(from[p].z, exp_of(from[p].x - most, kLog2e), at_1);
            }
            at_t = team.sum(at_t);
            at_1 = team.sum(at_1);
        } else if (t.soft || t.hard) {
            scan_part(a, team, x, 0, a.classes, most, at_t, at_1);
        }
        if (piece == 0) {
            if (a.stats && team.lane == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(most, at_t, at_1, 0.f);
            if (a.loss || a.part) {
                const float loss = row_loss(a, team, t, most, at_t, at_1, logit);
                if (a.loss && team.lane == 0) a.loss[row] = loss;
                total += loss;
            }
        }
        if (a.grad) {
            team.sync();  // all have read the amounts
            const Factors f = entry_amounts(a, row, team, t, at_t, at_1);
            T* const g = static_cast<T*>(a.grad) + row * a.classes;
            // The same in every lane: the loops over the row have no choice left in them.
            const float soft = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(f.soft)));
            const float hard = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(f.hard)));
            const float c = kLog2e * a.inv_t;
            if (soft == 0.f && hard == 0.f) write_part<AROUND, T>(team, x, g, begin, end, [&](float) { return 0.f; });
            else if (hard == 0.f) write_part<AROUND, T>(team, x, g, begin, end, [&](float v) { return soft * exp_of(v - most, c); });
            else write_part<AROUND, T>(team, x, g, begin, end, [&](float v) {
                return fmaf(hard, exp_of(v - most, kLog2e), soft * exp_of(v - most, c));
            });
            __threadfence_block();
            team.sync();
            const int n = entries_of(a);
            for (int e = team.lane; e < n; e += team.lanes) {
                const int32_t j = t.place[e];
                if (j < begin || j >= end) continue;
                bool first;
                const float off = class_amount(t, n, e, first);
                if (first) g[j] = (T)(f(a, logit(j) - most) - off);
            }
        }
        team.sync();
    }
    if (!a.part) return;
    if constexpr (kWave) {
        if (team.lane == 0) part64[unit] = total;
        __syncthreads();
        for (int u = 1; u < units; ++u) total += part64[u];
    }
    if (threadIdx.x == 0) a.part[blockIdx.x] = total;
}

// The workgroups' parts in order.
__global__ __launch_bounds__(1024) void distill_reduce(const double* __restrict__ part, int parts, double scale, float* loss) {
    __shared__ double sums[16];
    double s = 0.0;
#pragma unroll 4
    for (int p = threadIdx.x; p < parts; p += 1024) s += part[p];
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

int64_t size_of(int32_t dtype) { return dtype == RA_DTYPE_F32 ? 4 : 2; }

// The gradient of long rows is written before what is kept of them has been read for the last time, so no output may
// take an input's place.
ra_status refuse_shared(const ra_distill_shape& s, std::initializer_list<Extent> outputs, const void* logits, const void* teacher,
                        const void* ids, const void* labels, const Extent& factor, const Extent& stats) {
    return refuse_overlap("distill", outputs,
                          {rows_of("logits", logits, s.rows, s.classes, s.ld_logits, size_of(s.dtype)),
                           rows_of("teacher", s.kept ? teacher : nullptr, s.rows, s.kept, s.ld_teacher, size_of(s.teacher_dtype)),
                           rows_of("ids", s.kept ? ids : nullptr, s.rows, s.kept, s.ld_ids, s.ids64 ? 8 : 4),
                           rows_of("labels", labels, s.rows, 1, 1, s.labels64 ? 8 : 4), factor, stats});
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
    a.inv_t = static_cast<float>(1.0 / s.temperature);
    a.soft = static_cast<float>((1.0 - s.hard) * s.temperature * s.temperature);
    a.hard = s.hard;
    a.soft_grad = static_cast<float>((1.0 - s.hard) * s.temperature);
    return a;
}

bool by_lanes(const ra_distill_shape& s) { return s.classes <= kLaneClasses && s.kept <= kLaneKept && s.rows >= kLaneRows; }
size_t lane_lds(const ra_distill_shape& s) { return (size_t)64 * ((s.classes | 1) * 4 + (s.kept | 1) * 5); }
int lane_blocks(const ra_distill_shape& s) { return static_cast<int>(std::min<int64_t>((s.rows + 63) / 64, kMaxBlocks)); }

bool is_short(const ra_distill_shape& s) { return s.classes <= kMaxShort && s.kept <= 256; }

// What the forward pass leaves for the backward pass: only long rows' statistics cost another reading.
int64_t stats_bytes(const ra_distill_shape& s) { return s.rows == 0 ? 0 : by_lanes(s) || is_short(s) ? 16 : s.rows * 16; }

// Short rows: lanes of a row and rows of a workgroup at once.  A lane takes 4 elements, and 16
// past 256 classes, or past 32 where rows are enough to fill the machine with a quarter of the
// lanes: what is done once a row is done by fewer (1e6 x 100 bf16 436 us with 4, 257 with 16);
// 8, 10 or 13 where the same lanes hold the row so (with 16 alone, 200 MB of logits in bf16:
// 1.54e6 x 65 212 us, 267, 1.25e6 x 80 182, 229, 333,333 x 300 181, 226, 156,250 x 640 176, 219;
// fp32 500,000 x 100 123, 144).  More lanes where the entries of all groups would pass 16 kB.
struct ShortPlan {
    int k, shift, rows, blocks;
    size_t lds;
};
ShortPlan short_plan(const ra_distill_shape& s) {
    const int size = s.dtype == RA_DTYPE_F32 ? 4 : 2, entries = s.kept + 1;
    ShortPlan p{};
    p.k = s.classes <= 256 && (s.classes <= 32 || s.rows * s.classes < 16 * 256 * kThreads) ? 4 : 16;
    if (p.k == 16) p.shift = 3;  // 8 lanes at least: kernels of their own for each number
    while ((p.k << p.shift) < s.classes || (kThreads >> p.shift) * entries * 16 > 4 * 257 * 16) ++p.shift;
    // Few rows: more lanes for each, and fewer rows a workgroup, so that all CUs have some.
    while (p.shift < 6 && (s.rows << p.shift) < 256 * kThreads && (1 << p.shift) < s.classes) ++p.shift;
    if (p.k == 16)
        for (int k : {13, 10, 8})
            if ((k << p.shift) >= s.classes) p.k = k;
    const int groups = kThreads >> p.shift;
    p.rows = std::max(groups, 8);  // 8 rows are whole packets
    while (2 * p.rows * s.classes * size <= kStageBytes && s.rows / (2 * p.rows) >= 1024) p.rows *= 2;
    p.blocks = static_cast<int>(std::min<int64_t>((s.rows + p.rows - 1) / p.rows, kMaxBlocks));
    p.lds = (size_t)(p.rows * s.classes * size + 15) / 16 * 16 + (size_t)groups * entries * 16 +
            ((size_t)groups * s.classes * 2 + 3) / 4 * 4 + 4;
    return p;
}

// Long rows: whole where there are two for every CU, else in pieces of at least 4,096 classes.
struct LongPlan {
    int pieces, piece, threads;
    bool wave;
};
LongPlan long_plan(const ra_distill_shape& s) {
    LongPlan p{};
    const int64_t want = s.rows ? (512 + s.rows - 1) / s.rows : 1;
    p.pieces = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, s.classes / 4096)));
    p.piece = (s.classes + p.pieces - 1) / p.pieces;
    p.threads = p.piece >= 16384 ? 512 : 256;
    // A wave a row, loss and gradient in one call (a workgroup a row): 15,000 rows of 2,000 in bf16 38 us
    // (102), 1,000 of them 11.2 (14.3), 7,500 of 4,000 34 (60), 500 of them 11.8 (11.8), 3,750 of 8,000 33 (38),
    // 1,250 of them 19.4 (17.9), 1,875 of 16,000 33 (36) and in fp32 937 of them 34.6 (33.0).
    p.wave = s.classes <= 2048 || (s.classes <= 8192 && s.rows >= 2048);
    return p;
}
int long_blocks(const ra_distill_shape& s, int pieces) {
    const int units = long_plan(s).wave ? kThreads / 64 : 1;
    return static_cast<int>(std::min<int64_t>((s.rows * pieces + units - 1) / units, kMaxBlocks));
}

// Workgroups that leave a part of the loss.
int loss_parts(const ra_distill_shape& s, bool grad) {
    if (s.rows == 0) return 0;
    if (by_lanes(s)) return lane_blocks(s);
    return is_short(s) ? short_plan(s).blocks : long_blocks(s, grad ? long_plan(s).pieces : 1);
}

template <int N>
using Int = std::integral_constant<int, N>;

template <typename F>
void by_type(int32_t dtype, F f) {
    if (dtype == RA_DTYPE_F32) f(float());
    else if (dtype == RA_DTYPE_F16) f(f16_t());
    else f(bf16_t());
}

void run(const ra_distill_shape& s, DistillArgs& a, hipStream_t st) {
    a.whole = (s.rows <= 1 || s.ld_logits == s.classes) && aligned16(a.logits) && aligned16(a.grad);
    if (by_lanes(s)) {
        by_type(s.dtype, [&](auto t) {
            using T = decltype(t);
            if (a.whole && s.classes % 2) distill_lanes<T, true><<<lane_blocks(s), 64, lane_lds(s), st>>>(a);
            else distill_lanes<T, false><<<lane_blocks(s), 64, lane_lds(s), st>>>(a);
        });
        return;
    }
    if (is_short(s)) {
        const ShortPlan p = short_plan(s);
        a.stage_rows = p.rows;
        a.lanes_shift = p.shift;
        by_type(s.dtype, [&](auto t) {
            using T = decltype(t);
            auto go = [&](auto k, auto shift) {
                if (s.hard > 0.f) distill_short<T, k.value, shift.value, true><<<p.blocks, kThreads, p.lds, st>>>(a);
                else distill_short<T, k.value, shift.value, false><<<p.blocks, kThreads, p.lds, st>>>(a);
            };
            auto by_shift = [&](auto k) {
                if (p.shift == 3) go(k, Int<3>());
                else if (p.shift == 4) go(k, Int<4>());
                else if (p.shift == 5) go(k, Int<5>());
                else go(k, Int<6>());
            };
            if (p.k == 4) go(Int<4>(), Int<-1>());
            else if (p.k == 8) by_shift(Int<8>());
            else if (p.k == 10) by_shift(Int<10>());
            else if (p.k == 13) by_shift(Int<13>());
            else by_shift(Int<16>());
        });
        return;
    }
    const LongPlan p = long_plan(s);
    a.pieces = p.pieces;
    a.piece = p.piece;
    const size_t lds = (size_t)(s.kept + 1) * 8;
    by_type(s.dtype, [&](auto t) {
        using T = decltype(t);
        if (a.kept_stats || p.pieces == 1) a.piece_stats = nullptr;
        else distill_pieces<T><<<long_blocks(s, p.pieces), p.threads, 0, st>>>(a);
        const int threads = a.grad || p.pieces == 1 ? p.threads : 256;
        const int blocks = long_blocks(s, a.grad ? p.pieces : 1);
        const bool around = a.grad && s.rows * s.classes * (int64_t)sizeof(T) > kAroundBytes;
        if (p.wave) {
            const size_t all = lds * (kThreads / 64);
            if (around) distill_long<T, true, WaveTeam><<<blocks, kThreads, all, st>>>(a);
            else distill_long<T, false, WaveTeam><<<blocks, kThreads, all, st>>>(a);
        } else if (around) {
            distill_long<T, true, WorkgroupTeam><<<blocks, threads, lds, st>>>(a);
        } else {
            distill_long<T, false, WorkgroupTeam><<<blocks, threads, lds, st>>>(a);
        }
    });
}

}  // namespace
}  // namespace ra

using ra::fail;

extern "C" {

ra_status ra_distill_workspace(const ra_distill_shape* s, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "distill: bytes is NULL");
    RA_TRY(ra::check(s));
    *bytes = 0;
    if (s->rows == 0) return RA_OK;
    if (s->reduction != RA_REDUCE_NONE) *bytes = (int64_t)ra::kMaxBlocks * (int64_t)sizeof(double);
    if (!ra::by_lanes(*s) && !ra::is_short(*s)) *bytes += s->rows * (ra::long_plan(*s).pieces > 1 ? ra::long_plan(*s).pieces : 0) * 16;
    return RA_OK;
}

ra_status ra_distill_stats_bytes(const ra_distill_shape* s, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "distill: bytes is NULL");
    RA_TRY(ra::check(s));
    *bytes = ra::stats_bytes(*s);
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
    if (!ra::aligned16(d_stats)) return fail(RA_ERR_INVALID_ARGUMENT, "distill: stats must be 16-byte aligned");
    RA_TRY(ra::refuse_shared(*s,
                             {ra::rows_of("loss", d_loss, s->reduction == RA_REDUCE_NONE ? s->rows : 1, 1, 1, sizeof(float)),
                              {"stats", d_stats, static_cast<uint64_t>(ra::stats_bytes(*s))},
                              ra::rows_of("the gradient", d_grad, s->rows, s->classes, s->classes, ra::size_of(s->dtype)),
                              {"the workspace", d_workspace, static_cast<uint64_t>(need)}},
                             d_logits, d_teacher, d_ids, d_labels, {"factor", d_factor, sizeof(float)}, {}));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    ra::DistillArgs a = ra::args_of(*s, d_logits, d_teacher, d_ids, d_labels);
    a.up = d_factor;
    a.stats = d_stats;
    a.grad = d_grad;
    char* work = static_cast<char*>(d_workspace);
    if (s->reduction == RA_REDUCE_NONE) {
        a.loss = d_loss;
    } else {
        a.part = reinterpret_cast<double*>(work);
        work += (int64_t)ra::kMaxBlocks * (int64_t)sizeof(double);
    }
    a.piece_stats = reinterpret_cast<float*>(work);
    if (s->rows) {
        ra::run(*s, a, st);
        RA_LAUNCH_CHECK("distill");
    }
    if (s->reduction != RA_REDUCE_NONE) {  // the mean of no rows is NaN
        const double scale = s->reduction == RA_REDUCE_SUM ? 1.0 : s->rows ? 1.0 / static_cast<double>(s->rows) : NAN;
        ra::distill_reduce<<<1, 1024, 0, st>>>(a.part, ra::loss_parts(*s, d_grad != nullptr), scale, d_loss);
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
    if (!ra::aligned16(d_stats)) return fail(RA_ERR_INVALID_ARGUMENT, "distill: stats must be 16-byte aligned");
    RA_TRY(ra::refuse_shared(*s, {ra::rows_of("the gradient", d_grad, s->rows, s->classes, s->classes, ra::size_of(s->dtype))}, d_logits,
                             d_teacher, d_ids, d_labels,
                             ra::rows_of("grad_loss", d_grad_loss, s->reduction == RA_REDUCE_NONE ? s->rows : 1, 1, 1, sizeof(float)),
                             {"stats", d_stats, static_cast<uint64_t>(ra::stats_bytes(*s))}));
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
