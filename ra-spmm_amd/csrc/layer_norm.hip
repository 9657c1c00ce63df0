// layer_norm.hip — layer norm of every row, of x or of x + residual, and its backward
// pass.
//
//     h = x + residual;  n = (h - mean(h)) r,  r = rsqrt(mean((h - mean(h))^2) + eps)
//     y = n w + b
//     dx = r (w g - mean(w g) - n mean(w g n)) + grad_sum;  dw = sum g n,  db = sum g
//
// Bound by memory: every element is read once and written once (x and residual to y and the sum
// forward, h and the gradients to dx backward).  A row lies in the registers of a group of lanes,
// so the variance is summed around the mean without reading again: of a part of a wave for short
// rows, of a wave up to 1,024 elements (at most 16 a lane), of a workgroup up to 16,384 (8 a
// lane, past 8,192 elements 16).  A lane's elements are K packets of 16 bytes, the packets of a
// row side by side over the lanes, at whatever address the row begins; the last packet of a row
// that is not made of whole ones ends with the row, and what it shares with the one before is
// left out of the sums (TAIL) and written by both, the same bits.  Backward, groups go on to
// further rows with the sums of dw and db in registers; a second launch adds the workgroups' sums
// in order.
//
// Measured, forward, backward and the last sum: 1e6 x 256 in bf16 with a residual 398 us (5.2 TB/s), 406
// (5.0) and 6; 4,096 x 8,192 in fp32 with a residual 91 (5.9: the inputs of a repeated pass are partly
// cached), 117 (4.6) and 8; 2,048 x 16,384 in fp32 with a residual 100 (5.4), 140 (3.8: up to 13 registers spilled) and
// 13; 150,000 x 147 in fp16 26 (3.4), 37 (3.6) and 5.  A large copy: 4.75 TB/s.
#include <algorithm>
#include <type_traits>

#include "lanes.hpp"
#include "overlap.hpp"
#include "ra_internal.hpp"
#include "vector_run.hpp"

namespace ra {
namespace {

constexpr int kThreads = 256;       // of a workgroup that holds several rows
constexpr int kMaxDim = 16384;
constexpr int kMaxLane = 16;        // elements of a row in a lane
constexpr int kForwardBlocks = 2048;
// Outputs past the last-level cache (256 MB) are written around the caches, where lines that wait
// to be written slow down what is read next: forward and backward pass of 1e6 x 256 in bf16,
// one after the other, 402 + 429 us, around the caches 398 + 407.
constexpr int64_t kAroundBytes = int64_t(256) << 20;
constexpr int kBackwardBlocks = 2048;
constexpr int kColumns = 16;        // columns of a workgroup that adds the parts of dw and db
constexpr int kAddThreads = 1024;   // and its threads

struct LayerNormArgs {
    const void *x, *res, *gy, *gs;
    void *y, *sum;
    const float *w, *b;
    float* stats;
    float* part;  // [workgroups][2][dim], or NULL
    int64_t rows, ldx, ldr;
    int32_t dim, lanes_shift;
    float eps, count;  // dim as a float
};

// P elements as they lie in memory, zeros where there are none.
template <typename T, int P>
struct Packet {
    typedef T vec __attribute__((ext_vector_type(P), aligned(sizeof(T))));
    vec v;
    __device__ __forceinline__ void load(const T* p, bool there) {
        v = *reinterpret_cast<const vec*>(there ? p : reinterpret_cast<const T*>(kZeroRun));
    }
    __device__ __forceinline__ float at(int e) const { return (float)v[e]; }
};
template <bool AROUND, typename T, int P>
__device__ __forceinline__ void store_packet(T* p, const float* f) {
    typename Packet<T, P>::vec v;
#pragma unroll
    for (int e = 0; e < P; ++e) v[e] = (T)f[e];
    auto* const to = reinterpret_cast<typename Packet<T, P>::vec*>(p);
    if constexpr (AROUND) __builtin_nontemporal_store(v, to);
    else *to = v;
}

// A packet's weights, `none` without any.
template <int P>
__device__ __forceinline__ void load_weights(float* to, const float* from, int at, bool there, float none) {
    Packet<float, P> p;
    p.load(from + at, from && there);
#pragma unroll
    for (int e = 0; e < P; ++e) to[e] = from ? p.at(e) : none;
}

// Where a lane's packets begin, which exist, and how many elements of one belong to the
// packet before.
template <int P, int K, bool TAIL>
struct Places {
    int at[K], skip[K];
    bool there[K];
    __device__ __forceinline__ Places(int lane, int lanes, int dim) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int first = (k * lanes + lane) * P;
            there[k] = first < dim;
            at[k] = TAIL ? min(first, dim - P) : first;
            skip[k] = first - at[k];
        }
    }
    __device__ __forceinline__ bool counts(int k, int e) const { return there[k] && (!TAIL || e >= skip[k]); }
};

// The group of lanes that a row lies in.  WAVE: a part of a wave; else the workgroup,
// whose waves exchange sums through LDS (two sets in turn, so that one barrier a sum is enough).
template <bool WAVE>
struct Group {
    int lane, lanes;
    float* lds;  // [2][2][16]
    int turn = 0;
    __device__ __forceinline__ void sum2(float& a, float& b) {
        if constexpr (WAVE) {
            a = over_lanes<Add>(a, lanes);
            b = over_lanes<Add>(b, lanes);
        } else {
            a = over_lanes<Add>(a, 64);
            b = over_lanes<Add>(b, 64);
            float* const to = lds + turn * 32;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) {
                to[threadIdx.x >> 6] = a;
                to[16 + (threadIdx.x >> 6)] = b;
            }
            __syncthreads();
            a = to[0];
            b = to[16];
            for (int w = 1; w < (int)(blockDim.x >> 6); ++w) {
                a += to[w];
                b += to[16 + w];
            }
        }
    }
    __device__ __forceinline__ float sum(float a) {
        if constexpr (WAVE) return over_lanes<Add>(a, lanes);
        float none = 0.f;
        sum2(a, none);
        return a;
    }
};

template <typename T, int P, int K, bool WAVE, bool TAIL, bool AROUND>
__global__ __launch_bounds__(WAVE ? kThreads : 1024) void layer_norm_forward(const LayerNormArgs a) {
    __shared__ float lds[64];
    Group<WAVE> group{};
    group.lds = lds;
    group.lanes = WAVE ? 1 << a.lanes_shift : blockDim.x;
    group.lane = WAVE ? threadIdx.x & (group.lanes - 1) : threadIdx.x;
    const int64_t units = WAVE ? (int64_t)gridDim.x * (kThreads >> a.lanes_shift) : gridDim.x;
    int64_t row = WAVE ? (int64_t)blockIdx.x * (kThreads >> a.lanes_shift) + (threadIdx.x >> a.lanes_shift) : blockIdx.x;
    const Places<P, K, TAIL> place(group.lane, group.lanes, a.dim);
    const auto& at = place.at;
    const auto& there = place.there;
    float w[K][P], b[K][P];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        load_weights<P>(w[k], a.w, at[k], there[k], 1.f);
        load_weights<P>(b[k], a.b, at[k], there[k], 0.f);
    }
    for (; row < a.rows; row += units) {
        const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
        const int64_t out = row * a.dim;
        Packet<T, P> px[K], pr[K];
#pragma unroll
        for (int k = 0; k < K; ++k) px[k].load(x + at[k], there[k]);
        float h[K][P], s = 0.f;
        if (a.res) {
            const T* const r = static_cast<const T*>(a.res) + row * a.ldr;
#pragma unroll
            for (int k = 0; k < K; ++k) pr[k].load(r + at[k], there[k]);
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int e = 0; e < P; ++e) h[k][e] = (float)(T)(px[k].at(e) + pr[k].at(e));  // the norm is that of the sum as it is kept
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < P; ++e) h[k][e] = px[k].at(e);
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < P; ++e) s += !TAIL || place.counts(k, e) ? h[k][e] : 0.f;
        const float mean = group.sum(s) / a.count;
        // From here on the whole row has been read, by all waves: the sum may take the place of x or of the residual.
        if (a.res) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (there[k]) store_packet<AROUND, T, P>(static_cast<T*>(a.sum) + out + at[k], h[k]);
        }
        s = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < P; ++e) {
                h[k][e] -= mean;
                s = place.counts(k, e) ? fmaf(h[k][e], h[k][e], s) : s;
            }
        const float inv = rsqrtf(group.sum(s) / a.count + a.eps);
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int e = 0; e < P; ++e) h[k][e] = fmaf(h[k][e] * inv, w[k][e], b[k][e]);
            if (there[k]) store_packet<AROUND, T, P>(static_cast<T*>(a.y) + out + at[k], h[k]);
        }
        if (a.stats && group.lane == 0) *reinterpret_cast<float2*>(a.stats + 2 * row) = make_float2(mean, inv);
    }
}

template <typename T, int P, int K, bool WAVE, bool TAIL, bool AROUND>
__global__ __launch_bounds__(WAVE ? kThreads : 1024, WAVE ? 3 : 4) void layer_norm_backward(const LayerNormArgs a) {
    __shared__ float lds[64];
    extern __shared__ float sums[];  // WAVE: [waves][2][dim]
    Group<WAVE> group{};
    group.lds = lds;
    group.lanes = WAVE ? 1 << a.lanes_shift : blockDim.x;
    group.lane = WAVE ? threadIdx.x & (group.lanes - 1) : threadIdx.x;
    const int64_t units = WAVE ? (int64_t)gridDim.x * (kThreads >> a.lanes_shift) : gridDim.x;
    int64_t row = WAVE ? (int64_t)blockIdx.x * (kThreads >> a.lanes_shift) + (threadIdx.x >> a.lanes_shift) : blockIdx.x;
    const Places<P, K, TAIL> place(group.lane, group.lanes, a.dim);
    const auto& at = place.at;
    const auto& there = place.there;
    float w[K][P], dw[K][P], db[K][P];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        load_weights<P>(w[k], a.w, at[k], there[k], 1.f);
#pragma unroll
        for (int e = 0; e < P; ++e) dw[k][e] = db[k][e] = 0.f;
    }
    for (; row < a.rows; row += units) {
        const int64_t out = row * a.dim;
        const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
        const T* const gy = static_cast<const T*>(a.gy) + out;
        Packet<T, P> px[K], pg[K], ps[K];
#pragma unroll
        for (int k = 0; k < K; ++k) px[k].load(x + at[k], there[k]);
#pragma unroll
        for (int k = 0; k < K; ++k) pg[k].load(gy + at[k], there[k]);
        if (a.gs) {
#pragma unroll
            for (int k = 0; k < K; ++k) ps[k].load(static_cast<const T*>(a.gs) + out + at[k], there[k]);
        }
        const float2 stats = *reinterpret_cast<const float2*>(a.stats + 2 * row);
        const float mean = stats.x, inv = stats.y;
        float n[K][P], g[K][P], s = 0.f, t = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < P; ++e) {
                n[k][e] = (px[k].at(e) - mean) * inv;
                const float from = pg[k].at(e);  // 0 where there is no element
                const bool counts = place.counts(k, e);
                dw[k][e] = counts ? fmaf(from, n[k][e], dw[k][e]) : dw[k][e];
                db[k][e] += from;  // not read where the element is the packet's before
                g[k][e] = from * w[k][e];
                s += !TAIL || counts ? g[k][e] : 0.f;
                t = counts ? fmaf(g[k][e], n[k][e], t) : t;
            }
        group.sum2(s, t);
        s /= a.count;
        t /= a.count;
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int e = 0; e < P; ++e) {
                g[k][e] = inv * (g[k][e] - s - n[k][e] * t);
                if (a.gs) g[k][e] += ps[k].at(e);
            }
            if (there[k]) store_packet<AROUND, T, P>(static_cast<T*>(a.y) + out + at[k], g[k]);
        }
    }
    if (!a.part) return;
    float* const part = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    if constexpr (!WAVE) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < P; ++e)
                if (place.counts(k, e)) {
                    part[at[k] + e] = dw[k][e];
                    part[a.dim + at[k] + e] = db[k][e];
                }
    } else {
        for (int o = group.lanes; o < 64; o <<= 1) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < P; ++e) {
                    dw[k][e] += __shfl_xor(dw[k][e], o, 64);
                    db[k][e] += __shfl_xor(db[k][e], o, 64);
                }
        }
        if ((int)(threadIdx.x & 63) < group.lanes) {
            float* const to = sums + (threadIdx.x >> 6) * 2 * a.dim;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < P; ++e)
                    if (place.counts(k, e)) {
                        to[at[k] + e] = dw[k][e];
                        to[a.dim + at[k] + e] = db[k][e];
                    }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < 2 * a.dim; d += kThreads) {
            float x = 0.f;
            for (int v = 0; v < kThreads / 64; ++v) x += sums[v * 2 * a.dim + d];
            part[d] = x;
        }
    }
}

// Sums of the workgroups' parts: kColumns columns a workgroup, its threads' slices of the
// parts in order.
__global__ __launch_bounds__(kAddThreads) void layer_norm_weights(const float* __restrict__ part, int parts, int dim,
                                                               float* dw, float* db) {
    constexpr int kSlices = kAddThreads / kColumns;
    __shared__ float sums[kSlices][kColumns];
    const int d = blockIdx.x * kColumns + threadIdx.x % kColumns, slice = threadIdx.x / kColumns;
    float s = 0.f;
    if (d < 2 * dim) {
#pragma unroll 8
        for (int p = slice; p < parts; p += kSlices) s += part[(int64_t)p * 2 * dim + d];
    }
    sums[slice][threadIdx.x % kColumns] = s;
    __syncthreads();
    if (slice == 0 && d < 2 * dim) {
        for (int i = 1; i < kSlices; ++i) s += sums[i][threadIdx.x];
        float* const to = d < dim ? dw : db;
        if (to) to[d < dim ? d : d - dim] = s;
    }
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

int64_t size_of(const ra_layer_norm_shape& s) { return s.dtype == RA_DTYPE_F32 ? 4 : 2; }

// An output in the place of an input row by row is fine (a row is read whole before any of it is written), any other
// overlap is not.
ra_status refuse_shared_rows(const ra_layer_norm_shape& s, std::initializer_list<Extent> outputs, const Extent& in, int64_t ld) {
    for (const Extent& o : outputs)
        if (overlap(o, in) && !(o.at == in.at && (s.rows <= 1 || ld == s.dim)))
            return fail(RA_ERR_INVALID_ARGUMENT, std::string("layer norm: ") + o.name + " overlaps " + in.name);
    return RA_OK;
}

// How a row lies in lanes: packets of P elements, K of them in a lane, groups of
// 1 << shift lanes (wave) or of `threads`.
struct Layout {
    int p, k, shift, threads, blocks;
    bool wave, tail;
};

// Packets of 16 bytes (single elements where a row has not one), as few in a lane as a wave
// needs.
Layout layout_of(const ra_layer_norm_shape& s, int most_blocks) {
    Layout l{};
    l.p = s.dtype == RA_DTYPE_F32 ? 4 : 8;
    if (s.dim < l.p) l.p = 1;
    l.tail = s.dim % l.p != 0;
    const int packets = (s.dim + l.p - 1) / l.p, most = kMaxLane / l.p;
    l.wave = packets <= 64 * most;
    l.k = 1;
    while (l.k < most && packets > 64 * l.k) l.k *= 2;
    if (l.wave) {
        while ((l.k << l.shift) < packets) ++l.shift;
        l.threads = kThreads;
    } else {
        l.k = 8 / l.p;  // 8 elements a lane up to 1,024 lanes: more rows in flight, no registers short
        if (packets > 1024 * l.k) l.k *= 2;
        l.threads = 128;
        while (l.threads * l.k < packets) l.threads *= 2;
    }
    const int64_t per = l.wave ? kThreads >> l.shift : 1;
    // Never more than min(rows, most_blocks): the workspace holds a part for each.
    l.blocks = static_cast<int>(std::min<int64_t>((s.rows + per - 1) / per, most_blocks));
    return l;
}

bool passes_caches(const ra_layer_norm_shape& s) {
    return s.rows * s.dim * (s.dtype == RA_DTYPE_F32 ? 4 : 2) > kAroundBytes;
}

// Workgroups of the backward pass that a CU holds at once, by their registers: with a
// few more, those would run alone at the end.
int resident(const Layout& l) {
    if (!l.wave) return 1024 / l.threads;
    const int elements = l.p * l.k;
    return elements <= 4 ? 8 : elements == 8 ? 5 : 3;
}

template <typename F>
void by_layout(int32_t dtype, const Layout& l, F f) {
    auto packets = [&](auto t, auto p, auto k) {
        auto tail = [&](auto wave) {
            if constexpr (decltype(p)::value > 1)
                if (l.tail) return f(t, p, k, wave, std::true_type());
            f(t, p, k, wave, std::false_type());
        };
        if (l.wave) tail(std::true_type());
        else if constexpr (decltype(p)::value * decltype(k)::value >= 8) tail(std::false_type());
    };
    auto of_type = [&](auto t) {
        constexpr int kPer = 16 / sizeof(t);
        using P = std::integral_constant<int, kPer>;
        using I1 = std::integral_constant<int, 1>;
        using I2 = std::integral_constant<int, 2>;
        using I4 = std::integral_constant<int, 4>;
        if (l.p == 1) return packets(t, I1(), I1());
        if constexpr (kPer == 4)
            if (l.k == 4) return packets(t, P(), I4());
        l.k == 1 ? packets(t, P(), I1()) : packets(t, P(), I2());
    };
    if (dtype == RA_DTYPE_F32) of_type(float());
    else if (dtype == RA_DTYPE_F16) of_type(f16_t());
    else of_type(bf16_t());
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
    if (reinterpret_cast<uintptr_t>(d_stats) % 8) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: stats must be 8-byte aligned");
    const int64_t size = ra::size_of(*s);
    const ra::Extent x = ra::rows_of("x", d_x, s->rows, s->dim, s->ldx, size);
    const ra::Extent residual = ra::rows_of("the residual", d_residual, s->rows, s->dim, s->ldr, size);
    const ra::Extent weight = ra::rows_of("weight", d_weight, 1, s->dim, 0, sizeof(float));
    const ra::Extent bias = ra::rows_of("bias", d_bias, 1, s->dim, 0, sizeof(float));
    const ra::Extent y = ra::rows_of("y", d_y, s->rows, s->dim, s->dim, size);
    const ra::Extent sum = ra::rows_of("the sum", d_sum, s->rows, s->dim, s->dim, size);
    const ra::Extent stats = ra::rows_of("stats", d_stats, s->rows, 2, 2, sizeof(float));
    RA_TRY(ra::refuse_overlap("layer norm", {y, sum}, {weight, bias}));
    RA_TRY(ra::refuse_overlap("layer norm", {stats}, {x, residual, weight, bias, y, sum}));
    RA_TRY(ra::refuse_shared_rows(*s, {y, sum}, x, s->ldx));
    RA_TRY(ra::refuse_shared_rows(*s, {y, sum}, residual, s->ldr));
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
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const ra::Layout l = ra::layout_of(*s, ra::kForwardBlocks);
    a.lanes_shift = l.shift;
    ra::by_layout(s->dtype, l, [&](auto t, auto p, auto k, auto wave, auto tail) {
        using T = decltype(t);
        constexpr int kPer = decltype(p)::value, kEach = decltype(k)::value;
        constexpr bool kWave = decltype(wave)::value, kTail = decltype(tail)::value;
        if (ra::passes_caches(*s)) ra::layer_norm_forward<T, kPer, kEach, kWave, kTail, true><<<l.blocks, l.threads, 0, st>>>(a);
        else ra::layer_norm_forward<T, kPer, kEach, kWave, kTail, false><<<l.blocks, l.threads, 0, st>>>(a);
    });
    RA_LAUNCH_CHECK("layer_norm");
    return RA_OK;
}

ra_status ra_layer_norm_workspace(const ra_layer_norm_shape* s, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: bytes is NULL");
    RA_TRY(ra::check(s));
    *bytes = s->rows == 0 ? 0 : std::min<int64_t>(s->rows, ra::kBackwardBlocks) * 2 * s->dim * (int64_t)sizeof(float);
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
    if (reinterpret_cast<uintptr_t>(d_stats) % 8) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: stats must be 8-byte aligned");
    if (bytes < need || (need && !d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: the workspace is too small");
    if (need && !ra::aligned16(d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "layer norm: the workspace must be 16-byte aligned");
    const int64_t size = ra::size_of(*s);
    const ra::Extent h = ra::rows_of("h", d_h, s->rows, s->dim, s->ldx, size);
    const ra::Extent weight = ra::rows_of("weight", d_weight, 1, s->dim, 0, sizeof(float));
    const ra::Extent stats = ra::rows_of("stats", d_stats, s->rows, 2, 2, sizeof(float));
    const ra::Extent grad_y = ra::rows_of("grad_y", d_grad_y, s->rows, s->dim, s->dim, size);
    const ra::Extent grad_sum = ra::rows_of("grad_sum", d_grad_sum, s->rows, s->dim, s->dim, size);
    const ra::Extent dx = ra::rows_of("dx", d_dx, s->rows, s->dim, s->dim, size);
    const ra::Extent dweight = ra::rows_of("dweight", d_dweight, 1, s->dim, 0, sizeof(float));
    const ra::Extent dbias = ra::rows_of("dbias", d_dbias, 1, s->dim, 0, sizeof(float));
    const ra::Extent workspace{"the workspace", d_workspace, static_cast<uint64_t>(need)};
    RA_TRY(ra::refuse_overlap("layer norm", {dx}, {weight, stats}));
    RA_TRY(ra::refuse_overlap("layer norm", {dweight, dbias, workspace}, {h, weight, stats, grad_y, grad_sum, dx}));
    RA_TRY(ra::refuse_shared_rows(*s, {dx}, h, s->ldx));
    RA_TRY(ra::refuse_shared_rows(*s, {dx}, grad_y, s->dim));
    RA_TRY(ra::refuse_shared_rows(*s, {dx}, grad_sum, s->dim));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    ra::LayerNormArgs a{};
    a.x = d_h;
    a.gy = d_grad_y;
    a.gs = d_grad_sum;
    a.w = d_weight;
    a.y = d_dx;
    a.stats = const_cast<float*>(d_stats);
    a.part = d_dweight || d_dbias ? static_cast<float*>(d_workspace) : nullptr;
    a.rows = s->rows;
    a.ldx = s->ldx;
    a.dim = s->dim;
    a.count = static_cast<float>(s->dim);
    ra::Layout l{};
    if (s->rows) {
        l = ra::layout_of(*s, ra::kBackwardBlocks);
        l.blocks = std::min(l.blocks, 256 * ra::resident(l));
        a.lanes_shift = l.shift;
        const size_t lds = l.wave && a.part ? (size_t)ra::kThreads / 64 * 2 * s->dim * sizeof(float) : 0;
        ra::by_layout(s->dtype, l, [&](auto t, auto p, auto k, auto wave, auto tail) {
            using T = decltype(t);
            constexpr int kPer = decltype(p)::value, kEach = decltype(k)::value;
            constexpr bool kWave = decltype(wave)::value, kTail = decltype(tail)::value;
            if (ra::passes_caches(*s)) ra::layer_norm_backward<T, kPer, kEach, kWave, kTail, true><<<l.blocks, l.threads, lds, st>>>(a);
            else ra::layer_norm_backward<T, kPer, kEach, kWave, kTail, false><<<l.blocks, l.threads, lds, st>>>(a);
        });
        RA_LAUNCH_CHECK("layer_norm backward");
    }
    if (d_dweight || d_dbias) {  // without rows the sums are empty
        ra::layer_norm_weights<<<(2 * s->dim + ra::kColumns - 1) / ra::kColumns, ra::kAddThreads, 0, st>>>(
            a.part, l.blocks, s->dim, d_dweight, d_dbias);
        RA_LAUNCH_CHECK("layer_norm_weights");
    }
    return RA_OK;
}

}  // extern "C"
