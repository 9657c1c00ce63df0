// head_norm.hip — RMS norm of every query and key head with the position rotation
// in the same pass, forward and backward.
//
//     n = x * r, r = rsqrt(mean(x^2) + eps);  y = R(position) (n * w)
//     g' = R^T g;  dw = sum g' n;  dx = r (w g' - n * mean(w g' n))
//
// Bound by memory: the forward pass reads and writes every element once, the
// backward pass reads x and g and writes dx.  A lane holds P coordinate pairs of a
// head, so that the rotation needs no exchange: two runs of P elements, R/2 apart in
// the half layout, side by side in the interleaved one (and past the rotated part).
// r needs one sum over the head's lanes.  Workgroups stay on one of q and k and
// stride over its heads, with the weights (and the sums of dw) in registers.
// Measured: 1e6 rows of 8 + 8 heads of 16 in bf16, cut out of one projection: forward 216 us
// (1.02 GB, 4.7 TB/s), backward 335 (1.54 GB, 4.6); a large copy reaches 5.1.  150,000 rows of 12 + 4
// heads of 20 in fp32, 12 of each head rotated, a table row per position: 85 and 137 us (4.6 and
// 4.2 TB/s).  One row: 3 us on the GPU.
#include <algorithm>
#include <type_traits>

#include "ra_internal.hpp"
#include "vector_run.hpp"

namespace ra {
namespace {

constexpr int kThreads = 256;

struct NormArgs {
    const void *x[2], *g[2];
    void* y[2];
    const float* w[2];
    float* dw;          // partial sums [workgroup][head_dim]
    const float2* table;  // [positions][rot / 2] (cos, sin)
    const int32_t* pos;
    int64_t ld[2];
    int32_t heads[2];
    uint32_t units[2];  // rows * heads
    int32_t blocks_q;
    int32_t dim, rot, positions, lanes_shift;
    bool half;
    bool table_packets;  // rows of the table are whole aligned 16-byte packets
    float eps, inv_dim;
};

// Where a lane's two runs start, and how many of their elements exist.  Half
// layout: lanes of the rotated part first, then lanes of 2 P elements that are only
// scaled.  `pair`: the first pair of the table, rot / 2 where there is none.
template <int P>
struct Runs {
    int a, b, na, nb, pair;
    bool apart;
    __device__ __forceinline__ Runs(const NormArgs& n, int lane) {
        const int rotated = n.half ? (n.rot / 2 + P - 1) / P : 0;
        apart = lane < rotated;
        if (apart) {
            pair = a = lane * P;
            b = a + n.rot / 2;
            na = nb = min(P, n.rot / 2 - a);
        } else {
            a = n.half ? n.rot + (lane - rotated) * 2 * P : lane * 2 * P;
            b = a + P;
            na = max(0, min(P, n.dim - a));
            nb = max(0, min(P, n.dim - b));
            pair = n.half ? n.rot / 2 : lane * P;
        }
    }
};

// Row of the table, -1 outside of it.
__device__ __forceinline__ int64_t table_row(const NormArgs& n, int64_t position) {
    return position >= 0 && position < n.positions ? position : -1;
}
// The table's entries for a lane's pairs (those past the rotated part are not used).
// Two pairs a load where rows of the table are whole 16-byte packets.
template <int P>
__device__ __forceinline__ void load_angles(const NormArgs& n, const Runs<P>& r, int64_t at, float2* turn) {
    const float2* const t = n.table + max(at, (int64_t)0) * (n.rot / 2);
    const int last = n.rot / 2 - 1;
    if (n.table_packets) {
        const float4* const t4 = reinterpret_cast<const float4*>(t);
#pragma unroll
        for (int i = 0; i < P; i += 2) {
            const float4 x = t4[min(r.pair + i, last) / 2];
            turn[i] = make_float2(x.x, x.y);
            turn[i + 1] = make_float2(x.z, x.w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) turn[i] = t[min(r.pair + i, last)];
    }
}
// Their cosines and sines; pairs past the rotated part stay as they are, and a
// position outside of the table gives NaN.
template <int P>
__device__ __forceinline__ void angles(const NormArgs& n, const Runs<P>& r, const float2* turn, bool inside, float* c,
                                       float* s) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const bool rotated = r.pair + i < n.rot / 2;
        c[i] = !rotated ? 1.f : inside ? turn[i].x : __builtin_nanf("");
        s[i] = !rotated ? 0.f : inside ? turn[i].y : __builtin_nanf("");
    }
}

// (f, s) -> (f c - s si, f si + s c) for the pairs of two runs.  Coordinates that are
// not rotated are not mixed, by factors of 1 and 0 either: what is inf or NaN at one
// of them stays there.
template <int P>
__device__ __forceinline__ void rotate(const NormArgs& n, const Runs<P>& r, float* a, float* b, const float* c,
                                       const float* s, float sign) {
    if (r.apart) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float x = a[i], y = b[i], si = sign * s[i];
            a[i] = x * c[i] - y * si;
            b[i] = x * si + y * c[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float& fx = 2 * i < P ? a[2 * i] : b[2 * i - P];
            float& fy = 2 * i + 1 < P ? a[2 * i + 1] : b[2 * i + 1 - P];
            const float x = fx, y = fy, si = sign * s[i];
            const bool rotated = r.pair + i < n.rot / 2;
            fx = rotated ? x * c[i] - y * si : x;
            fy = rotated ? x * si + y * c[i] : y;
        }
    }
}

__device__ __forceinline__ float head_sum(float x, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}

template <typename T, int P, bool VEC, bool BACK>
__global__ __launch_bounds__(kThreads) void head_norm(const NormArgs n) {
    const int side = (int)blockIdx.x >= n.blocks_q;
    const uint32_t blocks = side ? gridDim.x - n.blocks_q : n.blocks_q, block = side ? blockIdx.x - n.blocks_q : blockIdx.x;
    const uint32_t thread = block * kThreads + threadIdx.x;
    const int lanes = 1 << n.lanes_shift;
    const Runs<P> r(n, thread & (lanes - 1));
    const uint32_t heads = n.heads[side], units = n.units[side], step = blocks * (kThreads >> n.lanes_shift);
    float wa[P], wb[P], da[P], db[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        wa[i] = i < r.na ? n.w[side][r.a + i] : 0.f;
        wb[i] = i < r.nb ? n.w[side][r.b + i] : 0.f;
        da[i] = db[i] = 0.f;
    }
    for (uint32_t unit = thread >> n.lanes_shift; unit < units; unit += step) {
        const uint32_t row = unit / heads, head = unit - row * heads;
        int64_t at = row;
        if (n.rot && n.pos) at = n.pos[row];
        const T* const x = static_cast<const T*>(n.x[side]) + row * n.ld[side] + (int64_t)head * n.dim;
        const int64_t out = (int64_t)unit * n.dim;
        Run<T, P> ra, rb, ga, gb;
        load_run<T, P, VEC>(ra, x + r.a, r.na);
        load_run<T, P, VEC>(rb, x + r.b, r.nb);
        if constexpr (BACK) {
            const T* const g = static_cast<const T*>(n.g[side]) + out;
            load_run<T, P, VEC>(ga, g + r.a, r.na);
            load_run<T, P, VEC>(gb, g + r.b, r.nb);
        }
        float2 turn[P];
        at = table_row(n, at);
        if (n.rot) load_angles<P>(n, r, at, turn);
        __builtin_amdgcn_sched_barrier(0);  // all loads before the first use
        float c[P], s[P], a[P], b[P];
        angles<P>(n, r, turn, at >= 0, c, s);
        ra.to_float(a);
        rb.to_float(b);
        float square = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) square = fmaf(a[i], a[i], fmaf(b[i], b[i], square));
        const float rms = rsqrtf(fmaf(head_sum(square, lanes), n.inv_dim, n.eps));
        if constexpr (!BACK) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                a[i] *= rms * wa[i];
                b[i] *= rms * wb[i];
            }
            rotate<P>(n, r, a, b, c, s, 1.f);
        } else {
            float fa[P], fb[P], inner = 0.f;
            ga.to_float(fa);
            gb.to_float(fb);
            rotate<P>(n, r, fa, fb, c, s, -1.f);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                a[i] *= rms;  // n
                b[i] *= rms;
                da[i] = fmaf(fa[i], a[i], da[i]);
                db[i] = fmaf(fb[i], b[i], db[i]);
                fa[i] *= wa[i];
                fb[i] *= wb[i];
                inner = fmaf(fa[i], a[i], fmaf(fb[i], b[i], inner));
            }
            inner = head_sum(inner, lanes) * n.inv_dim;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                a[i] = rms * (fa[i] - a[i] * inner);
                b[i] = rms * (fb[i] - b[i] * inner);
            }
        }
        T* const y = static_cast<T*>(n.y[side]) + out;
        store_run<T, P, VEC>(y + r.a, a, r.na);
        store_run<T, P, VEC>(y + r.b, b, r.nb);
    }
    if constexpr (BACK) {
        // dw of the workgroup: a wave's lanes of one place by shuffles, the waves in
        // order.
        extern __shared__ float sums[];  // [waves][dim]
        for (int o = lanes; o < 64; o <<= 1) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                da[i] += __shfl_xor(da[i], o, 64);
                db[i] += __shfl_xor(db[i], o, 64);
            }
        }
        if ((int)(threadIdx.x & 63) < lanes) {
            float* const to = sums + (threadIdx.x >> 6) * n.dim;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if (i < r.na) to[r.a + i] = da[i];
                if (i < r.nb) to[r.b + i] = db[i];
            }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < n.dim; d += kThreads) {
            float x = 0.f;
            for (int w = 0; w < kThreads / 64; ++w) x += sums[w * n.dim + d];
            n.dw[(int64_t)blockIdx.x * n.dim + d] = x;
        }
    }
}

// Sum of the workgroups' dw: a workgroup per (side, element), in a fixed order.
__global__ __launch_bounds__(kThreads) void head_norm_weights(const float* __restrict__ partial, int blocks_q, int blocks,
                                                              int dim, float* __restrict__ dwq, float* __restrict__ dwk) {
    __shared__ float part[kThreads / 64];
    const int side = blockIdx.x >= dim, d = blockIdx.x - side * dim;
    const int first = side ? blocks_q : 0, end = side ? blocks : blocks_q;
    float x = 0.f;
    for (int b = first + threadIdx.x; b < end; b += kThreads) x += partial[(int64_t)b * dim + d];
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) (side ? dwk : dwq)[d] = part[0] + part[1] + part[2] + part[3];
}

constexpr int kMaxDim = 256;
constexpr int kMaxBlocks = 2048;  // of both sides: 8 workgroups for every CU

struct Launch {
    NormArgs a{};
    int blocks = 0, p = 4;
    bool vec = false;
};

int lanes_of(const ra_norm_shape& s, int p) {
    if (s.layout == RA_ROTATION_HALF)
        return (s.rot_dim / 2 + p - 1) / p + (s.head_dim - s.rot_dim + 2 * p - 1) / (2 * p);
    return (s.head_dim + 2 * p - 1) / (2 * p);
}

// Workgroups of the two sides, in proportion to their heads.
void blocks_of(const ra_norm_shape& s, int p, int32_t& q, int32_t& both, int& shift) {
    shift = 0;
    while ((1 << shift) < lanes_of(s, p)) ++shift;
    const int64_t per = kThreads >> shift;  // heads of a workgroup
    const int64_t nq = ((int64_t)s.rows * s.q_heads + per - 1) / per, nk = ((int64_t)s.rows * s.k_heads + per - 1) / per;
    if (nq + nk <= kMaxBlocks) {
        q = static_cast<int32_t>(nq);
        both = static_cast<int32_t>(nq + nk);
        return;
    }
    both = kMaxBlocks;
    q = static_cast<int32_t>((int64_t)kMaxBlocks * s.q_heads / ((int64_t)s.q_heads + s.k_heads));
    if (s.q_heads && s.k_heads) q = std::min(std::max(q, 1), kMaxBlocks - 1);
}

// Pairs of a lane: as many as fill a 16-byte packet, or 4 (whole packets of 8 bytes
// where the sizes and addresses have them, else element by element).
Launch launch_of(const ra_norm_shape& s, const void* const x[2], const void* const g[2], void* const y[2],
                 const float* const w[2], const float* table, const int32_t* pos) {
    Launch l;
    NormArgs& a = l.a;
    const int64_t size = s.dtype == RA_DTYPE_F32 ? 4 : 2;
    const int64_t ld[2] = {s.ldq, s.ldk};
    const int32_t heads[2] = {s.q_heads, s.k_heads};
    for (int p = static_cast<int>(16 / size); p >= 4 && !l.vec; p /= 2) {
        const int64_t packet = p * size;
        l.p = p;
        l.vec = s.head_dim % p == 0 && (s.layout != RA_ROTATION_HALF || (s.rot_dim / 2) % p == 0);
        auto whole = [&](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % packet == 0; };
        for (int i = 0; i < 2; ++i)
            if (heads[i])
                l.vec = l.vec && whole(x[i]) && whole(y[i]) && (!g || whole(g[i])) && (s.rows <= 1 || ld[i] * size % packet == 0);
    }
    for (int i = 0; i < 2; ++i) {
        if (!heads[i]) continue;
        a.x[i] = x[i];
        a.g[i] = g ? g[i] : nullptr;
        a.y[i] = y[i];
        a.w[i] = w[i];
        a.ld[i] = ld[i];
        a.heads[i] = heads[i];
        a.units[i] = static_cast<uint32_t>((int64_t)s.rows * heads[i]);
    }
    blocks_of(s, l.p, a.blocks_q, l.blocks, a.lanes_shift);
    a.table = reinterpret_cast<const float2*>(table);
    a.pos = pos;
    a.dim = s.head_dim;
    a.rot = s.rot_dim;
    a.positions = s.positions;
    a.half = s.layout == RA_ROTATION_HALF;
    a.table_packets = aligned16(table) && s.rot_dim % 4 == 0;
    a.eps = s.eps;
    a.inv_dim = 1.f / static_cast<float>(s.head_dim);
    return l;
}

template <bool BACK>
void run(const Launch& l, int32_t dtype, hipStream_t st) {
    const size_t lds = BACK ? kThreads / 64 * l.a.dim * sizeof(float) : 0;
    auto go = [&](auto tag, auto p, auto vec) {
        head_norm<decltype(tag), decltype(p)::value, decltype(vec)::value, BACK><<<l.blocks, kThreads, lds, st>>>(l.a);
    };
    using Four = std::integral_constant<int, 4>;
    using Eight = std::integral_constant<int, 8>;
    auto by_type = [&](auto tag) {
        if (!l.vec) return go(tag, Four(), std::false_type());
        if constexpr (sizeof(tag) == 2)
            if (l.p == 8) return go(tag, Eight(), std::true_type());
        go(tag, Four(), std::true_type());
    };
    if (dtype == RA_DTYPE_F32) by_type(float());
    else if (dtype == RA_DTYPE_F16) by_type(f16_t());
    else by_type(bf16_t());
}

ra_status check(const ra_norm_shape* s) {
    if (!s) return fail(RA_ERR_INVALID_ARGUMENT, "head norm: shape is NULL");
    if (s->dtype != RA_DTYPE_F32 && s->dtype != RA_DTYPE_F16 && s->dtype != RA_DTYPE_BF16)
        return fail(RA_ERR_INVALID_ARGUMENT, "head norm: unknown dtype");
    if (s->layout != RA_ROTATION_HALF && s->layout != RA_ROTATION_INTERLEAVED)
        return fail(RA_ERR_INVALID_ARGUMENT, "head norm: unknown layout");
    if (s->rows < 0 || s->q_heads < 0 || s->k_heads < 0 || s->q_heads + (int64_t)s->k_heads == 0 || s->head_dim < 1)
        return fail(RA_ERR_INVALID_ARGUMENT, "head norm: bad sizes");
    if (s->rot_dim < 0 || s->rot_dim % 2 || s->rot_dim > s->head_dim)
        return fail(RA_ERR_INVALID_ARGUMENT, "head norm: rot_dim must be even and at most head_dim");
    if (s->head_dim > kMaxDim) return fail(RA_ERR_UNSUPPORTED, "head norm: head_dim is at most 256");
    if ((int64_t)s->rows * std::max(s->q_heads, s->k_heads) > INT32_MAX - (int64_t)kMaxBlocks * kThreads)
        return fail(RA_ERR_UNSUPPORTED, "head norm: too many heads (2^31 at most)");
    if (s->rows > 1 && ((s->q_heads && s->ldq < (int64_t)s->q_heads * s->head_dim) ||
                        (s->k_heads && s->ldk < (int64_t)s->k_heads * s->head_dim)))
        return fail(RA_ERR_INVALID_ARGUMENT, "head norm: rows overlap (a leading dimension is too small)");
    return RA_OK;
}

// A position outside of the table takes row 0 and gives NaN: there has to be a row.
ra_status check_table(const ra_norm_shape& s, const float* table) {
    if (s.rot_dim && !table) return fail(RA_ERR_INVALID_ARGUMENT, "head norm: NULL table");
    if (s.rot_dim && s.positions < 1) return fail(RA_ERR_INVALID_ARGUMENT, "head norm: the table is empty");
    return RA_OK;
}

}  // namespace
}  // namespace ra

using ra::fail;

extern "C" {

ra_status ra_head_norm(const ra_norm_shape* s, const void* d_q, const void* d_k, const float* d_wq, const float* d_wk,
                       const float* d_table, const int32_t* d_positions, void* d_out_q, void* d_out_k,
                       ra_stream_t stream) {
    RA_TRY(ra::check(s));
    if (s->rows == 0) return RA_OK;
    RA_TRY(ra::check_table(*s, d_table));
    if ((s->q_heads && (!d_q || !d_wq || !d_out_q)) || (s->k_heads && (!d_k || !d_wk || !d_out_k)))
        return fail(RA_ERR_INVALID_ARGUMENT, "head norm: NULL tensor");
    const void* x[2] = {d_q, d_k};
    void* y[2] = {d_out_q, d_out_k};
    const float* w[2] = {d_wq, d_wk};
    ra::run<false>(ra::launch_of(*s, x, nullptr, y, w, d_table, d_positions), s->dtype, reinterpret_cast<hipStream_t>(stream));
    RA_LAUNCH_CHECK("head_norm");
    return RA_OK;
}

ra_status ra_head_norm_workspace(const ra_norm_shape* s, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "head norm: bytes is NULL");
    RA_TRY(ra::check(s));
    *bytes = s->rows == 0 ? 0 : (int64_t)ra::kMaxBlocks * s->head_dim * (int64_t)sizeof(float);
    return RA_OK;
}

ra_status ra_head_norm_backward(const ra_norm_shape* s, const void* d_q, const void* d_k, const float* d_wq,
                                const float* d_wk, const float* d_table, const int32_t* d_positions,
                                const void* d_grad_q, const void* d_grad_k, void* d_dq, void* d_dk, float* d_dwq,
                                float* d_dwk, void* d_workspace, int64_t bytes, ra_stream_t stream) {
    int64_t need = 0;
    RA_TRY(ra_head_norm_workspace(s, &need));
    if ((s->q_heads && !d_dwq) || (s->k_heads && !d_dwk))
        return fail(RA_ERR_INVALID_ARGUMENT, "head norm: NULL weight gradient");
    if (s->rows > 0) RA_TRY(ra::check_table(*s, d_table));
    if (s->rows > 0 && ((s->q_heads && (!d_q || !d_wq || !d_grad_q || !d_dq)) ||
                        (s->k_heads && (!d_k || !d_wk || !d_grad_k || !d_dk))))
        return fail(RA_ERR_INVALID_ARGUMENT, "head norm: NULL tensor");
    if (bytes < need || (need && !d_workspace)) return fail(RA_ERR_INVALID_ARGUMENT, "head norm: the workspace is too small");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const void* x[2] = {d_q, d_k};
    const void* g[2] = {d_grad_q, d_grad_k};
    void* y[2] = {d_dq, d_dk};
    const float* w[2] = {d_wq, d_wk};
    ra::Launch l;
    if (s->rows > 0) {
        l = ra::launch_of(*s, x, g, y, w, d_table, d_positions);
        l.a.dw = static_cast<float*>(d_workspace);
        ra::run<true>(l, s->dtype, st);
        RA_LAUNCH_CHECK("head_norm backward");
    }
    // Without rows the sums are empty.
    const int sides = (s->q_heads > 0) + (s->k_heads > 0);
    float* const dwq = s->q_heads ? d_dwq : d_dwk;
    ra::head_norm_weights<<<sides * s->head_dim, ra::kThreads, 0, st>>>(
        static_cast<const float*>(d_workspace), s->q_heads ? l.a.blocks_q : l.blocks, l.blocks, s->head_dim, dwq, d_dwk);
    RA_LAUNCH_CHECK("head_norm_weights");
    return RA_OK;
}

}  // extern "C"
