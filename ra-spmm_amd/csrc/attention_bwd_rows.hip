// attention_bwd_rows.hip — backward pass of the graph attention over its rows:
// dq, the row sums that the column pass needs, d lam.
//
// With p the weights of a map, dp_j = dout . v_j and delta = sum_j p_j dp_j,
//     ds_j = c p_j (dp_j - delta)   (c = 1 for map 0, -lam for map 1)
//     dq   = scale * sum_j ds_j k_j = scale * c * (sum_j p_j dp_j k_j - delta sum_j p_j k_j)
// The second form needs one pass over the edges: delta is known at its end.  In a
// row's last step it is known before k is added, and the first form is used (for all
// of a row only where it has no more edges than a step).  The weights come from the forward pass' maxima and sums.  Lanes as
// in the forward pass; the pieces of a long row are plain sums.  It gathers what the
// forward pass does: power-law graph of 1e6 rows, 23e6 edges of 512 bytes: 1.72 ms, 6.9 TB/s.
#include <type_traits>

#include "attention.hpp"

namespace ra {
namespace {

// Six waves a SIMD for whole packets of 16-bit types (82 registers without the bound; power-law graph
// of 1e6 rows: 1.73 against 1.83 ms).
template <typename T, int LM, int NV, int PB, bool WIDE>
__global__ __launch_bounds__(kAttnThreads, PB == 16 ? (sizeof(T) == 2 ? 6 : 4) : 1) void attn_rows(const AttnArgs a) {
    const Unit u = unit_of(a);
    if (!u.live) return;
    const Place<LM, NV> p(a, u.head_block, a.q_heads);
    const int kv = p.head / a.group, slots = p.slots;
    const Gather<T, 8, PB, WIDE> k(a.k, (kv * 2 + p.map) * a.head_dim, 8 * p.lm, p.kcount);
    const Gather<T, NV, PB, WIDE> v(a.v, kv * a.value_dim, NV * p.l, p.vcount);

    Edges<kDeep> now, next;
    if (u.begin < u.end) load_edges<false>(a, now, u.begin, u.end - u.begin, p.es, slots);
    Run<T, 8> q;
    load_run<T, 8, PB == 16>(
        q, static_cast<const T*>(a.q) + u.row * a.ldq + (int64_t)(p.head * 2 + p.map) * a.head_dim + 8 * p.lm, p.kcount);
    Run<T, NV> g;
    load_run<T, NV, PB == 16>(
        g, static_cast<const T*>(a.grad) + ((int64_t)u.row * a.q_heads + p.head) * a.value_dim + NV * p.l, p.vcount);
    // The two-term instruction of bf16 too rounds downwards a little more often: every second lane's part of dp is formed
    // with its sign turned, so that over the lanes it does not add up (300,000 rows: dlam off by 1e-9 a row without).
    const uint32_t turned = std::is_same<T, bf16_t>::value && (threadIdx.x & 1) ? 0x80000000u : 0u;
    if constexpr (std::is_same<T, bf16_t>::value) {
#pragma unroll
        for (int i = 0; i < NV / 2; ++i) g.w[i] ^= turned | turned >> 16;
    }
    const int64_t at = ((int64_t)u.row * a.q_heads + p.head) * 2 + p.map;
    const float2 st = reinterpret_cast<const float2*>(a.stats)[at];
    const bool whole = u.slot < 0;
    float delta = 0.f, pdk[8], pk[8], dq[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) pdk[i] = pk[i] = dq[i] = 0.f;

    over_edges(u.begin, u.end, slots, [&](auto deep, auto is_last, int e0) {
        constexpr int DEEP = decltype(deep)::value;
        constexpr bool LAST = decltype(is_last)::value;
        Run<T, 8> kr[DEEP];
        Run<T, NV> vr[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            k.load(kr[d], now.other[d], a.k_pitch);
            v.load(vr[d], now.other[d], a.v_pitch);
        }
        if constexpr (!LAST) load_edges<false>(a, next, e0 + kDeep * slots, u.end - e0 - kDeep * slots, p.es, slots);
        __builtin_amdgcn_sched_barrier(0);
        bool live[DEEP];
        close_edges<DEEP, LAST>(a, now, live, u.end - e0, p.es, slots);
        if (LAST || a.ragged || a.bias) {
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                k.mask(kr[d], live[d]);
                v.mask(vr[d], live[d]);
            }
        }
        float w[DEEP], dp[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            w[d] = exp2_of(fmaf(lanes_sum<LM>(dot(q, kr[d])), a.scale2, now.add[d]) - st.x) * st.y;
            dp[d] = lanes_sum<2 * LM>(__uint_as_float(__float_as_uint(dot_rounded(g, vr[d])) ^ turned));
            if (!live[d]) w[d] = dp[d] = 0.f;
            delta = fmaf(w[d], dp[d], delta);
        }
        if (LAST && whole) {
            delta = slots_sum(delta, slots);
            if (e0 != u.begin) {
#pragma unroll
                for (int i = 0; i < 8; ++i) dq[i] = fmaf(-delta, pk[i], pdk[i]);
            }
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const float ds = w[d] * (dp[d] - delta);
                float kf[8];
                kr[d].to_float(kf);
#pragma unroll
                for (int i = 0; i < 8; ++i) dq[i] = fmaf(ds, kf[i], dq[i]);
            }
            return;
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const float wd = w[d] * dp[d];
            float kf[8];
            kr[d].to_float(kf);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                pdk[i] = fmaf(wd, kf[i], pdk[i]);
                pk[i] = fmaf(w[d], kf[i], pk[i]);
            }
        }
        if constexpr (!LAST) now = next;
    });
    if (whole) {
        scatter_sum<8>(dq, slots);
        if (!p.live) return;
        const float c = (p.map == 0 ? 1.f : -a.lam[p.head]) * a.scale;
#pragma unroll
        for (int i = 0; i < 8; ++i) dq[i] *= c;
        store_scattered<T, 8, PB == 16>(static_cast<T*>(a.out) + at * a.head_dim + 8 * p.lm, dq, slots, p.kcount);
        if (p.lm == 0 && p.es == 0) record_at(a, u.row, p.head)[p.map] = make_float4(st.x, st.y, delta, 0.f);
        return;
    }
    // A piece: [heads][2 maps][delta], then [heads][2 maps][2][head_dim].
    delta = slots_sum(delta, slots);
    scatter_sum<8>(pdk, slots);
    scatter_sum<8>(pk, slots);
    if (!p.live) return;
    float* const base = a.partial + (int64_t)u.slot * a.q_heads * (4 * a.head_dim + 2);
    if (p.lm == 0 && p.es == 0) base[p.head * 2 + p.map] = delta;
    float* const to = base + a.q_heads * 2 + (int64_t)(p.head * 2 + p.map) * 2 * a.head_dim + 8 * p.lm;
    store_scattered<float, 8, false>(to, pdk, slots, p.kcount);
    store_scattered<float, 8, false>(to + a.head_dim, pk, slots, p.kcount);
}

// Joins a cut row's pieces: a workgroup per (row, head).  Threads are piece groups x
// 64 .. 256 elements of the two maps' sums.
constexpr int kJoinThreads = 256;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void attn_rows_join(const AttnArgs a, const int4* __restrict__ splits) {
    __shared__ float first[kJoinThreads], second[kJoinThreads], sum[kJoinThreads];
    const int head = blockIdx.x % a.q_heads;
    const int4 sp = splits[blockIdx.x / a.q_heads];
    const int64_t stride = (int64_t)a.q_heads * (4 * a.head_dim + 2);
    const float* const base = a.partial + (int64_t)sp.y * stride;
    int width = 64;
    while (width < 2 * a.head_dim) width *= 2;  // at most 256
    const int part = threadIdx.x / width, parts = kJoinThreads / width, at = threadIdx.x & (width - 1);
    const bool live = at < 2 * a.head_dim;
    const int map = live && at >= a.head_dim, i = at - map * a.head_dim;
    float pdk = 0.f, pk = 0.f, delta = 0.f;
    if (live) {
        const float* const x = base + a.q_heads * 2 + (int64_t)(head * 2 + map) * 2 * a.head_dim + i;
#pragma unroll 4
        for (int s = part; s < sp.z; s += parts) {
            pdk += x[s * stride];
            pk += x[s * stride + a.head_dim];
            delta += base[s * stride + head * 2 + map];
        }
    }
    first[threadIdx.x] = pdk;
    second[threadIdx.x] = pk;
    sum[threadIdx.x] = delta;
    __syncthreads();
    if (part != 0 || !live) return;
    for (int x = 1; x < parts; ++x) {
        pdk += first[x * width + at];
        pk += second[x * width + at];
        delta += sum[x * width + at];
    }
    const int64_t to = ((int64_t)sp.x * a.q_heads + head) * 2 + map;
    const float c = (map == 0 ? 1.f : -a.lam[head]) * a.scale;
    static_cast<T*>(a.out)[to * a.head_dim + i] = (T)(c * (pdk - delta * pk));
    if (i == 0) {
        const float2 st = reinterpret_cast<const float2*>(a.stats)[to];
        record_at(a, sp.x, head)[map] = make_float4(st.x, st.y, delta, 0.f);
    }
}

// d lam[h] = -sum_i delta of map 1: a workgroup sums a run of rows for one head, then
// one workgroup the workgroups' sums, both in a fixed order.  In 64 bits: the terms
// cancel down to about their number's root, and fp32 sums would round at that size.
__device__ __forceinline__ double wave_sum(double x) {
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
    return x;
}
__global__ __launch_bounds__(256) void attn_lam_partial(const AttnArgs a, double* __restrict__ partial) {
    __shared__ double part[4];
    const int64_t per = ((int64_t)a.rows + gridDim.x - 1) / gridDim.x;
    const int64_t first = blockIdx.x * per, end = min(first + per, (int64_t)a.rows);
    const int h = blockIdx.y;
    double x = 0.;
#pragma unroll 4
    for (int64_t i = first + threadIdx.x; i < end; i += 256) x += record_at(a, i, h)[1].z;
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) partial[(int64_t)blockIdx.x * a.q_heads + h] = part[0] + part[1] + part[2] + part[3];
}
__global__ __launch_bounds__(64) void attn_lam_final(const double* __restrict__ partial, int blocks, int heads,
                                                     float* __restrict__ dlam) {
    const int h = blockIdx.x;
    double x = 0.;
    for (int b = threadIdx.x; b < blocks; b += 64) x += partial[(int64_t)b * heads + h];
    x = wave_sum(x);
    if (threadIdx.x == 0) dlam[h] = static_cast<float>(-x);
}

}  // namespace

ra_status attn_rows_launch(int32_t dtype, const AttnLayout& l, const AttnArgs& a, hipStream_t st) {
    return attn_launches(a, [&](const AttnArgs& part, unsigned blocks) {
        RA_ATTN_DISPATCH(attn_rows, dtype, l, dim3(blocks), st, part);
        RA_LAUNCH_CHECK("attn_rows");
        return RA_OK;
    });
}

ra_status attn_rows_join_launch(int32_t dtype, const AttnArgs& a, const int4* splits, int64_t n, hipStream_t st) {
    return join_launches(n, a.q_heads, [&](int first, dim3 grid) {
        if (dtype == RA_DTYPE_F32) attn_rows_join<float><<<grid, kJoinThreads, 0, st>>>(a, splits + first);
        else if (dtype == RA_DTYPE_F16) attn_rows_join<f16_t><<<grid, kJoinThreads, 0, st>>>(a, splits + first);
        else attn_rows_join<bf16_t><<<grid, kJoinThreads, 0, st>>>(a, splits + first);
        RA_LAUNCH_CHECK("attn_rows_join");
        return RA_OK;
    });
}

ra_status attn_lam_launch(const AttnArgs& a, double* partial, float* dlam, hipStream_t st) {
    attn_lam_partial<<<dim3(kLamBlocks, a.q_heads), 256, 0, st>>>(a, partial);
    RA_LAUNCH_CHECK("attn_lam_partial");
    attn_lam_final<<<a.q_heads, 64, 0, st>>>(partial, kLamBlocks, a.q_heads, dlam);
    RA_LAUNCH_CHECK("attn_lam_final");
    return RA_OK;
}

}  // namespace ra
