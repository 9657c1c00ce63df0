// attention_bwd_cols.hip — backward pass of the graph attention over its columns:
// dk and dv, from the transposed lists.
//
// A wave works on one piece of a column's list for one block of key/value heads;
// per edge it gathers the row's q, dout and record (maximum, 1/sum and delta of both
// maps), and forms the weights again:
//     dk += scale * c p (dp - delta) q,   dv += (p_0 - lam p_1) dout
// A key/value head's query heads are taken one after another, into the same sums:
// nothing is added atomically, and the order is fixed.  Bound by the gathers: power-law
// graph of 1e6 rows, 23e6 edges of 640 bytes: 1.88 ms, 7.9 TB/s.
#include <type_traits>

#include "attention.hpp"

namespace ra {
namespace {

// ONE: a key/value head has one query head.
template <typename T, int LM, int NV, int PB, bool WIDE, bool ONE>
__device__ __forceinline__ void attn_cols(const AttnArgs& a) {
    const Unit u = unit_of(a);
    if (!u.live) return;
    const Place<LM, NV> p(a, u.head_block, a.kv_heads);
    const int slots = p.slots;
    float dk[8], dv[NV];
    Run<T, 8> k;
    load_run<T, 8, PB == 16>(
        k, static_cast<const T*>(a.k) + u.row * a.ldk + (int64_t)(p.head * 2 + p.map) * a.head_dim + 8 * p.lm, p.kcount);
    Run<T, NV> v;
    load_run<T, NV, PB == 16>(v, static_cast<const T*>(a.v) + u.row * a.ldv + (int64_t)p.head * a.value_dim + NV * p.l,
                              p.vcount);
#pragma unroll
    for (int i = 0; i < 8; ++i) dk[i] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) dv[i] = 0.f;

    // Of the first of the head's query heads; the others lie `sub` strides further on.
    const int first = ONE ? p.head : p.head * a.group;
    const Gather<T, 8, PB, WIDE> q(a.q, (first * 2 + p.map) * a.head_dim, 8 * p.lm, p.kcount);
    const Gather<T, NV, PB, WIDE> g(a.grad, first * a.value_dim, NV * p.l, p.vcount);
    const uint64_t record_first = first * a.record_head + p.map * sizeof(float4);
    const float lam = a.lam[first];

    Edges<kDeep> now, next;
    if (u.begin < u.end) load_edges<true>(a, now, u.begin, u.end - u.begin, p.es, slots);
    over_edges(u.begin, u.end, slots, [&](auto deep, auto is_last, int e0) {
        constexpr int DEEP = decltype(deep)::value;
        constexpr bool LAST = decltype(is_last)::value;
        if constexpr (!LAST) load_edges<true>(a, next, e0 + kDeep * slots, u.end - e0 - kDeep * slots, p.es, slots);
        bool live[DEEP];
        close_edges<DEEP, LAST>(a, now, live, u.end - e0, p.es, slots);
        for (int sub = 0; sub < (ONE ? 1 : a.group); ++sub) {
            const char* const record = reinterpret_cast<const char*>(a.record) + sub * a.record_head;
            Run<T, 8> qr[DEEP];
            Run<T, NV> gr[DEEP];
            float4 st[DEEP];  // maximum, 1 / sum, delta
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                q.load(qr[d], now.other[d], a.q_pitch, sub * 2 * a.head_dim * (int)sizeof(T));
                g.load(gr[d], now.other[d], a.g_pitch, sub * a.value_dim * (int)sizeof(T));
                if constexpr (WIDE)
                    st[d] = *reinterpret_cast<const float4*>(record + (uint64_t)now.other[d] * a.record_row + record_first);
                else
                    st[d] = *reinterpret_cast<const float4*>(record + (__umul24(now.other[d], a.record_row) +
                                                                       static_cast<uint32_t>(record_first)));
            }
            float c = p.map == 0 ? 1.f : -lam;
            if (sub > 0) c = p.map == 0 ? 1.f : -a.lam[first + sub];
            __builtin_amdgcn_sched_barrier(0);
            if (LAST || a.ragged || a.bias) {
#pragma unroll
                for (int d = 0; d < DEEP; ++d) {
                    q.mask(qr[d], live[d]);
                    g.mask(gr[d], live[d]);
                }
            }
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const float t = lanes_sum<LM>(dot(k, qr[d])), dp = lanes_sum<2 * LM>(dot(v, gr[d]));
                float w = c * exp2_of(fmaf(t, a.scale2, now.add[d]) - st[d].x) * st[d].y;
                float ds = w * (dp - st[d].z);
                if (!live[d]) w = ds = 0.f;
                const float mix = w + other_map<LM>(w);
                float qf[8], gf[NV];
                qr[d].to_float(qf);
                gr[d].to_float(gf);
#pragma unroll
                for (int i = 0; i < 8; ++i) dk[i] = fmaf(ds, qf[i], dk[i]);
#pragma unroll
                for (int i = 0; i < NV; ++i) dv[i] = fmaf(mix, gf[i], dv[i]);
            }
        }
        if constexpr (!LAST) now = next;
    });
    scatter_sum<8>(dk, slots);
    scatter_sum<NV>(dv, slots);
    if (!p.live) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) dk[i] *= a.scale;
    if (u.slot >= 0) {  // [heads][2 maps][head_dim], then [heads][value_dim]
        float* const base = a.partial + (int64_t)u.slot * a.kv_heads * (2 * a.head_dim + a.value_dim);
        store_scattered<float, 8, false>(base + (int64_t)(p.head * 2 + p.map) * a.head_dim + 8 * p.lm, dk, slots, p.kcount);
        store_scattered<float, NV, false>(
            base + (int64_t)a.kv_heads * 2 * a.head_dim + (int64_t)p.head * a.value_dim + NV * p.l, dv, slots, p.vcount);
        return;
    }
    const int64_t at = (int64_t)u.row * a.kv_heads + p.head;
    store_scattered<T, 8, PB == 16>(static_cast<T*>(a.out) + (at * 2 + p.map) * a.head_dim + 8 * p.lm, dk, slots, p.kcount);
    store_scattered<T, NV, PB == 16>(static_cast<T*>(a.out2) + at * a.value_dim + NV * p.l, dv, slots, p.vcount);
}

template <typename T, int LM, int NV, int PB, bool WIDE>
__global__ __launch_bounds__(kAttnThreads) void attn_cols_one(const AttnArgs a) {
    attn_cols<T, LM, NV, PB, WIDE, true>(a);
}
template <typename T, int LM, int NV, int PB, bool WIDE>
__global__ __launch_bounds__(kAttnThreads) void attn_cols_many(const AttnArgs a) {
    attn_cols<T, LM, NV, PB, WIDE, false>(a);
}

// Joins a cut column's pieces: plain sums of every element, in order.  Threads are
// four piece groups x 64 elements.
template <typename T>
__global__ __launch_bounds__(256) void attn_cols_join(const AttnArgs a, const int4* __restrict__ splits, int blocks_per) {
    __shared__ float sum[256];
    const int4 sp = splits[blockIdx.x / blocks_per];
    const int keys = a.kv_heads * 2 * a.head_dim, width = keys + a.kv_heads * a.value_dim;
    const int at = (blockIdx.x % blocks_per) * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
    float x = 0.f;
    if (at < width) {
        const float* const base = a.partial + (int64_t)sp.y * width + at;
#pragma unroll 4
        for (int s = part; s < sp.z; s += 4) x += base[(int64_t)s * width];
    }
    sum[threadIdx.x] = x;
    __syncthreads();
    if (part != 0 || at >= width) return;
    x = x + sum[64 + at % 64] + sum[128 + at % 64] + sum[192 + at % 64];
    if (at < keys) static_cast<T*>(a.out)[(int64_t)sp.x * keys + at] = (T)x;
    else static_cast<T*>(a.out2)[(int64_t)sp.x * (width - keys) + at - keys] = (T)x;
}

}  // namespace

ra_status attn_cols_launch(int32_t dtype, const AttnLayout& l, const AttnArgs& a, hipStream_t st) {
    // Without the loop over a head's query heads: power-law graph of 1e6 rows 1.88 against 2.04 ms, social graph of
    // 50,000 rows of 80 472 against 504 us.
    return attn_launches(a, [&](const AttnArgs& part, unsigned blocks) {
        if (a.group == 1) RA_ATTN_DISPATCH(attn_cols_one, dtype, l, dim3(blocks), st, part);
        else RA_ATTN_DISPATCH(attn_cols_many, dtype, l, dim3(blocks), st, part);
        RA_LAUNCH_CHECK("attn_cols");
        return RA_OK;
    });
}

ra_status attn_cols_join_launch(int32_t dtype, const AttnArgs& a, const int4* splits, int64_t n, hipStream_t st) {
    const int per = (a.kv_heads * (2 * a.head_dim + a.value_dim) + 63) / 64;
    return join_launches(n, per, [&](int first, dim3 grid) {
        if (dtype == RA_DTYPE_F32) attn_cols_join<float><<<grid, 256, 0, st>>>(a, splits + first, per);
        else if (dtype == RA_DTYPE_F16) attn_cols_join<f16_t><<<grid, 256, 0, st>>>(a, splits + first, per);
        else attn_cols_join<bf16_t><<<grid, 256, 0, st>>>(a, splits + first, per);
        RA_LAUNCH_CHECK("attn_cols_join");
        return RA_OK;
    });
}

}  // namespace ra
