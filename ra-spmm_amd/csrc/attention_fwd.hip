// attention_fwd.hip — differential attention over neighbour lists, forward.
//
// A wave works on one piece of a row (at most 256 edges of it) for one block of
// heads.  Its lanes are edge slots x heads x 2 maps x LM lanes, so that a load
// instruction takes whole runs of the gathered k and v rows: a lane holds 8
// elements of its map's half of a key and NV of the head's value row.  One pass
// over the edges, two a slot at a time, with a running maximum and sum per (edge
// slot, head, map).  Until the last step of a row its final weights are not known, so
// the two maps' sums of v are kept apart; in the last step the slots' maxima and sums
// are joined first, and v is added once with its final weight p_0 / l_0 - lam p_1 / l_1.
// It is a row's only step where the list has no more edges than a step (8 on the
// power-law graph: 40 % of its rows, 11 % of its edges; 4 on the community graph: hardly
// a row), so most edges are added twice.  Pieces of a long row are joined by a second
// launch.
// (All keys of a row first, scores in LDS, then the values with final weights: fewer
// vector instructions, but two chains of gathers after one another; 1.35 against
// 1.03 ms at 512,000 rows of 32 in fp16.)
// Bound by the gathers of k and v where they miss the L2s: power-law graph of 1e6 rows,
// 23e6 edges of 512 bytes: 1.67 ms, 7.1 TB/s, what a bare gather from HBM reaches.  Where they
// hit, by the vector unit (two dot products, two exponentials and two scaled sums an edge,
// 93 % busy): community graph of 512,000 rows of 32, 1 KB an edge: 1.0 ms, 16.8 TB/s.
#include <type_traits>

#include "attention.hpp"

namespace ra {
namespace {

// Softmax state of a (slot, head): of the lane's own map, and v sums of both.
template <int NV>
struct State {
    float m, l;
    float own[NV], other[NV];
};

// Joins the slots of a piece and writes its state: [heads][2 maps][max, sum], then
// [heads][2 maps][value_dim].
template <int LM, int NV>
__device__ __forceinline__ void store_piece(const AttnArgs& a, const Unit& u, const Place<LM, NV>& p, State<NV>& s) {
    const float top = slots_max(s.m, p.slots);
    const float keep = s.m == -INFINITY ? 0.f : exp2_of(s.m - top), keep_x = other_map<LM>(keep);
    const float sum = slots_sum(s.l * keep, p.slots);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        s.own[i] *= keep;
        s.other[i] *= keep_x;
    }
    scatter_sum<NV>(s.own, p.slots);
    scatter_sum<NV>(s.other, p.slots);
    if (!p.live) return;
    float* base = a.partial + (int64_t)u.slot * a.q_heads * (2 * a.value_dim + 4);
    if (p.lm == 0 && p.es == 0) {
        float* ml = base + (p.head * 2 + p.map) * 2;
        ml[0] = top;
        ml[1] = sum;
    }
    float* acc = base + a.q_heads * 4 + (int64_t)p.head * 2 * a.value_dim + NV * p.l;
    store_scattered<float, NV, false>(acc + (p.map ? a.value_dim : 0), s.own, p.slots, p.vcount);
    store_scattered<float, NV, false>(acc + (p.map ? 0 : a.value_dim), s.other, p.slots, p.vcount);
}

template <typename T, int LM, int NV, int PB, bool WIDE>
__global__ __launch_bounds__(kAttnThreads) void attn_forward(const AttnArgs a) {
    const Unit u = unit_of(a);
    if (!u.live) return;
    const Place<LM, NV> p(a, u.head_block, a.q_heads);
    const int kv = p.head / a.group, slots = p.slots;
    const Gather<T, 8, PB, WIDE> k(a.k, (kv * 2 + p.map) * a.head_dim, 8 * p.lm, p.kcount);
    const Gather<T, NV, PB, WIDE> v(a.v, kv * a.value_dim, NV * p.l, p.vcount);

    const bool whole = u.slot < 0;
    const int64_t at = (int64_t)u.row * a.q_heads + p.head;
    T* const out = static_cast<T*>(a.out) + at * a.value_dim + NV * p.l;
    State<NV> s;
    s.m = -INFINITY;
    s.l = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s.own[i] = s.other[i] = 0.f;
    if (u.begin == u.end && whole) {
        if (!p.live) return;
        store_scattered<T, NV, PB == 16>(out, s.own, slots, p.vcount);
        if (a.stats && p.lm == 0 && p.es == 0) reinterpret_cast<float2*>(a.stats)[at * 2 + p.map] = make_float2(0.f, 0.f);
        return;
    }
    Edges<kDeep> now, next;
    if (u.begin < u.end) load_edges<false>(a, now, u.begin, u.end - u.begin, p.es, slots);
    Run<T, 8> q;
    load_run<T, 8, PB == 16>(
        q, static_cast<const T*>(a.q) + u.row * a.ldq + (int64_t)(p.head * 2 + p.map) * a.head_dim + 8 * p.lm, p.kcount);
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
        float score[DEEP], top = s.m;
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            score[d] = fmaf(lanes_sum<LM>(dot(q, kr[d])), a.scale2, now.add[d]);
            if (!live[d]) score[d] = -INFINITY;
            top = fmaxf(top, score[d]);  // a NaN score makes its weight NaN below
        }
        // No live edge so far: every weight is exp2(-inf) = 0.
        const float ref = top == -INFINITY ? 0.f : top;
        const float keep = exp2_of(s.m - ref);
        float w[DEEP], sum = s.l * keep;
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            w[d] = exp2_of(score[d] - ref);
            sum += w[d];
        }
        if (LAST && whole) {
            const float all = slots_max(top, slots);
            const float part = top == -INFINITY ? (sum == 0.f ? 0.f : sum) : exp2_of(top - all);
            const float total = slots_sum(sum * part, slots);
            const float il = total > 0.f ? 1.f / total : total;  // 0, or a NaN that stays
            const float f = (p.map == 0 ? il : -a.lam[p.head] * il) * part;
            float o[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) o[i] = 0.f;
            if (e0 != u.begin) {
                const float c = f * keep, cx = other_map<LM>(c);
#pragma unroll
                for (int i = 0; i < NV; ++i) o[i] = fmaf(s.own[i], c, s.other[i] * cx);
            }
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const float wf = w[d] * f, mix = wf + other_map<LM>(wf);
                float vf[NV];
                vr[d].to_float(vf);
#pragma unroll
                for (int i = 0; i < NV; ++i) o[i] = fmaf(mix, vf[i], o[i]);
            }
            scatter_sum<NV>(o, slots);
            if (p.live) {
                store_scattered<T, NV, PB == 16>(out, o, slots, p.vcount);
                if (a.stats && p.lm == 0 && p.es == 0)
                    reinterpret_cast<float2*>(a.stats)[at * 2 + p.map] = make_float2(all == -INFINITY ? 0.f : all, il);
            }
            return;
        }
        s.m = top;
        s.l = sum;
        if (e0 != u.begin) {
            const float keep_x = other_map<LM>(keep);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                s.own[i] *= keep;
                s.other[i] *= keep_x;
            }
        }
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const float wx = other_map<LM>(w[d]);
            float vf[NV];
            vr[d].to_float(vf);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                s.own[i] = fmaf(w[d], vf[i], s.own[i]);
                s.other[i] = fmaf(wx, vf[i], s.other[i]);
            }
        }
        if constexpr (!LAST) now = next;
    });
    if (whole) return;
    store_piece(a, u, p, s);
}

// Joins the pieces of a cut row: a workgroup per (row, head).  The pieces' weights
// are formed once, in LDS, for up to kJoinPieces of them at a time (a running maximum
// over those steps); the v sums then go over piece groups x value_dim threads.
constexpr int kJoinThreads = 256, kJoinPieces = 1024;

// A pair over the workgroup; `lds` is not read by others any more.
template <typename F>
__device__ __forceinline__ void join_reduce(float* x, float2* lds, F f) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        x[0] = f(x[0], __shfl_xor(x[0], off, 64));
        x[1] = f(x[1], __shfl_xor(x[1], off, 64));
    }
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = make_float2(x[0], x[1]);
    __syncthreads();
    const float2 a = lds[0], b = lds[1], c = lds[2], d = lds[3];
    x[0] = f(f(a.x, b.x), f(c.x, d.x));
    x[1] = f(f(a.y, b.y), f(c.y, d.y));
}

// AHEAD: values of a thread that are under way together with the maxima.
template <typename T, int AHEAD>
__global__ __launch_bounds__(kJoinThreads) void attn_forward_join(const AttnArgs a, const int4* __restrict__ splits) {
    __shared__ float weight[2][kJoinPieces], sums[2][kJoinThreads];
    __shared__ float2 tops[kJoinThreads / 64], totals[kJoinThreads / 64];
    const int head = blockIdx.x % a.q_heads, which = blockIdx.x / a.q_heads;
    const int4 sp = splits ? splits[which] : make_int4(which, 0, a.pieces, 0);
    const int64_t slot0 = splits ? sp.y : (int64_t)which * a.pieces;
    const int64_t stride = (int64_t)a.q_heads * (2 * a.value_dim + 4);
    const float* const first = a.partial + slot0 * stride;
    int width = 16;
    while (width < a.value_dim) width *= 2;  // at most 256
    const int part = threadIdx.x / width, parts = kJoinThreads / width, at = threadIdx.x & (width - 1);

    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, acc[2] = {0.f, 0.f};
    for (int i0 = 0; i0 < sp.z; i0 += kJoinPieces) {
        const int n = min(kJoinPieces, sp.z - i0);
        constexpr int kEach = kJoinPieces / kJoinThreads;
        float4 ml[kEach];  // max, sum of both maps
        float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = threadIdx.x + j * kJoinThreads;
            ml[j] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
            if (i < n) {
                const float* const x = first + (i0 + i) * stride + head * 4;
                ml[j] = make_float4(x[0], x[1], x[2], x[3]);
            }
            most[0] = fmaxf(most[0], ml[j].x);
            most[1] = fmaxf(most[1], ml[j].z);
        }
        const float* const v = first + i0 * stride + a.q_heads * 4 + (int64_t)head * 2 * a.value_dim + min(at, a.value_dim - 1);
        float ahead[AHEAD + 1][2];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int64_t i = min(part + u * parts, n - 1);
            ahead[u][0] = v[i * stride];
            ahead[u][1] = v[i * stride + a.value_dim];
        }
        join_reduce(most, tops, [](float x, float y) { return fmaxf(x, y); });
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const float now = fmaxf(top[m], most[m]);
            const float ref = now == -INFINITY ? 0.f : now, keep = exp2_of(top[m] - ref);
            sum[m] *= keep;  // of the thread's pieces
            acc[m] *= keep;
            top[m] = now;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const float w = exp2_of((m == 0 ? ml[j].x : ml[j].z) - ref);
                weight[m][threadIdx.x + j * kJoinThreads] = w;
                sum[m] = fmaf(m == 0 ? ml[j].y : ml[j].w, w, sum[m]);
            }
        }
        __syncthreads();
        if (at < a.value_dim) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = part + u * parts;
                if (i < n) {
                    acc[0] = fmaf(ahead[u][0], weight[0][i], acc[0]);
                    acc[1] = fmaf(ahead[u][1], weight[1][i], acc[1]);
                }
            }
#pragma unroll 8
            for (int i = part + AHEAD * parts; i < n; i += parts) {
                acc[0] = fmaf(v[i * stride], weight[0][i], acc[0]);
                acc[1] = fmaf(v[i * stride + a.value_dim], weight[1][i], acc[1]);
            }
        }
        __syncthreads();  // before the next step's weights
    }
    sums[0][threadIdx.x] = acc[0];
    sums[1][threadIdx.x] = acc[1];
    join_reduce(sum, totals, [](float x, float y) { return x + y; });
    if (part != 0 || at >= a.value_dim) return;
    float il[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        for (int x = 1; x < parts; ++x) acc[m] += sums[m][x * width + at];
        il[m] = sum[m] > 0.f ? 1.f / sum[m] : sum[m];  // 0, or a NaN that stays
    }
    const int64_t to = (int64_t)sp.x * a.q_heads + head;
    const float o = sum[0] == 0.f ? 0.f : acc[0] * il[0] - a.lam[head] * il[1] * acc[1];
    static_cast<T*>(a.out)[to * a.value_dim + at] = (T)o;
    if (a.stats && at == 0)
        reinterpret_cast<float4*>(a.stats)[to] =
            make_float4(top[0] == -INFINITY ? 0.f : top[0], il[0], top[1] == -INFINITY ? 0.f : top[1], il[1]);
}

}  // namespace

ra_status attn_forward_launch(int32_t dtype, const AttnLayout& l, const AttnArgs& a, hipStream_t st) {
    return attn_launches(a, [&](const AttnArgs& part, unsigned blocks) {
        RA_ATTN_DISPATCH(attn_forward, dtype, l, dim3(blocks), st, part);
        RA_LAUNCH_CHECK("attn_forward");
        return RA_OK;
    });
}

ra_status attn_forward_join_launch(int32_t dtype, const AttnArgs& a, const int4* splits, int64_t n, hipStream_t st) {
    // Workgroups that are all resident wait for their loads: 8 of them ahead (4 rows of 6,000 edges, 8 heads: 6.8
    // against 9.5 us).  More are bound by the loads, and most of them have 2 or 3 pieces (power-law graph: 76 against
    // 103 us with 8 ahead).
    constexpr int64_t kResident = 2048;
    return join_launches(n, a.q_heads, [&](int first, dim3 grid) {
        AttnArgs part = a;
        const int4* const rows = splits ? splits + first : nullptr;
        if (!splits) {  // row 0 of the launch
            part.partial += (int64_t)first * a.pieces * a.q_heads * (2 * a.value_dim + 4);
            part.out = static_cast<char*>(a.out) + (int64_t)first * a.q_heads * a.value_dim * (dtype == RA_DTYPE_F32 ? 4 : 2);
        }
        const auto go = [&](auto tag) {
            using T = decltype(tag);
            if (n * a.q_heads <= kResident) attn_forward_join<T, 8><<<grid, kJoinThreads, 0, st>>>(part, rows);
            else attn_forward_join<T, 0><<<grid, kJoinThreads, 0, st>>>(part, rows);
        };
        if (dtype == RA_DTYPE_F32) go(float{});
        else if (dtype == RA_DTYPE_F16) go(f16_t{});
        else go(bf16_t{});
        RA_LAUNCH_CHECK("attn_forward_join");
        return RA_OK;
    });
}

}  // namespace ra
