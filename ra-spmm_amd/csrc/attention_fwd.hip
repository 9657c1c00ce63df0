// attention_fwd.hip — differential attention over neighbour lists, forward.
//
// A wave works on one piece of a row (at most 256 edges of it) for one block of
// heads.  Its lanes are edge slots x heads x 2 maps x LM lanes, so that a load
// instruction takes whole runs of the gathered k and v rows: a lane holds 8
// elements of its map's half of a key and NV of the head's value row.  One pass
// over the edges with a running maximum and sum per (edge slot, head, map); the
// two maps' sums of v are kept apart, because their weights are only known at the
// end.  The slots are joined by shuffles, pieces of a long row by a second launch.
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

// Writes a finished row, or a piece's state to its slot:
// [heads][2 maps][max, sum], then [heads][2 maps][value_dim].
template <typename T, int LM, int NV, int PB>
__device__ __forceinline__ void finish(const AttnArgs& a, const Unit& u, const Place<LM, NV>& p, const State<NV>& s) {
    if (p.es != 0 || !p.live) return;
    if (u.slot >= 0) {
        float* base = a.partial + (int64_t)u.slot * a.q_heads * (2 * a.value_dim + 4);
        if (p.lm == 0) {
            float* ml = base + (p.head * 2 + p.map) * 2;
            ml[0] = s.m;
            ml[1] = s.l;
        }
        // Map 0's lanes hold map 0's sums in `own`.
        float* acc = base + a.q_heads * 4 + (int64_t)p.head * 2 * a.value_dim + NV * p.l;
        const bool first = p.map == 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i < p.vcount) {
                acc[i] = first ? s.own[i] : s.other[i];
                acc[a.value_dim + i] = first ? s.other[i] : s.own[i];
            }
        return;
    }
    const float il = s.l > 0.f ? 1.f / s.l : s.l == 0.f ? 0.f : s.l;  // NaN stays
    const float w = p.map == 0 ? il : -a.lam[p.head] * il;
    const float wx = other_map<LM>(w);
    float o[NV];
    // No edge left: zeros, whatever lam is.
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i] = s.l == 0.f ? 0.f : s.own[i] * w + s.other[i] * wx;
    store_run<T, NV, PB == 16>(static_cast<T*>(a.out) + ((int64_t)u.row * a.q_heads + p.head) * a.value_dim + NV * p.l, o,
                          p.vcount);
    if (a.stats && p.lm == 0)
        reinterpret_cast<float2*>(a.stats)[((int64_t)u.row * a.q_heads + p.head) * 2 + p.map] =
            make_float2(s.m == -INFINITY ? 0.f : s.m, il);
}

template <typename T, int LM, int NV, int PB>
__global__ __launch_bounds__(kAttnThreads) void attn_forward(const AttnArgs a) {
    const Unit u = unit_of(a);
    if (!u.live) return;
    const Place<LM, NV> p(a, u.head_block, a.q_heads);
    const int kv = p.head / a.group;
    const Gather<T, 8, PB> k(static_cast<const T*>(a.k) + (int64_t)(kv * 2 + p.map) * a.head_dim, 8 * p.lm, p.kcount);
    const Gather<T, NV, PB> v(static_cast<const T*>(a.v) + (int64_t)kv * a.value_dim, NV * p.l, p.vcount);

    Run<T, 8> q;
    load_run<T, 8, PB == 16>(
        q, static_cast<const T*>(a.q) + u.row * a.ldq + (int64_t)(p.head * 2 + p.map) * a.head_dim + 8 * p.lm, p.kcount);
    State<NV> s;
    s.m = -INFINITY;
    s.l = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s.own[i] = s.other[i] = 0.f;

    Edges now, next;
    if (u.begin < u.end) load_edges<false>(a, now, u.begin, u.end, p.es, p.slots);
    const int step_edges = kDeep * p.slots;
    for (int e0 = u.begin; e0 < u.end; e0 += step_edges) {
        Run<T, 8> kr[kDeep];
        Run<T, NV> vr[kDeep];
        const bool last = e0 + step_edges >= u.end;
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            k.load(kr[d], now.other[d], a.k_pitch);
            v.load(vr[d], now.other[d], a.v_pitch);
        }
        if (!last) load_edges<false>(a, next, e0 + step_edges, u.end, p.es, p.slots);
        __builtin_amdgcn_sched_barrier(0);
        if (last) close_edges(now, e0, u.end, p.es, p.slots);
        if (last || a.ragged || a.bias) {
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                k.mask(kr[d], now.add[d] != -INFINITY);
                v.mask(vr[d], now.add[d] != -INFINITY);
            }
        }
        float score[kDeep], top = s.m;
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            score[d] = fmaf(lanes_sum<LM>(dot(q, kr[d])), a.scale, now.add[d]);
            if (now.add[d] == -INFINITY) score[d] = -INFINITY;
            top = score[d] > top || score[d] != score[d] ? score[d] : top;  // a NaN stays
        }
        // All edges so far left out: every weight is 0, not exp(-inf + inf).
        const float ref = top == -INFINITY ? 0.f : top;
        const float keep = exp_of(s.m - ref), keep_x = other_map<LM>(keep);
        s.m = top;
        s.l *= keep;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            s.own[i] *= keep;
            s.other[i] *= keep_x;
        }
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            const float w = exp_of(score[d] - ref), wx = other_map<LM>(w);
            s.l += w;
            float vf[NV];
            vr[d].to_float(vf);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                s.own[i] = fmaf(w, vf[i], s.own[i]);
                s.other[i] = fmaf(wx, vf[i], s.other[i]);
            }
        }
        now = next;
    }
    for (int step = 32 / p.slots * 2; step < 64; step <<= 1) {
        const float m2 = __shfl_xor(s.m, step, 64);
        const float top = m2 > s.m || m2 != m2 ? m2 : s.m;
        const float ref = top == -INFINITY ? 0.f : top;
        const float keep = exp_of(s.m - ref), keep2 = exp_of(m2 - ref);
        const float keep_x = other_map<LM>(keep), keep2_x = other_map<LM>(keep2);
        s.l = s.l * keep + __shfl_xor(s.l, step, 64) * keep2;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            s.own[i] = s.own[i] * keep + __shfl_xor(s.own[i], step, 64) * keep2;
            s.other[i] = s.other[i] * keep_x + __shfl_xor(s.other[i], step, 64) * keep2_x;
        }
        s.m = top;
    }
    finish<T, LM, NV, PB>(a, u, p, s);
}

// Joins the pieces of a cut row: a workgroup per (row, head).  Its threads are
// piece groups x value_dim (padded to 64 at least); each group runs over its share
// of the pieces.
constexpr int kJoinThreads = 256;
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void attn_forward_join(const AttnArgs a, const int4* __restrict__ splits) {
    __shared__ float top_of[2][kJoinThreads / 64], sum_of[2][kJoinThreads / 64], acc_of[2][kJoinThreads];
    const int head = blockIdx.x % a.q_heads;
    int4 sp;
    if (splits) sp = splits[blockIdx.x / a.q_heads];
    else {
        const int row = blockIdx.x / a.q_heads;
        sp = make_int4(row, 0, a.pieces, 0);
    }
    const int64_t slot0 = splits ? sp.y : (int64_t)sp.x * a.pieces;
    const int n = sp.z;
    const int64_t stride = (int64_t)a.q_heads * (2 * a.value_dim + 4);
    const float* const ml = a.partial + slot0 * stride + head * 4;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;

    float top[2] = {-INFINITY, -INFINITY};
    for (int i = threadIdx.x; i < n; i += kJoinThreads)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const float x = ml[i * stride + 2 * m];
            top[m] = x > top[m] || x != x ? x : top[m];
        }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        for (int off = 32; off > 0; off >>= 1) {
            const float x = __shfl_xor(top[m], off, 64);
            top[m] = x > top[m] || x != x ? x : top[m];
        }
        if (lane == 0) top_of[m][wave] = top[m];
    }
    __syncthreads();
    float ref[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        top[m] = top_of[m][0];
        for (int w = 1; w < kJoinThreads / 64; ++w)
            top[m] = top_of[m][w] > top[m] || top_of[m][w] != top_of[m][w] ? top_of[m][w] : top[m];
        ref[m] = top[m] == -INFINITY ? 0.f : top[m];
    }
    float sum[2] = {0.f, 0.f};
    for (int i = threadIdx.x; i < n; i += kJoinThreads)
#pragma unroll
        for (int m = 0; m < 2; ++m) sum[m] += ml[i * stride + 2 * m + 1] * exp_of(ml[i * stride + 2 * m] - ref[m]);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        for (int off = 32; off > 0; off >>= 1) sum[m] += __shfl_xor(sum[m], off, 64);
        if (lane == 0) sum_of[m][wave] = sum[m];
    }
    // The v sums.
    int width = 64;
    while (width < a.value_dim) width *= 2;  // at most 256
    const int part = threadIdx.x / width, parts = kJoinThreads / width, at = threadIdx.x & (width - 1);
    float acc[2] = {0.f, 0.f};
    if (at < a.value_dim) {
        const float* const v = a.partial + slot0 * stride + a.q_heads * 4 + (int64_t)head * 2 * a.value_dim + at;
#pragma unroll 4
        for (int i = part; i < n; i += parts)
#pragma unroll
            for (int m = 0; m < 2; ++m)
                acc[m] = fmaf(v[i * stride + m * a.value_dim], exp_of(ml[i * stride + 2 * m] - ref[m]), acc[m]);
    }
    acc_of[0][threadIdx.x] = acc[0];
    acc_of[1][threadIdx.x] = acc[1];
    __syncthreads();
    if (part != 0 || at >= a.value_dim) return;
    float il[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        sum[m] = sum_of[m][0];
        for (int w = 1; w < kJoinThreads / 64; ++w) sum[m] += sum_of[m][w];
        for (int x = 1; x < parts; ++x) acc[m] += acc_of[m][x * width + at];
        il[m] = sum[m] > 0.f ? 1.f / sum[m] : sum[m] == 0.f ? 0.f : sum[m];
    }
    const int64_t to = (int64_t)sp.x * a.q_heads + head;
    const float o = sum[0] == 0.f ? 0.f : acc[0] * il[0] - a.lam[head] * il[1] * acc[1];
    static_cast<T*>(a.out)[to * a.value_dim + at] = (T)o;
    if (a.stats && at == 0)
        reinterpret_cast<float4*>(a.stats)[to] = make_float4(ref[0], il[0], ref[1], il[1]);
}

}  // namespace

ra_status attn_forward_launch(int32_t dtype, const AttnLayout& l, const AttnArgs& a, hipStream_t st) {
    unsigned blocks = 0;
    RA_TRY(attn_grid(a, blocks));
    if (blocks == 0) return RA_OK;
    RA_ATTN_DISPATCH(attn_forward, dtype, l, dim3(blocks), st, a);
    RA_LAUNCH_CHECK("attn_forward");
    return RA_OK;
}

ra_status attn_forward_join_launch(int32_t dtype, const AttnArgs& a, const int4* splits, int64_t n, hipStream_t st) {
    if (n == 0) return RA_OK;
    const int64_t blocks = n * a.q_heads;
    if (blocks > INT32_MAX) return fail(RA_ERR_UNSUPPORTED, "attention: too many rows");
    const dim3 grid((unsigned)blocks);
    if (dtype == RA_DTYPE_F32) attn_forward_join<float><<<grid, kJoinThreads, 0, st>>>(a, splits);
    else if (dtype == RA_DTYPE_F16) attn_forward_join<f16_t><<<grid, kJoinThreads, 0, st>>>(a, splits);
    else attn_forward_join<bf16_t><<<grid, kJoinThreads, 0, st>>>(a, splits);
    RA_LAUNCH_CHECK("attn_forward_join");
    return RA_OK;
}

}  // namespace ra
