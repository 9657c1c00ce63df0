// attention.hpp — what the graph-attention kernels share: the plan, the launch
// arguments, the lanes' layout and the row loads.
#pragma once

#include <type_traits>

#include "ra_internal.hpp"
#include "vector_run.hpp"

namespace ra {

// Edges of a piece: a row longer than this is cut into pieces that waves work on
// in parallel; their partial results are joined in a second launch.  Steps with pieces of
// 128, 256, 512 and 1024: skewed rows in fp32 1.92, 1.93, 2.01 and 2.18 ms (long pieces
// leave the last waves alone); social graph 1.29, 1.20, 1.20 and 1.21, power-law graph 5.61,
// 5.47, 5.43 and 5.52 (short ones are written and joined more often).
constexpr int kAttnPiece = 256;

// One side of a plan: the rows (or, transposed, the columns) as pieces.
struct AttnSide {
    const int32_t* ptr = nullptr;  // rows + 1
    const int32_t* idx = nullptr;  // the edge's other end
    const int32_t* edge = nullptr; // its number in CSR order (transposed side only)
    const int4* items = nullptr;   // row, first edge, end, slot or -1
    const int4* splits = nullptr;  // row, first slot, slots, 0
    int32_t rows = 0, num_items = 0, num_splits = 0;
    int64_t num_slots = 0;
    DeviceBuffer lists;
};

}  // namespace ra

struct ra_attn_plan {
    ra_attn_info info{};
    int device = 0;
    ra::AttnSide side[2];       // rows, columns
    ra::DeviceBuffer transposed;  // ptr, idx, edge of side[1]
    ra::DeviceBuffer partial, record;
};

namespace ra {

struct AttnArgs {
    // The pieces: a list, or (items == nullptr) `pieces` equal parts of every row.
    const int4* items;
    const int32_t* ptr;
    const int32_t* idx;
    const int32_t* edge;
    uint32_t num_units;   // pieces * head blocks (attn_check_units)
    uint32_t first_unit;  // of the launch
    int32_t pieces;       // per row, without a list
    int32_t head_blocks;  // waves that share a piece
    int32_t head_items;   // 0: a piece's waves are neighbours; else pieces, all of one head block's first
    int32_t hb_shift;     // log2 of the heads of a wave
    int32_t q_heads, kv_heads, group, head_dim, value_dim;
    int32_t rows;
    float scale, scale2;  // scale2 = scale * log2(e): scores are held in powers of two
    int64_t ldq, ldk, ldv;
    uint32_t q_pitch, k_pitch, v_pitch, g_pitch;  // bytes between rows
    bool ragged;          // some lane's run is not whole: loaded words are masked
    bool wide;            // gathered offsets need 64 bits
    const void *q, *k, *v, *grad;
    const float *lam, *bias;
    float* stats;    // [rows, q_heads, 2] (max in powers of two, 1 / sum)
    // What the column pass takes of a row and head: per map (max, 1 / sum, sum p dp, 0).
    float4* record;
    uint32_t record_row;  // distances in bytes: [rows][q_heads] or [q_heads][rows]
    int64_t record_head;
    void *out, *out2;
    float* partial;
};

// Lanes of a head: 2 maps x LM lanes of 8 head_dim elements each; value_dim goes
// over all 2 * LM of them, NV elements each.
struct AttnLayout {
    int lm;      // 1, 2, 4, 8, 16
    int nv;      // 4 or 8
    int packet;  // bytes that a lane loads at once: 16 (value rows of NV = 4: 4 elements), 4 or 2
    bool ragged;
    int hb_shift;
    int head_blocks;
};

struct AttnPtrs {
    const void *q, *k, *v, *grad;
    int64_t ldq, ldk, ldv, ldg;
};

// pieces: of the launch; by_head: attn_by_head.
AttnLayout attn_layout(const ra_attn_shape& s, int heads, const AttnPtrs& p, int64_t pieces, bool by_head);
bool attn_by_head(const ra_attn_shape& s, int64_t rows, int64_t gathered, int64_t nnz);
ra_status attn_check(const ra_attn_shape* s, int32_t M, int32_t K);

// Floats of a slot of partial results.
inline int64_t attn_forward_slot(const ra_attn_shape& s) { return (int64_t)s.q_heads * (2 * s.value_dim + 4); }
inline int64_t attn_row_slot(const ra_attn_shape& s) { return (int64_t)s.q_heads * (4 * s.head_dim + 2); }
inline int64_t attn_col_slot(const ra_attn_shape& s) { return (int64_t)s.kv_heads * (2 * s.head_dim + s.value_dim); }

// Threads of a launch: the runtime takes fewer than 2^32.  Larger ones are cut.
constexpr int64_t kMostThreads = (int64_t{1} << 32) - 1024;
constexpr int64_t kMostBlocks = kMostThreads / 256;
constexpr int64_t kMostUnits = kMostBlocks * 4;  // a wave each, four in a workgroup

// Units are numbered in 32 bits.  Checked before the first launch of a call.
inline ra_status attn_check_units(int64_t pieces, const AttnLayout& l) {
    if (pieces * l.head_blocks >= int64_t{1} << 32) return fail(RA_ERR_UNSUPPORTED, "attention: too many rows and heads");
    return RA_OK;
}

// launch(part of a, workgroups) for every part of the units.
template <typename F>
ra_status attn_launches(const AttnArgs& a, F launch) {
    AttnArgs part = a;
    for (int64_t first = 0; first < a.num_units; first += kMostUnits) {
        const int64_t units = a.num_units - first;
        part.first_unit = static_cast<uint32_t>(first);
        RA_TRY(launch(part, static_cast<unsigned>(((units < kMostUnits ? units : kMostUnits) + 3) / 4)));
    }
    return RA_OK;
}
// launch(first row, workgroups) for `n` rows of `each` workgroups.
template <typename F>
ra_status join_launches(int64_t n, int64_t each, F launch) {
    const int64_t most = kMostBlocks / each;
    for (int64_t first = 0; first < n; first += most) {
        const int64_t rows = n - first < most ? n - first : most;
        RA_TRY(launch(static_cast<int>(first), dim3(static_cast<unsigned>(rows * each))));
    }
    return RA_OK;
}
ra_status attn_forward_launch(int32_t dtype, const AttnLayout& l, const AttnArgs& a, hipStream_t st);
ra_status attn_rows_launch(int32_t dtype, const AttnLayout& l, const AttnArgs& a, hipStream_t st);
ra_status attn_cols_launch(int32_t dtype, const AttnLayout& l, const AttnArgs& a, hipStream_t st);
// Second launches: the cut rows' pieces (splits == nullptr: every row, a.pieces each).
ra_status attn_forward_join_launch(int32_t dtype, const AttnArgs& a, const int4* splits, int64_t n, hipStream_t st);
ra_status attn_rows_join_launch(int32_t dtype, const AttnArgs& a, const int4* splits, int64_t n, hipStream_t st);
ra_status attn_cols_join_launch(int32_t dtype, const AttnArgs& a, const int4* splits, int64_t n, hipStream_t st);
// d lam from the records; `partial` holds kLamBlocks * q_heads doubles.
constexpr int kLamBlocks = 128;
ra_status attn_lam_launch(const AttnArgs& a, double* partial, float* dlam, hipStream_t st);

// ------------------------------------------------------------- device side
constexpr int kAttnThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;
// A bias past kBiasLarge would leave float32's range in powers of two: from there on it goes half as fast.
constexpr float kBiasLarge = 1e38f;

// Lane moves.  Within a row of 16 lanes by data-parallel moves, between rows and
// halves by the swaps of two registers' rows and halves.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kRotate = 0x120;

struct Pair {
    float a, b;
};
// (x of the even rows, y of the even rows), (x of the odd rows, y of the odd rows).
__device__ __forceinline__ Pair swap_rows(float x, float y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
// The same of the lower and the upper half.
__device__ __forceinline__ Pair swap_halves(float x, float y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}

// Sum over runs of W lanes (a power of two): every lane gets it.
template <int W>
__device__ __forceinline__ float lanes_sum(float x) {
    if constexpr (W >= 2) x += dpp<kXor1>(x);
    if constexpr (W >= 4) x += dpp<kXor2>(x);
    if constexpr (W >= 8) x += dpp<kHalfMirror>(x);
    if constexpr (W >= 16) x += dpp<kMirror>(x);
    if constexpr (W >= 32) {
        const Pair p = swap_rows(x, x);
        x = p.a + p.b;
    }
    return x;
}
// The value of the lane LM away (the other map's), where all lanes of a map hold
// the same value.
template <int LM>
__device__ __forceinline__ float other_map(float x) {
    if constexpr (LM == 1) return dpp<kXor1>(x);
    if constexpr (LM == 2) return dpp<kXor2>(x);
    if constexpr (LM == 4) return dpp<kHalfMirror>(x);
    if constexpr (LM == 8) return dpp<kMirror>(x);
    const Pair p = swap_rows(x, x);
    return threadIdx.x & 16 ? p.a : p.b;
}
// Over the edge slots, which lie 64 / slots lanes apart: every lane gets it.
template <typename F>
__device__ __forceinline__ float over_slots(float x, int slots, F f) {
    if (slots >= 8) x = f(x, dpp<kRotate + 8>(x));
    if (slots >= 16) x = f(x, dpp<kRotate + 4>(x));
    if (slots >= 32) x = f(x, dpp<kRotate + 2>(x));
    if (slots >= 4) {
        const Pair p = swap_rows(x, x);
        x = f(p.a, p.b);
    }
    if (slots >= 2) {
        const Pair p = swap_halves(x, x);
        x = f(p.a, p.b);
    }
    return x;
}
__device__ __forceinline__ float slots_sum(float x, int slots) {
    return over_slots(x, slots, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float slots_max(float x, int slots) {
    return over_slots(x, slots, [](float a, float b) { return fmaxf(a, b); });
}

// Sums of N values over the edge slots.  With two slots a lane ends with half of
// them, with more with a quarter, starting at scattered_first(): x[0 ..].
template <int N>
__device__ __forceinline__ void scatter_sum(float* x, int slots) {
    if (slots >= 8) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] += dpp<kRotate + 8>(x[i]);
    }
    if (slots >= 16) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] += dpp<kRotate + 4>(x[i]);
    }
    if (slots >= 32) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] += dpp<kRotate + 2>(x[i]);
    }
    if (slots >= 2) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const Pair p = swap_halves(x[i], x[i + N / 2]);
            x[i] = p.a + p.b;
        }
    }
    if (slots >= 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const Pair p = swap_rows(x[i], x[i + N / 4]);
            x[i] = p.a + p.b;
        }
    }
}
template <int N>
__device__ __forceinline__ int scattered_first(int slots) {
    const int lane = threadIdx.x & 63;
    return (slots >= 2 && lane & 32 ? N / 2 : 0) + (slots >= 4 && lane & 16 ? N / 4 : 0);
}
// Of the lanes that hold the same sums, the one that stores them.
__device__ __forceinline__ bool scattered_stores(int slots) {
    return slots <= 4 || (int)(threadIdx.x & 15) < 64 / slots;
}
// Stores what scatter_sum left, of a run at p of which `count` elements exist.
// WHOLE: the run is whole packets.
template <typename T, int N, bool WHOLE>
__device__ __forceinline__ void store_scattered(T* p, const float* sums, int slots, int count) {
    // In a vector: the compiler would merge the branches' stores into one of a
    // variable element and move the array to LDS.
    typedef float values __attribute__((ext_vector_type(N)));
    values x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = sums[i];
    if (!scattered_stores(slots)) return;
    const int first = scattered_first<N>(slots);
    auto put = [&](auto n) {
        constexpr int kN = decltype(n)::value;
        if constexpr (WHOLE) {
            if (first >= count) return;
            constexpr int kMost = (int)(16 / sizeof(T)) < kN ? (int)(16 / sizeof(T)) : kN;
            typedef T part __attribute__((ext_vector_type(kMost)));
#pragma unroll
            for (int j = 0; j < kN / kMost; ++j) {
                if (first + j * kMost >= count) break;
                part v;
#pragma unroll
                for (int i = 0; i < kMost; ++i) v[i] = (T)x[j * kMost + i];
                *reinterpret_cast<part*>(p + first + j * kMost) = v;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i)
                if (first + i < count) p[first + i] = (T)x[i];
        }
    };
    if (slots == 1) put(std::integral_constant<int, N>());
    else if (slots == 2) put(std::integral_constant<int, N / 2>());
    else put(std::integral_constant<int, N / 4>());
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float4* record_at(const AttnArgs& a, int64_t row, int head) {
    return reinterpret_cast<float4*>(reinterpret_cast<char*>(a.record) + row * a.record_row + head * a.record_head);
}
// Piece and heads of a wave.
struct Unit {
    int row, begin, end, slot;
    int head_block;
    bool live;
};

__device__ __forceinline__ Unit unit_of(const AttnArgs& a) {
    // Consecutive workgroups go to the 8 XCDs in turn: workgroup b takes the
    // (b / 8)-th part of XCD (b % 8)'s run of the pieces, so that pieces that lie
    // side by side (rows that share neighbours) share an L2.
    const int64_t per = (gridDim.x + 7) / 8;
    const int64_t full = gridDim.x - (per - 1) * 8;  // XCDs with `per` workgroups
    const int64_t x = blockIdx.x & 7, y = blockIdx.x >> 3;
    const int64_t block = x < full ? x * per + y : full * per + (x - full) * (per - 1) + y;
    // Fewer than 2^32 units (attn_check_units): 32-bit divisions.
    const uint64_t at = (int64_t)a.first_unit + block * (kAttnThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Unit u{};
    u.live = at < a.num_units;
    if (!u.live) return u;
    const uint32_t unit = static_cast<uint32_t>(at), blocks = a.head_blocks;
    uint32_t item = unit;
    if (blocks != 1) {
        if (a.head_items) {
            u.head_block = static_cast<int>(unit / static_cast<uint32_t>(a.head_items));
            item = unit - static_cast<uint32_t>(u.head_block) * static_cast<uint32_t>(a.head_items);
        } else {
            item = unit / blocks;
            u.head_block = static_cast<int>(unit - item * blocks);
        }
    }
    if (a.items) {
        const int4 it = a.items[item];
        u.row = it.x, u.begin = it.y, u.end = it.z, u.slot = it.w;
    } else {
        const uint32_t pieces = a.pieces, row = pieces == 1 ? item : item / pieces, part = item - row * pieces;
        const int64_t b = a.ptr[row], n = a.ptr[row + 1] - b;
        u.row = static_cast<int>(row);
        // Whole multiples of the first part's length, rounded up.
        const int64_t each = pieces == 1 ? n : (int64_t)(((uint32_t)n + pieces - 1) / pieces);
        u.begin = static_cast<int>(b + min(n, each * part));
        u.end = static_cast<int>(b + min(n, each * (part + 1)));
        u.slot = pieces == 1 ? -1 : static_cast<int>(item);
    }
    return u;
}

// A lane's place: edge slot es of `slots`, head, map, and its runs.
template <int LM, int NV>
struct Place {
    int es, slots, head, map, lm, l;
    int kcount, vcount;  // elements of its runs that exist
    bool live;
    __device__ __forceinline__ Place(const AttnArgs& a, int head_block, int heads) {
        const int lane = threadIdx.x & 63;
        l = lane & (2 * LM - 1);
        map = l / LM;
        lm = l & (LM - 1);
        const int hl = (lane / (2 * LM)) & ((1 << a.hb_shift) - 1);
        head = (head_block << a.hb_shift) + hl;
        slots = (32 / LM) >> a.hb_shift;
        es = (lane / (2 * LM)) >> a.hb_shift;
        live = head < heads;
        kcount = live ? max(0, min(8, a.head_dim - 8 * lm)) : 0;
        vcount = live ? max(0, min(NV, a.value_dim - NV * l)) : 0;
        if (!live) head = 0;
    }
};

// Edges in flight per slot: their loads are all issued before the first is used
// (the scheduler would otherwise wait for each in turn to save registers).  Two
// leave registers for 5 or 6 waves a SIMD, four for 4 (power-law graph of 1e6 rows,
// forward: 1.66 against 1.81 ms; skewed fp32 rows 0.50 against 0.61).
constexpr int kDeep = 2;

// The next DEEP edges of every slot.  Past the end the last edge again.
template <int DEEP>
struct Edges {
    uint32_t other[DEEP];
    float add[DEEP];  // bias in powers of two, where there is one
};

// left: edges from e0 on, at least 1.  A uniform address and a lane's offset (opaque
// to the compiler, which would widen it to 64 bits).
template <bool TRANSPOSED, int DEEP>
__device__ __forceinline__ void load_edges(const AttnArgs& a, Edges<DEEP>& x, int e0, int left, int es, int slots) {
    const uint32_t last = static_cast<uint32_t>(min(left - 1, 255)) * 4;  // a step has at most 64 edges
    auto take = [](const auto* p, uint32_t bytes) {
        return *reinterpret_cast<decltype(p)>(reinterpret_cast<const char*>(p) + bytes);
    };
    uint32_t at[DEEP];
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
        at[d] = min(static_cast<uint32_t>(d * slots + es) * 4, last);
        asm("" : "+v"(at[d]));
        x.other[d] = take(a.idx + e0, at[d]);
    }
    if (a.bias) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) x.add[d] = TRANSPOSED ? a.bias[take(a.edge + e0, at[d])] : take(a.bias + e0, at[d]);
    }
}
// Live edges of a step: in the list (a LAST step only may pass its end), and not
// left out by their bias, which becomes powers of two here.  A finite bias stays
// finite, and the order of two is kept: past +-1e38 their difference is halved, which
// is beyond any other score's size either way.
template <int DEEP, bool LAST, int N>
__device__ __forceinline__ void close_edges(const AttnArgs& a, Edges<N>& x, bool* live, int left, int es, int slots) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
        live[d] = !LAST || d * slots + es < left;
        if (!a.bias) x.add[d] = 0.f;
    }
    if (a.bias) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            const float b = x.add[d];
            live[d] = live[d] && b != -INFINITY;
            const float half = fmaf(b, 0.5f * kLog2e, copysignf(0.5f * kLog2e * kBiasLarge, b));
            x.add[d] = fabsf(b) > kBiasLarge ? half : b * kLog2e;
        }
    }
}

// Runs step(DEEP, LAST, first edge) over a wave's edges: whole steps of kDeep edges a
// slot, then one of as few as hold the rest.  Straight-line bodies: conditions on
// single edges would have each load waited for on its own.
template <typename F>
__device__ __forceinline__ void over_edges(int begin, int end, int slots, F step) {
    if (begin >= end) return;
    int e0 = begin;
    for (; end - e0 > kDeep * slots; e0 += kDeep * slots) step(std::integral_constant<int, kDeep>(), std::false_type(), e0);
    if (end - e0 <= slots) step(std::integral_constant<int, 1>(), std::true_type(), e0);
    else step(std::integral_constant<int, kDeep>(), std::true_type(), e0);
}

__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c, f16_t) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, a), __builtin_bit_cast(h2, b), c, false);
}
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c, bf16_t) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, a), __builtin_bit_cast(b2, b), c, false);
}
// Products of two runs, summed in fp32 (16-bit pairs by the two-term instruction).
template <typename T, int N>
__device__ __forceinline__ float dot(const Run<T, N>& a, const Run<T, N>& b) {
    float t = 0.f;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) t = fmaf(a.w[i], b.w[i], t);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) t = dot2(a.w[i], b.w[i], t, T());
    }
    return t;
}

// The same by correctly rounded fused multiply-adds.  The two-term instruction of fp16 rounds downwards a little more often
// than upwards, which a sum over all rows keeps (dlam: 310,108 rows, 2e-9 of the terms' magnitudes, 2e-6 of the result).
template <int N>
__device__ __forceinline__ float dot_rounded(const Run<f16_t, N>& a, const Run<f16_t, N>& b) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    float even = 0.f, odd = 0.f;  // one chain would be made that instruction again
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const h2 x = __builtin_bit_cast(h2, a.w[i]), y = __builtin_bit_cast(h2, b.w[i]);
        even = fmaf((float)x[0], (float)y[0], even);
        odd = fmaf((float)x[1], (float)y[1], odd);
    }
    return even + odd;
}
template <typename T, int N>
__device__ __forceinline__ float dot_rounded(const Run<T, N>& a, const Run<T, N>& b) {
    return dot(a, b);
}

// A lane's run in the rows of a gathered matrix, in packets of PB bytes.  Packets
// that do not exist are loaded from the start of the row's part instead, and masked.
// WIDE: offsets of 64 bits; else of 32, from 24-bit factors (one full-rate
// instruction, and half of the address registers).
template <typename T, int N, int PB, bool WIDE>
struct Gather {
    static constexpr int kBytes = N * (int)sizeof(T);
    static constexpr int kPacket = PB < kBytes ? PB : kBytes;
    static constexpr int kPackets = kBytes / kPacket;
    const char* base;  // of the matrix
    uint32_t offset;   // of the run in row 0
    uint32_t delta[kPackets];
    bool there[kPackets];
    // part: first element of the head's part of a row; the run starts `first`
    // elements into it.
    __device__ __forceinline__ Gather(const void* matrix, int part, int first, int count) {
        there[0] = count > 0;
        base = static_cast<const char*>(matrix);
        offset = static_cast<uint32_t>(there[0] ? part + first : part) * sizeof(T);
        delta[0] = 0;
#pragma unroll
        for (int i = 1; i < kPackets; ++i) {
            there[i] = i * (kPacket / (int)sizeof(T)) < count;
            delta[i] = there[i] ? i * kPacket : 0;
        }
    }
    // further: bytes from the run, the same in all lanes.
    __device__ __forceinline__ void load(Run<T, N>& r, uint32_t row, uint32_t pitch, int further = 0) const {
        const char* const base = this->base + further;
        uint32_t* const w = reinterpret_cast<uint32_t*>(r.w);
#pragma unroll
        for (int i = 0; i < kPackets; ++i) {
            const char* p;
            if constexpr (WIDE) p = base + (static_cast<uint64_t>(row) * pitch + (offset + delta[i]));
            else p = base + (__umul24(row, pitch) + (offset + delta[i]));
            if constexpr (kPacket == 16) {
                const uint4 x = *reinterpret_cast<const uint4*>(p);
                w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
            } else if constexpr (kPacket == 8) {
                const uint2 x = *reinterpret_cast<const uint2*>(p);
                w[2 * i] = x.x, w[2 * i + 1] = x.y;
            } else if constexpr (kPacket == 4) {
                w[i] = *reinterpret_cast<const uint32_t*>(p);
            } else {
                const uint32_t x = *reinterpret_cast<const uint16_t*>(p);
                w[i / 2] = i & 1 ? w[i / 2] | (x << 16) : x;
            }
        }
    }
    __device__ __forceinline__ void mask(Run<T, N>& r, bool live) const {
        uint32_t* const w = reinterpret_cast<uint32_t*>(r.w);
        if constexpr (kPacket == 2) {
#pragma unroll
            for (int i = 0; i < kPackets / 2; ++i) {
                const uint32_t low = live && there[2 * i] ? 0xFFFFu : 0u, high = live && there[2 * i + 1] ? 0xFFFF0000u : 0u;
                w[i] &= low | high;
            }
        } else {
            constexpr int kWords = kPacket / 4;
#pragma unroll
            for (int i = 0; i < kPackets; ++i)
#pragma unroll
                for (int j = 0; j < kWords; ++j) w[kWords * i + j] = live && there[i] ? w[kWords * i + j] : 0u;
        }
    }
};

// Calls KERNEL<T, LM, NV, PB, WIDE> for a layout.
#define RA_ATTN_DISPATCH(KERNEL, dtype, l, grid, st, args)                                                  \
    do {                                                                                                    \
        auto by_type = [&](auto tag) {                                                                      \
            using T = decltype(tag);                                                                        \
            auto by_lm = [&](auto lm) {                                                                     \
                constexpr int LM = decltype(lm)::value;                                                     \
                if ((l).packet == 16 && !(args).wide) {                                                     \
                    if ((l).nv == 4) KERNEL<T, LM, 4, 16, false><<<grid, ra::kAttnThreads, 0, st>>>(args);  \
                    else KERNEL<T, LM, 8, 16, false><<<grid, ra::kAttnThreads, 0, st>>>(args);              \
                } else if ((l).packet == 16) {                                                              \
                    if ((l).nv == 4) KERNEL<T, LM, 4, 16, true><<<grid, ra::kAttnThreads, 0, st>>>(args);   \
                    else KERNEL<T, LM, 8, 16, true><<<grid, ra::kAttnThreads, 0, st>>>(args);               \
                } else if (sizeof(T) == 4 || (l).packet == 4) {                                             \
                    KERNEL<T, LM, 8, 4, true><<<grid, ra::kAttnThreads, 0, st>>>(args);                     \
                } else if constexpr (sizeof(T) == 2) {                                                      \
                    KERNEL<T, LM, 8, 2, true><<<grid, ra::kAttnThreads, 0, st>>>(args);                     \
                }                                                                                           \
            };                                                                                              \
            switch ((l).lm) {                                                                               \
                case 1: by_lm(std::integral_constant<int, 1>()); break;                                     \
                case 2: by_lm(std::integral_constant<int, 2>()); break;                                     \
                case 4: by_lm(std::integral_constant<int, 4>()); break;                                     \
                case 8: by_lm(std::integral_constant<int, 8>()); break;                                     \
                default: by_lm(std::integral_constant<int, 16>());                                          \
            }                                                                                               \
        };                                                                                                  \
        if ((dtype) == RA_DTYPE_F32) by_type(float());                                                      \
        else if ((dtype) == RA_DTYPE_F16) by_type(ra::f16_t());                                             \
        else by_type(ra::bf16_t());                                                                         \
    } while (0)

}  // namespace ra
