// weight_grad8.hip — weight gradient of a linear layer from its 8-bit input:
// out [O, C] = grad^T (code * scale), summed over rows.
//
// code * scale has at most 8 significant bits, so it is exact in bf16.  grad is cut
// into bf16 pieces that add up to it exactly: an fp32 value's 24 bits are three runs
// of 8, an fp16 value's 11 bits two, a bf16 value is one.  Every product is then
// exact in the matrix cores and only the fp32 sums round, at 1 to 3 matrix products
// of 2.5 PFLOP/s in place of one of 157 TFLOP/s in fp32.
//
// The reduction runs over the rows, so both operands want 8 consecutive rows of one
// column per lane.  A thread therefore loads 8 rows of a column (neighbouring lanes
// the neighbouring columns, whole lines), cuts and packs them in registers and
// writes one 16-byte vector per piece to LDS, where they are read as they lie.  Each
// element is converted once per workgroup.  Workgroups hold up to 128 x 256 of the
// output and split the rows; a second launch adds their sums in order.
// Measured: 1e6 rows, 256 columns, fp32 grad of 47: 128 us and 8 for the joining launch (0.45 GB,
// 3.3 TB/s); 512,000 rows, 128 columns, bf16 grad of 256: 96 and 7 (0.33 GB, 3.2 TB/s, 0.32
// PFLOP/s).  Bound by the turn of a stage: loads, cut, LDS and barrier, with two stages in flight.
#include <type_traits>

#include "pack8.hpp"
#include "vector_run.hpp"

namespace ra {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kRows = 32;  // rows of a stage
constexpr int kTile = 64;  // a wave's part of the output, both ways

struct GradArgs {
    const void* grad;
    const uint8_t *codes, *scales;
    float* out;  // the result, or the workgroups' parts [splits][O][C]
    int64_t rows, ldg, rows_per_split, scale_pitch;
    int32_t O, C, groups, tiles_o, tiles_c, splits;
    bool even;  // pairs of 16-bit columns lie on 4-byte addresses
};

template <typename T>
constexpr int kPieces = sizeof(T) == 4 ? 3 : std::is_same<T, f16_t>::value ? 2 : 1;

__device__ __forceinline__ uint32_t high_halves(uint32_t lo, uint32_t hi) {  // (hi's upper half, lo's upper half)
    return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}

// The upper 8 significant bits of x, and what is left of x (exact; nothing is left of
// an inf, which the first piece holds).
template <bool FIRST>
__device__ __forceinline__ uint32_t take_piece(float& x) {
    const uint32_t top = __float_as_uint(x) & 0xFFFF0000u;
    const float rest = x - __uint_as_float(top);
    x = FIRST && fabsf(x) == INFINITY ? 0.f : rest;
    return top;
}

// Pieces of 8 values of a column: one vector of 8 bf16 each.
template <int PIECES>
__device__ __forceinline__ void cut(const float* x, uint4* piece) {
    uint32_t word[PIECES][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float rest = x[i];
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
            word[p][i] = p + 1 == PIECES ? __float_as_uint(rest) : p == 0 ? take_piece<true>(rest) : take_piece<false>(rest);
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
        piece[p] = make_uint4(high_halves(word[p][0], word[p][1]), high_halves(word[p][2], word[p][3]),
                              high_halves(word[p][4], word[p][5]), high_halves(word[p][6], word[p][7]));
}

// Waves a SIMD that shared memory leaves room for: the three pieces of float32 take 24 KB for every wave of WO.
template <typename T, int WO, int WI>
constexpr int kWavesPerSimd = kPieces<T> == 3 && WO > 1 && WI == 1 ? 1 : 2;

// WO x WI waves.
template <typename T, int WO, int WI, bool SIGNED, bool FEW>
__global__ __launch_bounds__(64 * WO * WI, (kWavesPerSimd<T, WO, WI>)) void weight_grad8(const GradArgs a) {
    constexpr int PIECES = kPieces<T>, BO = WO * kTile, BI = WI * kTile, NT = 64 * WO * WI, KB = kRows / 8;
    constexpr bool PAIRS = sizeof(T) == 2;
    // Staging work: (8 rows, column or pair of columns) of grad, (8 rows, 4 columns)
    // of the codes.
    constexpr int G_ITEMS = KB * BO / (PAIRS ? 2 : 1), G_EACH = (G_ITEMS + NT - 1) / NT;
    constexpr int C_ITEMS = KB * BI / 4, C_EACH = (C_ITEMS + NT - 1) / NT;
    __shared__ uint4 gs[2][PIECES][KB][BO];
    __shared__ uint4 cs[2][KB][BI];
    // A thread's neighbouring columns lie BO / 2 and BI / 4 vectors apart, so that the
    // lanes of a write lie side by side; the output's rows and columns come in that
    // order.
    auto o_of = [](int slot) { return PAIRS ? slot % (BO / 2) * 2 + slot / (BO / 2) : slot; };
    auto c_of = [](int slot) { return slot % (BI / 4) * 4 + slot / (BI / 4); };

    const int tiles = a.tiles_o * a.tiles_c;
    const int split = blockIdx.x / tiles, tile = blockIdx.x - split * tiles;
    const int o0 = tile / a.tiles_c * BO, c0 = tile % a.tiles_c * BI;
    const int64_t first = split * a.rows_per_split, end = min(first + a.rows_per_split, a.rows);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

    // Where a thread's parts lie: rows of 8 and the first column.  Columns past the
    // output's give results that are not stored; they load the last ones.
    int g_row[G_EACH], g_col[G_EACH], c_row[C_EACH], c_col[C_EACH];
#pragma unroll
    for (int e = 0; e < G_EACH; ++e) {
        const int item = tid + e * NT, o = o0 + item % (G_ITEMS / KB) * (PAIRS ? 2 : 1);
        g_row[e] = item / (G_ITEMS / KB) * 8 % kRows;
        g_col[e] = min(o, PAIRS && a.even ? a.O - 2 : a.O - 1);
    }
#pragma unroll
    for (int e = 0; e < C_EACH; ++e) {
        const int item = tid + e * NT;
        c_row[e] = item / (BI / 4) * 8 % kRows;
        c_col[e] = min(c0 + item % (BI / 4) * 4, a.groups * kPackGroup - 4);
    }
    // Two stages' loads are in flight: one stage's products take a tenth of the time
    // of a load.
    struct Raw {
        uint32_t g[G_EACH][8], c[C_EACH][8];
        uint2 s[C_EACH];  // scales of the 8 rows
    } raw[2];
    const int64_t pitch = (int64_t)a.groups * kPackGroup;
    // Every stage loads kRows whole rows, without a condition that the wait for the
    // stage before would have to allow for: the last one starts early enough, and the
    // rows that were counted before are masked.  FEW: fewer rows than a stage in all;
    // the last one stands in for those that do not exist.
    auto base_of = [&](int64_t m0) { return FEW ? m0 : min(m0, end - kRows); };
    auto load = [&](Raw& r, int64_t m0) {
        const int64_t base = base_of(m0);
        const int last = FEW ? static_cast<int>(end - base) - 1 : kRows - 1;
#pragma unroll
        for (int e = 0; e < G_EACH; ++e)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // A uniform row and a 32-bit offset.
                const T* const p = FEW ? static_cast<const T*>(a.grad) + (base + min(g_row[e] + i, last)) * a.ldg + g_col[e]
                                       : static_cast<const T*>(a.grad) + (base + i) * a.ldg +
                                             static_cast<uint32_t>(g_row[e] * static_cast<int>(a.ldg) + g_col[e]);
                if constexpr (!PAIRS) {
                    r.g[e][i] = __builtin_bit_cast(uint32_t, *p);
                } else if (a.even) {
                    r.g[e][i] = *reinterpret_cast<const uint32_t*>(p);
                } else {
                    const uint16_t* const h = reinterpret_cast<const uint16_t*>(p);
                    r.g[e][i] = h[0] | static_cast<uint32_t>(h[g_col[e] + 1 < a.O ? 1 : 0]) << 16;
                }
            }
#pragma unroll
        for (int e = 0; e < C_EACH; ++e) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint8_t* const p = FEW ? a.codes + (base + min(c_row[e] + i, last)) * pitch + c_col[e]
                                             : a.codes + (base + i) * pitch +
                                                   static_cast<uint32_t>(c_row[e] * static_cast<int>(pitch) + c_col[e]);
                r.c[e][i] = *reinterpret_cast<const uint32_t*>(p);
            }
            const uint8_t* const p = a.scales + (c_col[e] / kPackGroup) * a.scale_pitch + base;
            if constexpr (FEW) {
                uint32_t w[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i / 4] |= static_cast<uint32_t>(p[min(c_row[e] + i, last)]) << (8 * (i & 3));
                r.s[e] = make_uint2(w[0], w[1]);
            } else {
                __builtin_memcpy(&r.s[e], p + c_row[e], 8);  // of any alignment in the last stage
            }
        }
    };
    auto store = [&](Raw& r, int stage, int64_t m0) {
        const int counted = static_cast<int>(m0 - base_of(m0)), rows = static_cast<int>(min(end - m0, (int64_t)kRows));
        if (counted > 0 || (FEW && rows < kRows)) {
#pragma unroll
            for (int e = 0; e < G_EACH; ++e)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int row = g_row[e] + i;
                    r.g[e][i] = row >= counted && (!FEW || row < rows) ? r.g[e][i] : 0u;
                }
        }
#pragma unroll
        for (int e = 0; e < G_EACH; ++e) {
            const int item = tid + e * NT;
            if (G_ITEMS % NT != 0 && item >= G_ITEMS) continue;
            const int kb = item / (G_ITEMS / KB), o = item % (G_ITEMS / KB) * (PAIRS ? 2 : 1);
            float x[2][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (PAIRS) unpack2(r.g[e][i], x[0][i], x[1][i], T());
                else x[0][i] = __uint_as_float(r.g[e][i]);
            }
#pragma unroll
            for (int h = 0; h < (PAIRS ? 2 : 1); ++h) {
                uint4 piece[PIECES];
                cut<PIECES>(x[h], piece);
#pragma unroll
                for (int p = 0; p < PIECES; ++p) gs[stage][p][kb][o / (PAIRS ? 2 : 1) + h * (BO / 2)] = piece[p];
            }
        }
#pragma unroll
        for (int e = 0; e < C_EACH; ++e) {
            const int item = tid + e * NT;
            if (C_ITEMS % NT != 0 && item >= C_ITEMS) continue;
            const int kb = item / (BI / 4), c = item % (BI / 4) * 4;
            float x[4][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v[4];
                pack8_values<SIGNED>(r.c[e][i], pack8_scale((i < 4 ? r.s[e].x : r.s[e].y) >> (8 * (i & 3)) & 0xFFu), v);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j][i] = v[j];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) cut<1>(x[j], &cs[stage][kb][c / 4 + j * (BI / 4)]);
        }
    };

    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    const int wo = wave / WI * kTile, wi = wave % WI * kTile, col = lane & 31, half = lane >> 5;

    // A stage is written while slower waves may still
    // read the other one; the barrier keeps them at most one apart.
    auto step = [&](Raw& r, int stage, int64_t m0) {
        store(r, stage, m0);
        if constexpr (!FEW) load(r, m0 + 2 * kRows);
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kRows / 16; ++kk) {
            bf16x8 b[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) b[j] = __builtin_bit_cast(bf16x8, cs[stage][2 * kk + half][wi + 32 * j + col]);
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bf16x8 g = __builtin_bit_cast(bf16x8, gs[stage][p][2 * kk + half][wo + 32 * i + col]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(g, b[j], acc[i][j], 0, 0, 0);
                }
        }
    };
    if (first < end) {
        load(raw[0], first);
        load(raw[1], FEW ? first : first + kRows);
        int64_t m0 = first;
        if constexpr (!FEW)
            for (; m0 + kRows < end; m0 += 2 * kRows) {
                step(raw[0], 0, m0);
                step(raw[1], 1, m0 + kRows);
            }
        if (m0 < end) step(raw[0], 0, m0);
    }

    float* const out = a.out + (int64_t)split * a.O * a.C;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int c = c0 + c_of(wi + 32 * j + col);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int o = o0 + o_of(wo + 32 * i + 8 * (e / 4) + 4 * half + e % 4);
                if (o < a.O && c < a.C) out[(int64_t)o * a.C + c] = acc[i][j][e];
            }
        }
}

// Sum of the splits, in order: 32 elements x 8 runs of the splits a workgroup.
__global__ __launch_bounds__(256) void weight_grad8_join(const float* __restrict__ parts, int64_t n, int splits,
                                                         float* __restrict__ out) {
    __shared__ float sum[8][32];
    const int at = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + at;
    float x = 0.f;
    if (i < n) {
#pragma unroll 8
        for (int s = part; s < splits; s += 8) x += parts[s * n + i];
    }
    sum[part][at] = x;
    __syncthreads();
    if (part != 0 || i >= n) return;
    for (int p = 1; p < 8; ++p) x += sum[p][at];
    out[i] = x;
}

// Waves of a workgroup in one direction.
int waves_for(int32_t n) { return n <= kTile ? 1 : n <= 2 * kTile ? 2 : 4; }

struct Split {
    int wo, wi, tiles_o, tiles_c, splits;
    int64_t rows_per_split;
};

// As many splits as give every CU its workgroups (8 waves of them, what their
// registers allow), of at least 128 rows.  A workgroup has 8 waves at most (more spill their sums): where both sides
// of the output are wide, it covers the columns first, because a second pass over
// grad costs up to four times a second pass over the codes.
Split split_of(int64_t rows, int32_t O, int32_t C) {
    Split s{};
    s.wo = waves_for(O);
    s.wi = waves_for(C);
    if (s.wo * s.wi > 8) s.wo = 2;
    if (rows < kRows) s.wo = s.wi = 1;
    s.tiles_o = (O + s.wo * kTile - 1) / (s.wo * kTile);
    s.tiles_c = (C + s.wi * kTile - 1) / (s.wi * kTile);
    const int64_t tiles = (int64_t)s.tiles_o * s.tiles_c;
    const int64_t wanted = std::max<int64_t>(1, 256 * std::min(4, 8 / (s.wo * s.wi)) / tiles);
    const int64_t per = std::max<int64_t>(128, (rows + wanted - 1) / wanted);
    s.rows_per_split = (per + kRows - 1) / kRows * kRows;
    s.splits = static_cast<int>(std::max<int64_t>(1, (rows + s.rows_per_split - 1) / s.rows_per_split));
    return s;
}

template <typename T, bool SIGNED>
void launch(const Split& s, const GradArgs& a, hipStream_t st) {
    const unsigned grid = static_cast<unsigned>(s.splits) * s.tiles_o * s.tiles_c;
    auto go = [&](auto wo, auto wi) {
        constexpr int WO = decltype(wo)::value, WI = decltype(wi)::value;
        weight_grad8<T, WO, WI, SIGNED, false><<<grid, 64 * WO * WI, 0, st>>>(a);
    };
    if (a.rows < kRows) {
        weight_grad8<T, 1, 1, SIGNED, true><<<grid, 64, 0, st>>>(a);
        return;
    }
    auto by_wi = [&](auto wo) {
        if (s.wi == 1) go(wo, std::integral_constant<int, 1>());
        else if (s.wi == 2) go(wo, std::integral_constant<int, 2>());
        else if constexpr (decltype(wo)::value < 4) go(wo, std::integral_constant<int, 4>());
    };
    if (s.wo == 1) by_wi(std::integral_constant<int, 1>());
    else if (s.wo == 2) by_wi(std::integral_constant<int, 2>());
    else by_wi(std::integral_constant<int, 4>());
}

ra_status check(int64_t rows, int32_t O, int32_t C) {
    if (rows < 0 || O < 1 || C < 1) return fail(RA_ERR_INVALID_ARGUMENT, "weight_grad8: bad sizes");
    if (rows > INT64_MAX / 8 / ((int64_t)C + 64) || (int64_t)O * C > INT32_MAX || C > (1 << 26))
        return fail(RA_ERR_UNSUPPORTED, "weight_grad8: too large");
    return RA_OK;
}

}  // namespace
}  // namespace ra

using ra::fail;

extern "C" {

ra_status ra_weight_grad8_workspace(int64_t rows, int32_t out, int32_t cols, int64_t* bytes) {
    if (!bytes) return fail(RA_ERR_INVALID_ARGUMENT, "weight_grad8: bytes is NULL");
    RA_TRY(ra::check(rows, out, cols));
    const ra::Split s = ra::split_of(rows, out, cols);
    *bytes = s.splits == 1 ? 0 : (int64_t)s.splits * out * cols * (int64_t)sizeof(float);
    return RA_OK;
}

ra_status ra_weight_grad8(const void* d_grad, const uint8_t* d_codes, const uint8_t* d_scales, int64_t rows,
                          int32_t out, int32_t cols, int64_t ldg, int32_t is_signed, int32_t dtype, float* d_out,
                          void* d_workspace, int64_t bytes, ra_stream_t stream) {
    int64_t need = 0;
    RA_TRY(ra_weight_grad8_workspace(rows, out, cols, &need));
    if (dtype != RA_DTYPE_F32 && dtype != RA_DTYPE_F16 && dtype != RA_DTYPE_BF16)
        return fail(RA_ERR_INVALID_ARGUMENT, "weight_grad8: unknown dtype");
    if (!d_out || (rows > 0 && (!d_grad || !d_codes || !d_scales)))
        return fail(RA_ERR_INVALID_ARGUMENT, "weight_grad8: NULL tensor");
    if (ldg >= int64_t{1} << 26) return fail(RA_ERR_UNSUPPORTED, "weight_grad8: rows lie at most 2^26 elements apart");
    if (rows > 1 && ldg < out) return fail(RA_ERR_INVALID_ARGUMENT, "weight_grad8: rows overlap (a leading dimension is too small)");
    if (!ra::aligned16(d_codes) || !ra::aligned16(d_scales) || !ra::aligned16(d_workspace) || bytes < need || (need && !d_workspace))
        return fail(RA_ERR_INVALID_ARGUMENT, "weight_grad8: the workspace is too small, or it, the codes or the scales are not 16-byte aligned");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const ra::Split s = ra::split_of(rows, out, cols);
    ra::GradArgs a{};
    a.grad = d_grad;
    a.codes = d_codes;
    a.scales = d_scales;
    a.out = s.splits == 1 ? d_out : static_cast<float*>(d_workspace);
    a.rows = rows;
    a.ldg = ldg;
    a.rows_per_split = s.rows_per_split;
    a.O = out;
    a.C = cols;
    a.groups = ra::pack8_groups(cols);
    a.scale_pitch = ra::pack8_scale_pitch(rows);
    a.tiles_o = s.tiles_o;
    a.tiles_c = s.tiles_c;
    a.splits = s.splits;
    a.even = reinterpret_cast<uintptr_t>(d_grad) % 4 == 0 && out % 2 == 0 && (rows <= 1 || ldg % 2 == 0);
    auto by_type = [&](auto tag) {
        if (is_signed) ra::launch<decltype(tag), true>(s, a, st);
        else ra::launch<decltype(tag), false>(s, a, st);
    };
    if (dtype == RA_DTYPE_F32) by_type(float());
    else if (dtype == RA_DTYPE_F16) by_type(ra::f16_t());
    else by_type(ra::bf16_t());
    RA_LAUNCH_CHECK("weight_grad8");
    if (s.splits > 1) {
        const int64_t n = (int64_t)out * cols;
        ra::weight_grad8_join<<<static_cast<unsigned>((n + 31) / 32), 256, 0, st>>>(a.out, n, s.splits, d_out);
        RA_LAUNCH_CHECK("weight_grad8_join");
    }
    return RA_OK;
}

}  // extern "C"
