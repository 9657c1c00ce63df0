// pack8.hip — activations kept in 8 bits: pack, ReLU and pack, unpack, the ReLU's
// gradient from the codes.
//
// Bound by memory.  Four lanes share a group of 32 columns, 8 each: a lane reads its
// run in whole packets, the group's largest magnitude takes two exchanges within the
// four lanes, and the codes go out as 8 bytes a lane.  The scale is a power of two,
// so code * scale and x / scale are exact and rounding happens once.  Measured: ReLU and
// pack of 1e6 x 256 fp32 428 us (2.31 GB, 5.4 TB/s), the ReLU's gradient 424 (5.4); 512,000 x
// 128 in bf16 51 and 53 us (6.5 and 6.2 TB/s, partly from the last-level cache); a large copy
// reaches 5.1.
#include <type_traits>

#include "pack8.hpp"
#include "vector_run.hpp"

namespace ra {
namespace {

constexpr int kThreads = 256;

struct PackArgs {
    const void* x;
    void* y;
    uint8_t *codes, *scales;
    int64_t rows, ld;  // rows of x lie ld elements apart
    int64_t scale_pitch;
    int32_t cols, groups;
};

// A wave takes 16 * STEPS consecutive (row, group) pairs, 16 at a time, with all
// steps' loads in flight together: 4 steps where that leaves enough waves (a wave for
// every slot of the GPU; pack of 512,000 x 128 bf16 53 against 63 us, of 1e6 x 256 fp32 436
// against 448), else 1 (10,000 rows of 2 groups: 3.5 against 5 us).
constexpr int64_t kManyPairs = 64 * 8192;
struct Spot {
    int64_t row;
    int group, col, count;
    bool live;
    __device__ __forceinline__ Spot() {}
    // pair: of the quad of lanes.
    __device__ __forceinline__ Spot(int64_t pair, const PackArgs& a) {
        const int64_t pairs = a.rows * a.groups;
        live = pair < pairs;
        pair = live ? pair : pairs - 1;
        row = a.groups == 1 ? pair : pair <= UINT32_MAX ? (int64_t)((uint32_t)pair / (uint32_t)a.groups) : pair / a.groups;
        group = static_cast<int>(pair - row * a.groups);
        col = group * kPackGroup + 8 * (threadIdx.x & 3);
        count = max(0, min(8, a.cols - col));
    }
    __device__ __forceinline__ int64_t code(const PackArgs& a) const { return (row * a.groups + group) * kPackGroup + (col & 31); }
};
// First pair of the wave, and how far it goes on.
template <int STEPS>
__device__ __forceinline__ int64_t first_pair() {
    return ((int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * (16 * STEPS);
}
template <int STEPS>
__device__ __forceinline__ int64_t pair_step() {
    return (int64_t)gridDim.x * (kThreads / 64 * 16 * STEPS);
}

__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xF, 0xF, true)));
    return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xF, 0xF, true)));
}

template <typename T, bool VEC, bool RELU, int STEPS>
__global__ __launch_bounds__(kThreads) void pack8(const PackArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t first = first_pair<STEPS>(); first < a.rows * a.groups; first += pair_step<STEPS>()) {
        Spot at[STEPS];
        Run<T, 8> r[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            at[i] = Spot(first + 16 * i + (lane >> 2), a);
            load_run<T, 8, VEC>(r[i], static_cast<const T*>(a.x) + at[i].row * a.ld + at[i].col, at[i].count);
        }
        __builtin_amdgcn_sched_barrier(0);
        int biased[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            float x[8], top = 0.f;
            r[s].to_float(x);
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (RELU) x[i] = x[i] <= 0.f ? 0.f : x[i];  // NaN stays
                bad |= !(fabsf(x[i]) <= 3.4028234663852886e38f);
                top = fmaxf(top, fabsf(x[i]));
            }
            top = quad_max(bad ? INFINITY : top);
            const bool finite = top <= 3.4028234663852886e38f;
            // Exponent of the largest magnitude, minus the bits of a code above its
            // point; magnitudes below 2^-120 share the smallest scale.
            const int exponent = static_cast<int>(__float_as_uint(top) >> 23);
            biased[s] = finite ? max(1, exponent - (RELU ? 7 : 6)) : 255;
            const float inverse = __uint_as_float(static_cast<uint32_t>(254 - min(biased[s], 253)) << 23);
            uint32_t word[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float c = rintf(x[i] * inverse);
                if (RELU) {
                    c = fminf(c, 255.f);
                    if (x[i] > 0.f) c = fmaxf(c, 1.f);
                    if (!finite) c = x[i] > 0.f || x[i] != x[i] ? 1.f : 0.f;
                } else {
                    c = fminf(fmaxf(c, -127.f), 127.f);
                    if (!finite) c = 0.f;
                }
                word[i / 4] |= (static_cast<uint32_t>(static_cast<int>(c)) & 0xFFu) << (8 * (i & 3));
            }
            if (at[s].live) {
                *reinterpret_cast<uint2*>(a.codes + at[s].code(a)) = make_uint2(word[0], word[1]);
                if (RELU) store_run<T, 8, VEC>(static_cast<T*>(a.y) + at[s].row * a.cols + at[s].col, x, at[s].count);
            }
        }
        // A lane per pair: one store of the scales, a row's neighbours beside each other.
        int mine = 0;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int x = __shfl(biased[i], 4 * (lane & 15), 64);
            if (lane >> 4 == i) mine = x;
        }
        const Spot own(first + lane, a);
        if (own.live && lane < 16 * STEPS) a.scales[own.group * a.scale_pitch + own.row] = static_cast<uint8_t>(mine);
    }
}

template <typename T, bool VEC, bool SIGNED, int STEPS>
__global__ __launch_bounds__(kThreads) void unpack8(const PackArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t first = first_pair<STEPS>(); first < a.rows * a.groups; first += pair_step<STEPS>()) {
        const Spot own(first + lane, a);
        const int scale_byte = a.scales[own.group * a.scale_pitch + own.row];
        Spot at[STEPS];
        uint2 w[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            at[i] = Spot(first + 16 * i + (lane >> 2), a);
            w[i] = *reinterpret_cast<const uint2*>(a.codes + at[i].code(a));
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const float scale = pack8_scale(static_cast<uint32_t>(__shfl(scale_byte, 16 * i + (lane >> 2), 64)));
            float x[8];
            pack8_values<SIGNED>(w[i].x, scale, x);
            pack8_values<SIGNED>(w[i].y, scale, x + 4);
            if (at[i].live) store_run<T, 8, VEC>(static_cast<T*>(a.y) + at[i].row * a.cols + at[i].col, x, at[i].count);
        }
    }
}

// One step a wave: it has two loads in flight already (1e6 x 256 fp32: 424 against 431 us with
// four steps, 512,000 x 128 bf16: 53 against 55).
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void relu_grad8(const PackArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t first = first_pair<1>(); first < a.rows * a.groups; first += pair_step<1>()) {
        const Spot at(first + (lane >> 2), a);
        Run<T, 8> r;
        const uint2 w = *reinterpret_cast<const uint2*>(a.codes + at.code(a));
        load_run<T, 8, VEC>(r, static_cast<const T*>(a.x) + at.row * a.ld + at.col, at.count);
        float x[8];
        r.to_float(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (i < 4 ? w.x : w.y) >> (8 * (i & 3)) & 0xFFu ? x[i] : 0.f;
        if (at.live) store_run<T, 8, VEC>(static_cast<T*>(a.y) + at.row * a.cols + at.col, x, at.count);
    }
}

int steps_for(const PackArgs& a) { return a.rows * a.groups >= kManyPairs ? 4 : 1; }
unsigned grid_for(const PackArgs& a, int steps) {
    const int64_t per = kThreads / 64 * 16 * steps;
    return static_cast<unsigned>(std::min<int64_t>((a.rows * a.groups + per - 1) / per, 65536));
}

ra_status check(int64_t rows, int32_t cols, int64_t ld, int32_t dtype, const void* codes, const void* scales) {
    if (rows < 0 || cols < 1) return fail(RA_ERR_INVALID_ARGUMENT, "pack8: bad sizes");
    if (rows > INT64_MAX / 8 / ((int64_t)cols + 64)) return fail(RA_ERR_INVALID_ARGUMENT, "pack8: bad sizes");
    if (dtype != RA_DTYPE_F32 && dtype != RA_DTYPE_F16 && dtype != RA_DTYPE_BF16)
        return fail(RA_ERR_INVALID_ARGUMENT, "pack8: unknown dtype");
    if (rows > 1 && ld < cols) return fail(RA_ERR_INVALID_ARGUMENT, "pack8: rows overlap (a leading dimension is too small)");
    if (rows > 0 && (!codes || !scales)) return fail(RA_ERR_INVALID_ARGUMENT, "pack8: NULL codes or scales");
    if (!aligned16(codes) || !aligned16(scales)) return fail(RA_ERR_INVALID_ARGUMENT, "pack8: codes or scales are not 16-byte aligned");
    return RA_OK;
}

PackArgs args_of(const void* x, void* y, const uint8_t* codes, const uint8_t* scales, int64_t rows, int32_t cols, int64_t ld) {
    PackArgs a{};
    a.x = x;
    a.y = y;
    a.codes = const_cast<uint8_t*>(codes);
    a.scales = const_cast<uint8_t*>(scales);
    a.rows = rows;
    a.cols = cols;
    a.groups = pack8_groups(cols);
    a.scale_pitch = pack8_scale_pitch(rows);
    a.ld = ld;
    return a;
}

// Whole packets on both sides: x with rows ld apart, y contiguous.
bool whole(const PackArgs& a, int32_t dtype) {
    const int64_t size = dtype == RA_DTYPE_F32 ? 4 : 2;
    return aligned16(a.x) && aligned16(a.y) && a.cols * size % 16 == 0 && (a.rows <= 1 || a.ld * size % 16 == 0);
}

// f(type, whole packets, steps)
template <typename F>
void by_type(int32_t dtype, const PackArgs& a, F f) {
    auto by_steps = [&](auto tag, auto vec) {
        if (steps_for(a) == 4) f(tag, vec, std::integral_constant<int, 4>());
        else f(tag, vec, std::integral_constant<int, 1>());
    };
    auto by_vec = [&](auto tag) {
        if (whole(a, dtype)) by_steps(tag, std::true_type());
        else by_steps(tag, std::false_type());
    };
    if (dtype == RA_DTYPE_F32) by_vec(float());
    else if (dtype == RA_DTYPE_F16) by_vec(f16_t());
    else by_vec(bf16_t());
}

}  // namespace
}  // namespace ra

using ra::fail;

extern "C" {

ra_status ra_pack8(const void* d_x, int64_t rows, int32_t cols, int64_t ldx, int32_t dtype, uint8_t* d_codes,
                   uint8_t* d_scales, ra_stream_t stream) {
    RA_TRY(ra::check(rows, cols, ldx, dtype, d_codes, d_scales));
    if (rows == 0) return RA_OK;
    if (!d_x) return fail(RA_ERR_INVALID_ARGUMENT, "pack8: NULL tensor");
    const ra::PackArgs a = ra::args_of(d_x, nullptr, d_codes, d_scales, rows, cols, ldx);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    ra::by_type(dtype, a, [&](auto tag, auto vec, auto steps) {
        ra::pack8<decltype(tag), decltype(vec)::value, false, decltype(steps)::value><<<ra::grid_for(a, steps), ra::kThreads, 0, st>>>(a);
    });
    RA_LAUNCH_CHECK("pack8");
    return RA_OK;
}

ra_status ra_relu_pack8(const void* d_x, int64_t rows, int32_t cols, int64_t ldx, int32_t dtype, void* d_y,
                        uint8_t* d_codes, uint8_t* d_scales, ra_stream_t stream) {
    RA_TRY(ra::check(rows, cols, ldx, dtype, d_codes, d_scales));
    if (rows == 0) return RA_OK;
    if (!d_x || !d_y) return fail(RA_ERR_INVALID_ARGUMENT, "pack8: NULL tensor");
    const ra::PackArgs a = ra::args_of(d_x, d_y, d_codes, d_scales, rows, cols, ldx);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    ra::by_type(dtype, a, [&](auto tag, auto vec, auto steps) {
        ra::pack8<decltype(tag), decltype(vec)::value, true, decltype(steps)::value><<<ra::grid_for(a, steps), ra::kThreads, 0, st>>>(a);
    });
    RA_LAUNCH_CHECK("relu_pack8");
    return RA_OK;
}

ra_status ra_unpack8(const uint8_t* d_codes, const uint8_t* d_scales, int64_t rows, int32_t cols, int32_t is_signed,
                     int32_t dtype, void* d_out, ra_stream_t stream) {
    RA_TRY(ra::check(rows, cols, cols, dtype, d_codes, d_scales));
    if (rows == 0) return RA_OK;
    if (!d_out) return fail(RA_ERR_INVALID_ARGUMENT, "unpack8: NULL tensor");
    const ra::PackArgs a = ra::args_of(nullptr, d_out, d_codes, d_scales, rows, cols, cols);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    ra::by_type(dtype, a, [&](auto tag, auto vec, auto steps) {
        using T = decltype(tag);
        if (is_signed) ra::unpack8<T, decltype(vec)::value, true, decltype(steps)::value><<<ra::grid_for(a, steps), ra::kThreads, 0, st>>>(a);
        else ra::unpack8<T, decltype(vec)::value, false, decltype(steps)::value><<<ra::grid_for(a, steps), ra::kThreads, 0, st>>>(a);
    });
    RA_LAUNCH_CHECK("unpack8");
    return RA_OK;
}

ra_status ra_relu_grad8(const void* d_grad, const uint8_t* d_codes, int64_t rows, int32_t cols, int64_t ldg,
                        int32_t dtype, void* d_out, ra_stream_t stream) {
    RA_TRY(ra::check(rows, cols, ldg, dtype, d_codes, d_codes));
    if (rows == 0) return RA_OK;
    if (!d_grad || !d_out) return fail(RA_ERR_INVALID_ARGUMENT, "relu_grad8: NULL tensor");
    const ra::PackArgs a = ra::args_of(d_grad, d_out, d_codes, nullptr, rows, cols, ldg);
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    ra::by_type(dtype, a, [&](auto tag, auto vec, auto) {
        ra::relu_grad8<decltype(tag), decltype(vec)::value><<<ra::grid_for(a, 1), ra::kThreads, 0, st>>>(a);
    });
    RA_LAUNCH_CHECK("relu_grad8");
    return RA_OK;
}

}  // extern "C"
