// pack8.hip — activations kept in 8 bits: pack, ReLU and pack, unpack, the ReLU's
// gradient from the codes.
//
// Bound by memory.  Four lanes share a group of 32 columns, 8 each: a lane reads its
// run in whole packets, the group's largest magnitude takes two exchanges within the
// four lanes, and the codes go out as 8 bytes a lane.  The scale is a power of two,
// so code * scale and x / scale are exact and rounding happens once.
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
    int32_t cols, groups;
};

// Row and group of a run of four lanes; the group index may pass 32 bits.
struct Spot {
    int64_t row;
    int group, col, count;
    __device__ __forceinline__ Spot(int64_t quad, int cols, int groups) {
        row = groups == 1 ? quad : quad <= UINT32_MAX ? (int64_t)((uint32_t)quad / (uint32_t)groups) : quad / groups;
        group = static_cast<int>(quad - row * groups);
        col = group * kPackGroup + 8 * (threadIdx.x & 3);
        count = max(0, min(8, cols - col));
    }
};

__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xF, 0xF, true)));
    return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xF, 0xF, true)));
}

template <typename T, bool VEC, bool RELU>
__global__ __launch_bounds__(kThreads) void pack8(const PackArgs a) {
    const int64_t quads = a.rows * a.groups, step = (int64_t)gridDim.x * (kThreads / 4);
    for (int64_t quad = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 2; quad < quads; quad += step) {
        const Spot at(quad, a.cols, a.groups);
        Run<T, 8> r;
        load_run<T, 8, VEC>(r, static_cast<const T*>(a.x) + at.row * a.ld + at.col, at.count);
        float x[8], top = 0.f;
        r.to_float(x);
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
        const int biased = finite ? max(1, exponent - (RELU ? 7 : 6)) : 255;
        const float inverse = __uint_as_float(static_cast<uint32_t>(254 - min(biased, 253)) << 23);
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
        *reinterpret_cast<uint2*>(a.codes + (at.row * a.groups + at.group) * kPackGroup + 8 * (threadIdx.x & 3)) =
            make_uint2(word[0], word[1]);
        if ((threadIdx.x & 3) == 0) a.scales[quad] = static_cast<uint8_t>(biased);
        if (RELU) store_run<T, 8, VEC>(static_cast<T*>(a.y) + at.row * a.cols + at.col, x, at.count);
    }
}

template <typename T, bool VEC, bool SIGNED>
__global__ __launch_bounds__(kThreads) void unpack8(const PackArgs a) {
    const int64_t quads = a.rows * a.groups, step = (int64_t)gridDim.x * (kThreads / 4);
    for (int64_t quad = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 2; quad < quads; quad += step) {
        const Spot at(quad, a.cols, a.groups);
        const uint2 w = *reinterpret_cast<const uint2*>(a.codes + quad * kPackGroup + 8 * (threadIdx.x & 3));
        const float scale = pack8_scale(a.scales[quad]);
        float x[8];
        pack8_values<SIGNED>(w.x, scale, x);
        pack8_values<SIGNED>(w.y, scale, x + 4);
        store_run<T, 8, VEC>(static_cast<T*>(a.y) + at.row * a.cols + at.col, x, at.count);
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void relu_grad8(const PackArgs a) {
    const int64_t quads = a.rows * a.groups, step = (int64_t)gridDim.x * (kThreads / 4);
    for (int64_t quad = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 2; quad < quads; quad += step) {
        const Spot at(quad, a.cols, a.groups);
        const uint2 w = *reinterpret_cast<const uint2*>(a.codes + quad * kPackGroup + 8 * (threadIdx.x & 3));
        Run<T, 8> r;
        load_run<T, 8, VEC>(r, static_cast<const T*>(a.x) + at.row * a.ld + at.col, at.count);
        float x[8];
        r.to_float(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (i < 4 ? w.x : w.y) >> (8 * (i & 3)) & 0xFFu ? x[i] : 0.f;
        store_run<T, 8, VEC>(static_cast<T*>(a.y) + at.row * a.cols + at.col, x, at.count);
    }
}

unsigned grid_for(const PackArgs& a) {
    const int64_t quads = a.rows * a.groups;
    return static_cast<unsigned>(std::min<int64_t>((quads + kThreads / 4 - 1) / (kThreads / 4), 256 * 32));
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
    a.ld = ld;
    return a;
}

// Whole packets on both sides: x with rows ld apart, y contiguous.
bool whole(const PackArgs& a, int32_t dtype) {
    const int64_t size = dtype == RA_DTYPE_F32 ? 4 : 2;
    return aligned16(a.x) && aligned16(a.y) && a.cols * size % 16 == 0 && (a.rows <= 1 || a.ld * size % 16 == 0);
}

template <typename F>
void by_type(int32_t dtype, bool vec, F f) {
    auto by_vec = [&](auto tag) {
        if (vec) f(tag, std::true_type());
        else f(tag, std::false_type());
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
    ra::by_type(dtype, ra::whole(a, dtype), [&](auto tag, auto vec) {
        ra::pack8<decltype(tag), decltype(vec)::value, false><<<ra::grid_for(a), ra::kThreads, 0, st>>>(a);
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
    ra::by_type(dtype, ra::whole(a, dtype), [&](auto tag, auto vec) {
        ra::pack8<decltype(tag), decltype(vec)::value, true><<<ra::grid_for(a), ra::kThreads, 0, st>>>(a);
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
    ra::by_type(dtype, ra::whole(a, dtype), [&](auto tag, auto vec) {
        using T = decltype(tag);
        if (is_signed) ra::unpack8<T, decltype(vec)::value, true><<<ra::grid_for(a), ra::kThreads, 0, st>>>(a);
        else ra::unpack8<T, decltype(vec)::value, false><<<ra::grid_for(a), ra::kThreads, 0, st>>>(a);
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
    ra::by_type(dtype, ra::whole(a, dtype), [&](auto tag, auto vec) {
        ra::relu_grad8<decltype(tag), decltype(vec)::value><<<ra::grid_for(a), ra::kThreads, 0, st>>>(a);
    });
    RA_LAUNCH_CHECK("relu_grad8");
    return RA_OK;
}

}  // extern "C"
