// lanes.hpp — sums and maxima over aligned groups of a wave's lanes and over the waves
// of a workgroup; every lane of the group gets the result, the order is fixed.
#pragma once

#include <hip/hip_runtime.h>

#include <cfloat>
#include <cstdint>

namespace ra {

struct Add {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
    static __device__ __forceinline__ double of(double a, double b) { return a + b; }
};
struct Max {
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};

// Over groups of `lanes` (a power of two, at most 64; the same in all lanes).  Steps
// within 16 lanes are register moves of the vector unit: after those of 1 and 2 the
// lanes of a quad are equal, so mirroring 8 and 16 lanes exchanges the halves.
template <typename Op>
__device__ __forceinline__ float over_lanes(float x, int lanes) {
    auto moved = [](float v, auto ctrl) {
        return __int_as_float(
            __builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    if (lanes > 1) x = Op::of(x, moved(x, std::integral_constant<int, 0xB1>()));   // lane ^ 1
    if (lanes > 2) x = Op::of(x, moved(x, std::integral_constant<int, 0x4E>()));   // lane ^ 2
    if (lanes > 4) x = Op::of(x, moved(x, std::integral_constant<int, 0x141>()));  // 7 - lane
    if (lanes > 8) x = Op::of(x, moved(x, std::integral_constant<int, 0x140>()));  // 15 - lane
    if (lanes > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if (lanes > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return x;
}
__device__ __forceinline__ double sum_lanes(double x, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// Over the workgroup (whole waves): `part` is LDS of one value a wave, that no lane
// still reads from an earlier call.
template <typename Op>
__device__ __forceinline__ float over_workgroup(float x, float* part) {
    x = over_lanes<Op>(x, 64);
    const int waves = blockDim.x >> 6;
    if (waves == 1) return x;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = part[0];
    for (int w = 1; w < waves; ++w) x = Op::of(x, part[w]);
    return x;
}
__device__ __forceinline__ double sum_workgroup(double x, double* part) {
    x = sum_lanes(x, 64);
    const int waves = blockDim.x >> 6;
    if (waves == 1) return x;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = part[0];
    for (int w = 1; w < waves; ++w) x += part[w];
    return x;
}

}  // namespace ra
