// vector_run.hpp — a lane's run of consecutive elements of a 16- or 32-bit type,
// loaded and stored as whole packets where the addresses allow it.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ra {

using f16_t = _Float16;
using bf16_t = __bf16;


__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi, bf16_t) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
}
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi, f16_t) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 h = __builtin_bit_cast(h2, w);
    lo = (float)h[0];
    hi = (float)h[1];
}

// N (4 or 8) elements as floats.
template <typename T, int N>
struct Run {
    uint32_t w[N / 2];
    __device__ __forceinline__ void to_float(float* f) const {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) unpack2(w[i], f[2 * i], f[2 * i + 1], T());
    }
};
template <int N>
struct Run<float, N> {
    float w[N];
    __device__ __forceinline__ void to_float(float* f) const {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = w[i];
    }
};

// What lanes without an edge (or past the end of a head) load instead: zeros.
// Never written; not const, so that both addresses of the choice are global ones.
static __device__ uint4 kZeroRun[2];

// A lane's run of N elements, the first `count` of them in memory (the others are
// 0).  VEC: runs are whole packets (16 bytes, or all of a shorter run) and aligned
// to them; `count` is then 0 or covers whole packets.
template <typename T, int N, bool VEC>
__device__ __forceinline__ void load_run(Run<T, N>& r, const T* p, int count) {
    if constexpr (VEC) {
        constexpr int kPerPacket = (int)(16 / sizeof(T)) < N ? (int)(16 / sizeof(T)) : N;
        constexpr int kWords = kPerPacket * (int)sizeof(T) / 4;
#pragma unroll
        for (int i = 0; i < N / kPerPacket; ++i) {
            const void* at = i * kPerPacket < count ? static_cast<const void*>(p + i * kPerPacket)
                                                    : static_cast<const void*>(kZeroRun);
            if constexpr (kWords == 4) {
                const uint4 x = *static_cast<const uint4*>(at);
                __builtin_memcpy(&r.w[i * 4], &x, 16);
            } else {
                const uint2 x = *static_cast<const uint2*>(at);
                __builtin_memcpy(&r.w[i * 2], &x, 8);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const T x = *(i < count ? p + i : reinterpret_cast<const T*>(kZeroRun));
            if constexpr (sizeof(T) == 4) {
                r.w[i] = x;
            } else {
                const uint32_t b = __builtin_bit_cast(uint16_t, x);
                if (i & 1) r.w[i / 2] |= b << 16;
                else r.w[i / 2] = b;
            }
        }
    }
}

template <typename T, int N, bool VEC>
__device__ __forceinline__ void store_run(T* p, const float* f, int count) {
    if constexpr (VEC) {
        constexpr int kPerPacket = (int)(16 / sizeof(T)) < N ? (int)(16 / sizeof(T)) : N;
#pragma unroll
        for (int i = 0; i < N / kPerPacket; ++i) {
            if (i * kPerPacket >= count) break;
            typedef T vec __attribute__((ext_vector_type(kPerPacket)));
            vec x;
#pragma unroll
            for (int e = 0; e < kPerPacket; ++e) x[e] = (T)f[i * kPerPacket + e];
            *reinterpret_cast<vec*>(p + i * kPerPacket) = x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < count) p[i] = (T)f[i];
    }
}

}  // namespace ra
