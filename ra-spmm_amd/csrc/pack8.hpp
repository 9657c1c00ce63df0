// pack8.hpp — the 8-bit format as its kernels share it (include/ra_spmm.h).
#pragma once

#include <algorithm>

#include "ra_internal.hpp"

namespace ra {

constexpr int kPackGroup = 32;  // columns of a scale

inline int32_t pack8_groups(int32_t cols) { return static_cast<int32_t>(((int64_t)cols + kPackGroup - 1) / kPackGroup); }

// Bytes between the groups' scales: one per row, padded to 8.
inline int64_t pack8_scale_pitch(int64_t rows) { return (rows + 7) / 8 * 8; }

// Scale of a byte: 2^(byte - 127), NaN for 255.
__device__ __forceinline__ float pack8_scale(uint32_t byte) {
    return __uint_as_float(byte << 23 | (byte == 255u ? 0x400000u : 0u));
}

// The four codes of a word times the scale: exact.
template <bool SIGNED>
__device__ __forceinline__ void pack8_values(uint32_t w, float scale, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float c = SIGNED ? static_cast<float>(static_cast<int8_t>(w >> (8 * i)))
                               : static_cast<float>(w >> (8 * i) & 0xFFu);
        x[i] = c * scale;
    }
}

}  // namespace ra
