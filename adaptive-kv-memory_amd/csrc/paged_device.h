// Device helpers shared by the attention kernels over the paged 4-bit cache.
#pragma once

#include "akv_common.h"
#include "paged.h"

namespace akv {
namespace {

constexpr float kMinMax = -0x1p126f;  // a finite start of the running maximum: a row that sees nothing stays at p = 0

// Masks of the two nibbles of a byte in both halves of a dword, in registers (so that mask and
// exponent are one v_and_or_b32), and a pair of codes less MID as float16: under the exponent of
// 1024 the low nibble reads as 1024 + c, under that of 64 the high one as 64 + c.
struct Nibbles {
    uint32_t lo, hi;
    __device__ __forceinline__ void init() {
        lo = 0x000F000Fu;
        hi = 0x00F000F0u;
        asm volatile("" : "+v"(lo), "+v"(hi));
    }
    template <int MID = 0>
    __device__ __forceinline__ h2 low(uint32_t w) const {
        return as_h2((w & lo) | 0x64006400u) - (h2){(_Float16)(1024.f + MID), (_Float16)(1024.f + MID)};
    }
    template <int MID = 0>
    __device__ __forceinline__ h2 high(uint32_t w) const {
        return as_h2((w & hi) | 0x54005400u) - (h2){(_Float16)(64.f + MID), (_Float16)(64.f + MID)};
    }
};

// The running maximum of a row whose largest score is top * kx, p being 2^(score * kx + (bias - maximum)):
// the next float above it where that exponent rounds to more than the bias, which scores past 2^23 let
// it, so that p never leaves float16.
__device__ __forceinline__ float running_max(float top, float kx, float bias) {
    const float m = top * kx;
    return __builtin_fmaf(top, kx, bias - m) > bias ? __builtin_fmaf(__builtin_fabsf(m), 0x1.8p-24f, m) : m;
}
// 1 / sum of a row's p; 0 for a row that sees nothing (and NaN stays).
__device__ __forceinline__ float row_inverse(float l) { return l > 0.0f || l != l ? 1.0f / l : 0.0f; }
// log of the sum of exp, from the maximum (log2 domain) and the sum of p times 2^bias.
__device__ __forceinline__ float row_lse(float m, float l, float bias) {
    return l > 0.0f || l != l ? 0.69314718055994531f * (m + (__builtin_log2f(l) - bias)) : -INFINITY;
}
// The halves of a pair of float16 that are not finite, as a mask.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return ((w & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((w & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}
__device__ __forceinline__ uint32_t to_pair(bool bf16, float a, float b) {
    return bf16 ? f32_to_bf16_rne(a) | ((uint32_t)f32_to_bf16_rne(b) << 16) : as_u32((h2){(_Float16)a, (_Float16)b});
}

}  // namespace
}  // namespace akv
