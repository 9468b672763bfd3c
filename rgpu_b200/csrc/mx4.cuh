// Device helpers of the microscaled 4-bit format (OCP microscaling
// specification 1.0, MXFP4: E2M1 elements, E8M0 scale per 32).
#pragma once

#include <cstdint>

#include "internal.h"

namespace rt {
namespace mx4 {

constexpr uint32_t kNanScale = 255;

// Scale byte of a block from the bit pattern of its largest magnitude:
// floor(log2 amax) is the exponent field less 127, the largest element (6) has
// exponent 2, so byte = field - 2 with 0 (2^-127) the least.  An infinity or a
// NaN has field 255 and takes the NaN scale.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    const int field = (int)(amax_bits >> 23);
    if (field == 255) return kNanScale;
    return field > 2 ? (uint32_t)(field - 2) : 0u;
}

// 2^(127 - byte), what the elements are multiplied by: exponent field
// 254 - byte, at least 1 for every byte below 254 (scale_byte gives at most
// 252, so the factor is a normal number; the NaN scale gives 0, not used).
__device__ __forceinline__ float inv_scale(uint32_t byte) {
    return __uint_as_float((byte == kNanScale ? 0u : 254u - byte) << 23);
}

// Two elements to E2M1 codes in one byte (lo in bits 0-3): round to nearest,
// ties to even, magnitudes above 6 to 6.
__device__ __forceinline__ uint32_t encode2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 c;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %1, %2;\n\t"
        "cvt.u32.u8 %0, c;\n\t}"
        : "=r"(r)
        : "f"(hi), "f"(lo));
    return r;
}

// Eight elements to eight codes (element i in bits
// 4i), each times `inv`.
__device__ __forceinline__ uint32_t encode8(const float (&v)[8], float inv) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv),
          "f"(v[6] * inv), "f"(v[7] * inv));
    return r;
}

// Byte offset of the scale of (row, block) in a matrix of `groups` scale
// tiles along k.
__device__ __forceinline__ int64_t scale_offset(int64_t row, int64_t block, int64_t groups) {
    const int r = (int)(row & 127);
    return ((row >> 7) * groups + (block >> 2)) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (block & 3);
}

}  // namespace mx4
}  // namespace rt
