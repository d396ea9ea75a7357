// MXFP4 (OCP microscaling formats, 4-bit): blocks of 32 values share a scale 2^e (E8M0: the byte e + 127, 255 for NaN), an
// element is E2M1: sign, 2 bits of exponent, 1 of mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6).
#pragma once

#include "frx_common.cuh"

namespace frx {

constexpr int kMxBlock = 32;       // values that share a scale
constexpr int kMxTileRows = 128;   // matrix rows of a tile: the M of the tensor core's instruction
constexpr int kMxUnitK = 128;      // columns of a unit: four scales a row, one 32-bit word
constexpr int kMxUnitCode = kMxTileRows * kMxUnitK / 2;
constexpr int kMxUnitBytes = kMxUnitCode + kMxTileRows * kMxUnitK / kMxBlock;   // 8192 + 512

// The scale byte of a block whose largest magnitude has these bits: 2^(floor(log2(amax)) - 2), so that the largest element lies in
// [4, 8), at least 2^-127 (a subnormal amax, whose exponent field is 0, comes out there too). NaN or infinity in the block: NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 1 / scale: 2^(127 - byte), exact for every byte up to 253
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : byte ? byte << 23 : 0x00400000u); }

// Eight values, already divided by their scale, to eight elements, the first in the low nibble: to nearest, ties to even,
// magnitudes beyond 6 to 6 (the one rounding of the format; the division by a power of two before it is exact, or
// falls below the smallest half step, 0.25, where the element is 0 either way).
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// and back, as values of the elements alone
__device__ __forceinline__ void mx_values8(uint32_t codes, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

}  // namespace frx
