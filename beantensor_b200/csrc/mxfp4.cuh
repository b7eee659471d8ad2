// The microscaled 4-bit format (OCP MX, MXFP4): along k, every 32 consecutive values share one power-of-two scale.
//   elements  E2M1, two per byte, even k in bits 0-3: 0, .5, 1, 1.5, 2, 3, 4, 6 and a sign in bit 3
//   scales    E8M0, one byte s = X + 127 for a block's factor 2^X; 255 is NaN
// Scales are kept in the order in which the tensor core takes them: blocks of 128 rows x 4 scales (128 k), 512 bytes
// each, block (R, C) at index R * ceil(K / 128) + C. Within a block, the scale c of row r is byte
// (r % 32) * 16 + (r / 32) * 4 + c: four 32-row bands side by side, so that 32 lanes x 16 bytes are one block. Rows of a
// grouped operand are cut per group into slots of 128 rows, and R counts the slots of all groups.
#pragma once
#include <stdint.h>

namespace btm {

constexpr int MX_BLOCK = 32;         // values per scale
constexpr int MX_CHUNK_K = 128;      // k per scale block
constexpr int MX_SCALE_BYTES = 512;  // bytes per scale block
constexpr uint32_t MX_NAN = 255u;

__host__ __device__ constexpr int mx_chunks(int K) { return (K + MX_CHUNK_K - 1) / MX_CHUNK_K; }
__host__ __device__ constexpr int mx_scale_at(int row_in_slot, int c) { return (row_in_slot & 31) * 16 + (row_in_slot >> 5) * 4 + c; }

// 2^(s - 127); s = 0 is the subnormal 2^-127, s = 255 NaN.
__device__ __forceinline__ float mx_scale_value(uint32_t s)
{
    return s == MX_NAN ? __uint_as_float(0x7FC00000u) : s == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23);
}

// Four bytes of packed codes -> eight values (even k first), exact in fp16.
__device__ __forceinline__ void mx_decode8(uint32_t packed, uint32_t (&h2)[4])
{
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h2[0]), "=r"(h2[1]), "=r"(h2[2]), "=r"(h2[3])
        : "r"(packed));
}

// Eight values -> four bytes of packed codes: round to nearest, ties to the even code, saturating at 6.
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8])
{
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

} // namespace btm
