#pragma once
// The microscaled 4-bit formats of minicompiler_b200_device.h as the kernels see them: geometry of the two arrays,
// conversions of codes and scales. Included by the kernels that write them (fp4_quantize.cu) and read them
// (fp4_gemm.cu, moe_layer.cu).

#include "minicompiler_b200_device.h"

namespace mcd {

constexpr int kFp4TileBytes = 512;  // scales of 128 rows x 4 blocks

struct Fp4Geometry {
    int block;                 // columns per scale
    long long blocks;          // per row
    long long pitch;           // bytes of codes per row
    long long row_tiles;       // groups of 128 rows
    long long k_tiles;         // groups of 4 blocks
    long long matrix_codes;    // bytes per matrix
    long long matrix_scales;
};

inline Fp4Geometry fp4_geometry(int format, long long rows, long long cols) {
    Fp4Geometry g;
    g.block = format == MCD_FP4_E8M0_32 ? 32 : 16;
    g.blocks = (cols + g.block - 1) / g.block;
    g.pitch = (cols + 31) / 32 * 16;
    g.row_tiles = (rows + 127) / 128;
    g.k_tiles = (g.blocks + 3) / 4;
    g.matrix_codes = rows * g.pitch;
    g.matrix_scales = g.row_tiles * g.k_tiles * kFp4TileBytes;
    return g;
}

#ifdef __CUDACC__

// Byte of row r, block b inside one matrix's scales.
__device__ __forceinline__ long long fp4_scale_offset(long long r, long long b, long long k_tiles) {
    return ((r >> 7) * k_tiles + (b >> 2)) * kFp4TileBytes + ((r & 31) << 4) + (((r >> 5) & 3) << 2) + (b & 3);
}

// The conversions below take words apart, and put them together, by vector moves of 8- and 16-bit registers: the compiler
// then lets the conversion itself pick its byte. With shifts and masks instead, eight codes take 12 integer
// instructions where these take 4 (10.5 against 5.3 words per cycle and SM).

// Eight codes from v[0 .. 7], round to nearest even, magnitudes over 6 become 6; v[0] goes to the lowest four bits.
__device__ __forceinline__ unsigned fp4_encode8(const float* v) {
    unsigned r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// The values of the eight codes of a word as four f16 pairs, the lowest four bits in the low half of the first.
__device__ __forceinline__ void fp4_decode8(unsigned word, unsigned (&pairs)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(pairs[0]), "=r"(pairs[1]), "=r"(pairs[2]), "=r"(pairs[3])
        : "r"(word));
}

__device__ __forceinline__ float f16_lo(unsigned h2) {
    float f;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.f32.f16 %0, a;\n\t}" : "=f"(f) : "r"(h2));
    return f;
}
__device__ __forceinline__ float f16_hi(unsigned h2) {
    float f;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.f32.f16 %0, b;\n\t}" : "=f"(f) : "r"(h2));
    return f;
}

// t >= 0 to e4m3, nearest even, at most 448.
__device__ __forceinline__ unsigned e4m3_encode(float t) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(t));
    return r & 0xffu;
}
__device__ __forceinline__ float e4m3_decode(unsigned byte) {
    unsigned h2;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h2) : "r"(byte & 0xffu));
    return f16_lo(h2);
}

// 2^(byte - 127); 255 stands for NaN.
__device__ __forceinline__ float e8m0_decode(unsigned byte) {
    const unsigned bits = byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23;
    return __uint_as_float(bits);
}

// A value times a * b, where a * b need not be a number that f32 holds well although the result is: one factor where it is,
// otherwise a and b one behind the other. They then lie on the same side of 1, so that the way there leaves f32 only where
// the result does.
struct TwoFactors {
    float first, second;
    __device__ __forceinline__ float times(float v) const { return v * first * second; }
};
__device__ __forceinline__ TwoFactors two_factors(float a, float b) {
    const float both = a * b;
    return fabsf(both) >= 1.17549435e-38f && fabsf(both) <= 3.402823466e38f ? TwoFactors{both, 1.0f} : TwoFactors{a, b};
}

#endif

}  // namespace mcd
