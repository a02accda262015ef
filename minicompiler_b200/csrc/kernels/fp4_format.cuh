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

// Two codes, round to nearest even, magnitudes over 6 become 6; `lo` goes to the low four bits.
__device__ __forceinline__ unsigned fp4_encode2(float lo, float hi) {
    unsigned r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The values of the two codes of the low byte, as packed f16 (the low half holds the low four bits).
__device__ __forceinline__ unsigned fp4_decode2(unsigned byte) {
    unsigned r;
    asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(r) : "r"(byte));
    return r;
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

#endif

}  // namespace mcd
