#pragma once
// The block-scaled tensor-core instructions of sm_100a and their operands: descriptors of 4-bit tiles and of scales in
// shared memory, copies of scales into TMEM, the multiply itself. Used by fp4_gemm.cu.

#include "kernels/async_copy.cuh"
#include "kernels/fp4_format.cuh"

namespace mcd {

// A tile row in shared memory is 128 bytes = 256 codes: one K block. An instruction takes 64 of them (32 bytes).
constexpr int kFp4BlockK = 256;
constexpr int kFp4MmaK = 64;

// K-major operand tile: rows of 128 bytes with the 128-byte swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ unsigned long long fp4_tile_desc(unsigned addr) {
    return static_cast<unsigned long long>((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<unsigned long long>(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}

// 512 bytes of scales: 32 rows of 16 bytes without a swizzle, groups of 8 rows 128 bytes apart.
__device__ __forceinline__ unsigned long long fp4_scale_desc(unsigned addr) {
    return static_cast<unsigned long long>((addr & 0x3FFFFu) >> 4) | (static_cast<unsigned long long>(128 >> 4) << 32) | (1ull << 46);
}

// Instruction descriptor: e2m1 for both operands, both K-major, dense; the scales' type, N and M.
template <int kFormat>
constexpr unsigned fp4_instruction(int m, int n) {
    return (1u << 7) | (1u << 10) | (static_cast<unsigned>(n >> 3) << 17) | ((kFormat == MCD_FP4_E8M0_32 ? 1u : 0u) << 23) |
           (static_cast<unsigned>(m >> 4) << 24);
}
// With 32 columns per scale an instruction needs two of the four scales that a TMEM column holds: 0, 1 or 2, 3.
constexpr unsigned kFp4UpperScales = (2u << 4) | (2u << 29);

// One scale tile into four TMEM columns, repeated for the four groups of 32 lanes.
template <int kGroup>
__device__ __forceinline__ void fp4_scales_to_tmem(unsigned taddr, unsigned long long desc) {
    if constexpr (kGroup == 1) {
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    } else {
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    }
}

template <int kFormat, int kGroup>
__device__ __forceinline__ void fp4_mma(unsigned tmem_d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned scale_a,
                                        unsigned scale_b, unsigned accumulate) {
#define MC_FP4_MMA(group, kind)                                                                                            \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::" group ".kind::" kind             \
                 " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),                                                   \
                 "l"(a), "l"(b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate)                                   \
                 : "memory")
    if constexpr (kFormat == MCD_FP4_E8M0_32) {
        if constexpr (kGroup == 1) {
            MC_FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
        } else {
            MC_FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
        }
    } else {
        if constexpr (kGroup == 1) {
            MC_FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
        } else {
            MC_FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
        }
    }
#undef MC_FP4_MMA
}

__device__ __forceinline__ void fp4_commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void fp4_bulk_load(unsigned smem_dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

__device__ __forceinline__ void tmem_load16(unsigned taddr, unsigned* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}

}  // namespace mcd
