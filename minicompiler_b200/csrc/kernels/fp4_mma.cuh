#pragma once
// The block-scaled tensor-core instructions of sm_100a and their operands: descriptors of 4-bit tiles and of scales in
// shared memory, copies of scales into TMEM, the multiply itself. Used by fp4_gemm.cu.

#include "kernels/async_copy.cuh"
#include "kernels/fp4_format.cuh"

namespace mcd {

// A tile row in shared memory is 128 bytes = 256 codes: one K block. An instruction takes 64 of them (32 bytes).
constexpr int kFp4BlockK = 256;
constexpr int kFp4MmaK = 64;

// K-major operand tile: rows of 128 bytes with the 128-byte swizzle, groups of 8 rows `apart` bytes from one another.
__device__ __forceinline__ unsigned long long fp4_tile_desc(unsigned addr, unsigned apart) {
    return static_cast<unsigned long long>((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<unsigned long long>(apart >> 4) << 32) |
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
__device__ __forceinline__ void fp4_scales_to_tmem(unsigned taddr, unsigned long long desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
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

// The same for an SM pair, the CTAs `first` and `first` + 1 of the cluster: arrives on the barrier at this offset in both.
__device__ __forceinline__ void fp4_commit_pair(unsigned bar, unsigned first) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<unsigned short>(3u << first))
                 : "memory");
}

// The address of `addr` (in this CTA's shared memory) in CTA `rank` of the cluster.
__device__ __forceinline__ unsigned cluster_address(unsigned addr, unsigned rank) {
    unsigned out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
    return out;
}
// One look at a barrier, without waiting.
__device__ __forceinline__ bool mbar_test(unsigned bar, unsigned parity) {
    unsigned done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ void mbar_arrive_cluster(unsigned cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// TMA loads into this CTA whose bytes are counted on a barrier of either CTA of the pair (no multicast).
__device__ __forceinline__ void tma_load_2d_pair(unsigned smem_dst, const McTensorMap* map, unsigned bar_cluster_addr, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_dst),
        "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar_cluster_addr), "r"(c0), "r"(c1)
        : "memory");
}
// A three-dimensional box, counted on a barrier of this CTA.
__device__ __forceinline__ void tma_load_3d(unsigned smem_dst, const McTensorMap* map, unsigned bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_dst),
        "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(unsigned smem_dst, const McTensorMap* map, unsigned bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_dst),
        "l"(reinterpret_cast<unsigned long long>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}
// One box out of shared memory; what lies outside the tensor is not written.
__device__ __forceinline__ void tma_store_2d(const McTensorMap* map, unsigned smem_src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<unsigned long long>(map)),
                 "r"(smem_src), "r"(c0), "r"(c1)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int kPending>
__device__ __forceinline__ void tma_store_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPending) : "memory");
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

__device__ __forceinline__ void load_shared_v4(unsigned addr, unsigned* v) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void tmem_store8(unsigned taddr, const unsigned* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ void tmem_load32(unsigned taddr, unsigned* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}

}  // namespace mcd
