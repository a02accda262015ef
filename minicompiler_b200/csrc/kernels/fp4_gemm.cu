// mcd_fp4_gemm: C[m,n] = A[m,k] * B[n,k]^T with both operands in a microscaled 4-bit format, on the tensor cores'
// block-scaled multiply (tcgen05.mma kind::mxf4 / kind::mxf4nvf4). The products code * code and the scales are exact in
// the multiplier; sums are f32.
//
//   sum over k of (a b) = sum over blocks of s_a s_b * (sum over the block of code_a code_b)
//
// An instruction covers 64 columns of k; the scales it needs lie in TMEM, brought there from shared memory. One CTA per
// tile: by tcgen05.cp, which the tensor core executes in order with the multiplies behind it. SM pairs, which multiply
// without a pause: by warps of their own.

#include "minicompiler_b200_device.h"

#include "device/driver_api.hpp"
#include "kernels/fp4_host.hpp"
#include "kernels/fp4_mma.cuh"

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

using namespace mcd;

namespace {

#define MC_FP4_ERR_PRODUCER 0x100u
#define MC_FP4_ERR_MMA 0x200u
#define MC_FP4_ERR_EPILOGUE 0x400u
#define MC_FP4_ERR_DRAIN 0x800u
#define MC_FP4_ERR_SCALES 0x1000u

constexpr int kTileRows = 128;   // TMEM lanes
constexpr int kRaster = 16;      // row tiles per band of work items
constexpr int kMaxCluster = 8;   // K slices that a cluster adds up

struct Fp4GemmParams {
    // "rows" is the operand on the 128 TMEM lanes, "columns" the one whose rows are accumulator columns
    const unsigned char* row_scales;
    const unsigned char* col_scales;
    long long k_tiles;  // scale tiles per 128 rows
    const float* row_scale;  // tensor scales, may be null
    const float* col_scale;
    void* c;
    float* workspace;
    unsigned* status;
    long long ldc;
    int c_type;
    int rows, cols, k;
    int k_blocks, k_blocks_per_split, splits;
    int swapped;    // 0: rows are C's rows; 1: rows are C's columns
    int wide;       // the row operand's map is the four-dimensional one
    int clustered;  // the K slices of a tile are the CTAs of a cluster, one item per CTA, and are added up there
};

__device__ __forceinline__ void store_c(void* c, int type, long long at, float v) {
    if (type == MCD_TYPE_F32) {
        static_cast<float*>(c)[at] = v;
    } else {
        unsigned short h;
        if (type == MCD_HALF_BF16) {
            asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(h) : "f"(v));
        } else {
            asm("cvt.rn.f16.f32 %0, %1;" : "=h"(h) : "f"(v));
        }
        static_cast<unsigned short*>(c)[at] = h;
    }
}

__device__ __forceinline__ unsigned pack_half2(float lo, float hi, int type) {
    unsigned d;
    if (type == MCD_HALF_BF16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    }
    return d;
}

// 16 neighbouring values of a row, 16-byte aligned.
__device__ __forceinline__ void store_row16(void* c, int type, long long at, const float (&f)[16]) {
    if (type == MCD_TYPE_F32) {
        auto* to = reinterpret_cast<float4*>(static_cast<float*>(c) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) to[j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
    } else {
        auto* to = reinterpret_cast<uint4*>(static_cast<unsigned short*>(c) + at);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float* q = f + 8 * j;
            to[j] = make_uint4(pack_half2(q[0], q[1], type), pack_half2(q[2], q[3], type), pack_half2(q[4], q[5], type), pack_half2(q[6], q[7], type));
        }
    }
}

// Four values at `at`, `at + step`, ...; step 1 and `vec`: aligned for one store. `left` of them exist.
__device__ __forceinline__ void store_quad(void* c, int type, long long at, long long step, const float (&f)[4], bool vec, int left) {
    if (vec && left >= 4) {
        if (type == MCD_TYPE_F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(c) + at) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
            *reinterpret_cast<uint2*>(static_cast<unsigned short*>(c) + at) = make_uint2(pack_half2(f[0], f[1], type), pack_half2(f[2], f[3], type));
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j < left) store_c(c, type, at + j * step, f[j]);
    }
}

__device__ __forceinline__ TwoFactors product_scale(const float* a, const float* b) {
    return two_factors(a != nullptr ? *a : 1.0f, b != nullptr ? *b : 1.0f);
}

// ------------------------------------------------------------------------------------------------ one CTA per tile
//
// 128 rows x kCols columns, K in blocks of 256 codes (128 bytes per tile row), kBlocks of them per stage. Warp 0 brings
// tiles and scales into a ring of stages, warp 1 issues copies of scales and multiplies, warps 2-5 drain one of two
// accumulators while the other is being filled.
//
// What bounds it: few columns, that is few tokens, read the whole of the row operand once (16384 x 16384 E8M0_32 codes,
// 143 MB: 41 to 50 us on different machines; bringing them to shared memory and nothing else took 33, in one run or not, most
// of the rest is the ramp of one wave of CTAs). Neither the multiplies nor the copies of scales are felt. A stage takes two
// or four K blocks, and one four-dimensional TMA box brings them in the order 8 rows x 128 bytes, the next 128 bytes of
// the same rows, ..., the next 8 rows (64 tokens, 8192 x 8192, K whole: 16.0 us, 16.9 block by block). In shared memory the 1024-byte
// atoms of a K block are then kBlocks apart, which is a stride of the operand descriptor. Matrices whose rows are no
// multiple of 8, or whose row pitch is none of 128 bytes, go block by block (such a box could reach past the end of the
// last row).

template <int kFormat, int kCols>
struct Fp4Tile {
    static constexpr int kBlocks = kCols <= 32 ? 4 : 2;
    static constexpr int kScaleTiles = kFormat == MCD_FP4_E8M0_32 ? 2 : 4;  // per K block
    static constexpr int kRowBytes = kTileRows * 128;                       // per K block, as the next two
    static constexpr int kColBytes = kCols * 128;
    static constexpr int kScaleBytes = kScaleTiles * kFp4TileBytes;
    static constexpr int kStageBytes = kBlocks * (kRowBytes + kColBytes + 2 * kScaleBytes);
    static constexpr int kStages = 221184 / kStageBytes;
    static constexpr int kBarrierBytes = 512;
    static constexpr int kTurnBytes = 4 * 32 * 17 * 4;  // see the epilogue
    static constexpr int kSmem = kStages * kStageBytes + 1024 + kBarrierBytes + kTurnBytes;
    static constexpr int kAccColumns = kCols < 32 ? 32 : kCols;
    static constexpr int kScaleColumns = kScaleTiles * 4;
    static constexpr int kScaleBase = 2 * kAccColumns;
    static_assert(kStages >= 2, "a ring");
    static_assert(kScaleBase + kStages * kBlocks * 2 * kScaleColumns <= 512, "TMEM columns");
    static_assert(kStages * 16 + 32 <= kBarrierBytes, "barriers");
};

constexpr int kOneCtaThreads = 64 + 128;

__device__ __forceinline__ void fp4_decode_item(int item, int tiles_r, int tiles_c, int splits, int& rb, int& cb, int& split) {
    split = item % splits;
    const int tile = item / splits;
    const int band_tiles = kRaster * tiles_c;
    const int band = tile / band_tiles;
    const int first = band * kRaster;
    const int band_rows = min(kRaster, tiles_r - first);
    const int within = tile - band * band_tiles;
    rb = first + within % band_rows;
    cb = within / band_rows;
}

template <int kFormat, int kCols>
__global__ void __launch_bounds__(kOneCtaThreads, 1)
mc_fp4_gemm(const __grid_constant__ McTensorMap map_rows, const __grid_constant__ McTensorMap map_cols, const Fp4GemmParams p) {
    using Tile = Fp4Tile<kFormat, kCols>;
    constexpr int stages = Tile::kStages;
    extern __shared__ unsigned char smem_raw[];
    const unsigned tiles_base = (mc_smem_addr(smem_raw) + 1023u) & ~1023u;
    const unsigned bars = tiles_base + stages * Tile::kStageBytes;
    const unsigned bar_full = bars, bar_empty = bars + 8 * stages, bar_acc_full = bars + 16 * stages, bar_acc_empty = bar_acc_full + 16;
    __shared__ unsigned tmem_slot;
    __shared__ int abort_storage;
    volatile int* abort_flag = &abort_storage;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tiles_r = (p.rows + kTileRows - 1) / kTileRows;
    const int tiles_c = (p.cols + kCols - 1) / kCols;
    const int items = tiles_r * tiles_c * p.splits;

    if (threadIdx.x == 0) {
        abort_storage = 0;
        for (int s = 0; s < stages; ++s) {
            mc_mbar_init(bar_full + 8 * s, 1);
            mc_mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mc_mbar_init(bar_acc_full + 8 * a, 1);
            mc_mbar_init(bar_acc_empty + 8 * a, 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mc_smem_addr(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_slot;
    // A programmatic dependent of the launch before it: global memory is touched only once that launch is complete.
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0, issued = 0;
            unsigned phase = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
                int rb, cb, split;
                fp4_decode_item(item, tiles_r, tiles_c, p.splits, rb, cb, split);
                const int kb_begin = split * p.k_blocks_per_split;
                const int kb_end = min(p.k_blocks, kb_begin + p.k_blocks_per_split);
                const unsigned char* row_scales = p.row_scales + rb * p.k_tiles * kFp4TileBytes;
                const unsigned char* col_scales = p.col_scales + (cb * kCols >> 7) * p.k_tiles * kFp4TileBytes;
                for (int kb = kb_begin; kb < kb_end; kb += Tile::kBlocks) {
                    ok = mc_mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.status, MC_FP4_ERR_PRODUCER);
                    if (!ok) break;
                    const unsigned full = bar_full + 8 * stage;
                    const unsigned rows_dst = tiles_base + stage * Tile::kStageBytes;
                    const unsigned cols_dst = rows_dst + Tile::kBlocks * Tile::kRowBytes;
                    const unsigned scales_dst = cols_dst + Tile::kBlocks * Tile::kColBytes;
                    const int blocks = min(Tile::kBlocks, kb_end - kb);
                    const int kt = kb * Tile::kScaleTiles;
                    const unsigned scale_bytes =
                        static_cast<unsigned>(min(static_cast<long long>(blocks * Tile::kScaleTiles), p.k_tiles - kt)) * kFp4TileBytes;
                    // a wide box counts whole, whatever of it lies outside the matrix
                    mc_mbar_expect_tx(full, (p.wide ? Tile::kBlocks : blocks) * Tile::kRowBytes + blocks * Tile::kColBytes + 2 * scale_bytes);
                    if (p.wide) {
                        tma_load_4d(rows_dst, &map_rows, full, 0, 0, kb, rb * (kTileRows / 8));
                    } else {
                        for (int i = 0; i < blocks; ++i) mc_tma_load_2d(rows_dst + i * Tile::kRowBytes, &map_rows, full, (kb + i) * 128, rb * kTileRows);
                    }
                    for (int i = 0; i < blocks; ++i) mc_tma_load_2d(cols_dst + i * Tile::kColBytes, &map_cols, full, (kb + i) * 128, cb * kCols);
                    fp4_bulk_load(scales_dst, row_scales + static_cast<long long>(kt) * kFp4TileBytes, scale_bytes, full);
                    fp4_bulk_load(scales_dst + Tile::kBlocks * Tile::kScaleBytes, col_scales + static_cast<long long>(kt) * kFp4TileBytes, scale_bytes,
                                  full);
                    ++issued;
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok) {
                // copies in flight land before shared memory is given up
                const int pending = min(issued, stages);
                for (int i = 0; i < pending; ++i) {
                    if (stage == 0) {
                        stage = stages;
                        phase ^= 1u;
                    }
                    --stage;
                    const unsigned long long t0 = mc_globaltimer();
                    while (!mc_mbar_try_wait(bar_full + 8 * stage, phase)) {
                        if (mc_globaltimer() - t0 > MC_WAIT_NS / 4) {
                            if (p.status != nullptr) atomicOr(p.status, MC_FP4_ERR_DRAIN);
                            break;
                        }
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr unsigned idesc = fp4_instruction<kFormat>(kTileRows, kCols);
            int stage = 0, acc = 0;
            unsigned phase = 0, acc_phase = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
                int rb, cb, split;
                fp4_decode_item(item, tiles_r, tiles_c, p.splits, rb, cb, split);
                const int kb_begin = split * p.k_blocks_per_split;
                const int kb_end = min(p.k_blocks, kb_begin + p.k_blocks_per_split);
                ok = mc_mbar_wait(bar_acc_empty + 8 * acc, acc_phase ^ 1u, abort_flag, p.status, MC_FP4_ERR_MMA);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned tmem_d = tmem + static_cast<unsigned>(acc * Tile::kAccColumns);
                for (int kb = kb_begin; kb < kb_end; kb += Tile::kBlocks) {
                    ok = mc_mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status, MC_FP4_ERR_MMA);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned rows_src = tiles_base + stage * Tile::kStageBytes;
                    const unsigned cols_src = rows_src + Tile::kBlocks * Tile::kRowBytes;
                    const unsigned scales_src = cols_src + Tile::kBlocks * Tile::kColBytes;
                    const unsigned scale_r = tmem + Tile::kScaleBase + static_cast<unsigned>(stage * Tile::kBlocks * 2 * Tile::kScaleColumns);
                    const unsigned scale_c = scale_r + Tile::kBlocks * Tile::kScaleColumns;
                    // Behind the last column there are no scale tiles: those instructions are left out (the codes there are
                    // 0, but what lies in the scales' place could be a NaN).
                    const int left = min(p.k, kb_end * kFp4BlockK) - kb * kFp4BlockK;
                    const int all_steps = (left + kFp4MmaK - 1) / kFp4MmaK;
#pragma unroll
                    for (int i = 0; i < Tile::kBlocks; ++i) {
                        const int steps = min(kFp4BlockK / kFp4MmaK, all_steps - i * (kFp4BlockK / kFp4MmaK));
#pragma unroll
                        for (int t = 0; t < Tile::kScaleTiles; ++t) {
                            const int tile = i * Tile::kScaleTiles + t;
                            if (t * (kFp4BlockK / kFp4MmaK / Tile::kScaleTiles) < steps) {
                                fp4_scales_to_tmem(scale_r + 4 * tile, fp4_scale_desc(scales_src + tile * kFp4TileBytes));
                                fp4_scales_to_tmem(scale_c + 4 * tile,
                                                      fp4_scale_desc(scales_src + (Tile::kBlocks * Tile::kScaleTiles + tile) * kFp4TileBytes));
                            }
                        }
                        const unsigned long long desc_r = p.wide ? fp4_tile_desc(rows_src + i * 1024, Tile::kBlocks * 1024)
                                                                 : fp4_tile_desc(rows_src + i * Tile::kRowBytes, 1024);
                        const unsigned long long desc_c = fp4_tile_desc(cols_src + i * Tile::kColBytes, 1024);
#pragma unroll
                        for (int ks = 0; ks < kFp4BlockK / kFp4MmaK; ++ks) {
                            if (ks < steps) {
                                const int tile = i * Tile::kScaleTiles + (kFormat == MCD_FP4_E8M0_32 ? ks >> 1 : ks);
                                const unsigned which = kFormat == MCD_FP4_E8M0_32 && (ks & 1) ? kFp4UpperScales : 0u;
                                fp4_mma<kFormat, 1>(tmem_d, desc_r + 2 * ks, desc_c + 2 * ks, idesc | which, scale_r + 4 * tile, scale_c + 4 * tile,
                                                    (kb > kb_begin || i > 0 || ks > 0) ? 1u : 0u);
                            }
                        }
                    }
                    fp4_commit(bar_empty + 8 * stage);
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                fp4_commit(bar_acc_full + 8 * acc);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1u;
            }
        }
    } else {
        const int quarter = warp & 3;
        constexpr int kChunk = 16;
        float* turn = reinterpret_cast<float*>(smem_raw + (tiles_base - mc_smem_addr(smem_raw)) + stages * Tile::kStageBytes + Tile::kBarrierBytes) + quarter * 32 * 17;
        const TwoFactors alpha = product_scale(p.row_scale, p.col_scale);
        int acc = 0;
        unsigned acc_phase = 0;
        bool ok = true;
        const long long m = p.swapped ? p.cols : p.rows;
        const long long n = p.swapped ? p.rows : p.cols;
        for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
            int rb, cb, split;
            fp4_decode_item(item, tiles_r, tiles_c, p.splits, rb, cb, split);
            ok = mc_mbar_wait(bar_acc_full + 8 * acc, acc_phase, abort_flag, p.status, MC_FP4_ERR_EPILOGUE);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int row = rb * kTileRows + quarter * 32 + lane;
            if (p.clustered) {
                // This CTA's multiplies are done, and with them its ring: the slice goes there, column by column.
                for (int chunk = 0; chunk < kCols / kChunk; ++chunk) {
                    unsigned v[kChunk];
                    tmem_load16(tmem + (static_cast<unsigned>(quarter * 32) << 16) + static_cast<unsigned>(chunk * kChunk), v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) {
                        asm volatile("st.shared.b32 [%0], %1;" ::"r"(tiles_base + static_cast<unsigned>((chunk * kChunk + j) * kTileRows + quarter * 32 + lane) * 4u),
                                     "r"(v[j])
                                     : "memory");
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                break;
            }
            const bool partial = p.splits > 1;
            void* dst = partial ? static_cast<void*>(p.workspace + split * m * n) : p.c;
            const long long ld = partial ? n : p.ldc;
            const int type = partial ? MCD_TYPE_F32 : p.c_type;
            const TwoFactors scale = partial ? TwoFactors{1.0f, 1.0f} : alpha;
            // rows of C that start on 16-byte boundaries leave in pieces of that size
            const bool vec = !p.swapped && (reinterpret_cast<unsigned long long>(dst) & 15) == 0 && (ld & (type == MCD_TYPE_F32 ? 3 : 7)) == 0;
            for (int chunk = 0; chunk < kCols / kChunk; ++chunk) {
                const int col0 = cb * kCols + chunk * kChunk;
                if (col0 >= p.cols) break;
                unsigned v[kChunk];
                tmem_load16(tmem + (static_cast<unsigned>(quarter * 32) << 16) + static_cast<unsigned>(acc * Tile::kAccColumns + chunk * kChunk), v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (row < p.rows && vec && col0 + kChunk <= p.cols) {
                    float f[kChunk];
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) f[j] = scale.times(__uint_as_float(v[j]));
                    store_row16(dst, type, static_cast<long long>(row) * ld + col0, f);
                } else if (p.swapped) {
                    if (row < p.rows) {
#pragma unroll
                        for (int j = 0; j < kChunk; ++j) {
                            if (col0 + j < p.cols) store_c(dst, type, static_cast<long long>(col0 + j) * ld + row, scale.times(__uint_as_float(v[j])));
                        }
                    }
                }
                if (!p.swapped && !(vec && col0 + kChunk <= p.cols)) {
                    // Rows of C that start anywhere: turned round in shared memory, so that half a warp writes a row's 16 values
                    // (65536 x 100 of them, one thread a row: 77 us, this way 37).
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < kChunk; ++j) turn[lane * 17 + j] = scale.times(__uint_as_float(v[j]));
                    __syncwarp();
                    const int c = col0 + (lane & 15);
                    const int first = row - lane + (lane >> 4);
#pragma unroll 1
                    for (int i = 0; i < 16; i += 8) {
                        float value[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) value[j] = turn[(2 * (i + j) + (lane >> 4)) * 17 + (lane & 15)];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int r = first + 2 * (i + j);
                            if (r < p.rows && c < p.cols) store_c(dst, type, static_cast<long long>(r) * ld + c, value[j]);
                        }
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mc_mbar_arrive(bar_acc_empty + 8 * acc);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1u;
        }
    }

    if (p.clustered) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        // Every CTA finishes its share of the columns, four rows of a column per thread: slices in their order.
        int rb, cb, rank;
        fp4_decode_item(blockIdx.x, tiles_r, tiles_c, p.splits, rb, cb, rank);
        const TwoFactors alpha = product_scale(p.row_scale, p.col_scale);
        const int valid = min(kCols, p.cols - cb * kCols);
        const int share = (valid + p.splits - 1) / p.splits;
        const int first = rank * share;
        const int quads = max(0, min(share, valid - first)) * (kTileRows / 4);
        const int bytes = p.c_type == MCD_TYPE_F32 ? 4 : 2;
        const bool vec = p.swapped && ((reinterpret_cast<unsigned long long>(p.c) | static_cast<unsigned long long>(p.ldc * bytes)) & (4 * bytes - 1)) == 0;
        constexpr int kAtOnce = 2;  // quads per thread and turn
        for (int base = threadIdx.x; base < quads; base += kAtOnce * kOneCtaThreads) {
            float4 part[kAtOnce][kMaxCluster];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const unsigned at = tiles_base + static_cast<unsigned>(first * (kTileRows / 4) + min(base + u * kOneCtaThreads, quads - 1)) * 16u;
#pragma unroll
                for (int z = 0; z < kMaxCluster; ++z) {
                    if (z < p.splits) {
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(part[u][z].x), "=f"(part[u][z].y), "=f"(part[u][z].z), "=f"(part[u][z].w)
                                     : "r"(cluster_address(at, static_cast<unsigned>(z)))
                                     : "memory");
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int q = base + u * kOneCtaThreads;
                const int row = rb * kTileRows + q % (kTileRows / 4) * 4, col = cb * kCols + first + q / (kTileRows / 4);
                if (q >= quads || row >= p.rows) continue;
                float sum[4] = {part[u][0].x, part[u][0].y, part[u][0].z, part[u][0].w};
#pragma unroll
                for (int z = 1; z < kMaxCluster; ++z) {
                    if (z < p.splits) sum[0] += part[u][z].x, sum[1] += part[u][z].y, sum[2] += part[u][z].z, sum[3] += part[u][z].w;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = alpha.times(sum[j]);
                store_quad(p.c, p.c_type, p.swapped ? static_cast<long long>(col) * p.ldc + row : static_cast<long long>(row) * p.ldc + col,
                           p.swapped ? 1 : p.ldc, sum, vec, p.rows - row);
            }
        }
        // shared memory stays until the last of the cluster has read it
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// --------------------------------------------------------------------------------------------- an SM pair per tile
//
// Two CTAs of a cluster own 256 x 256 of C, or a slice of K of it (see the rule at the host side): each stages its own 128 rows of A, its own 128 of the 256 rows of B, the
// scales of its rows of A and of all 256 rows of B; the leader's cta_group::2 instructions read both CTAs' shared memory
// and leave each CTA's 128 rows in its TMEM.
//
// TMEM: two accumulators of 256 columns and the scales do not fit into 512 columns, so the accumulators overlap. The second
// one begins kOverlap columns before the first one ends, which leaves kOverlap columns for the scales of three K blocks (24
// columns each for E8M0_32, 48 for E4M3_16). The epilogue takes the shared columns of a tile into registers first and gives
// them back before it does anything else, so the multiplies of the next tile wait for a few TMEM reads only.
//
// Scales reach TMEM through registers: four warps of each CTA load them from shared memory and store them to their quarter
// of the lanes, three K blocks ahead of the multiplies. Brought by tcgen05.cp they would stand in the tensor core's own
// queue and cost it about 40 cycles per 512 bytes, six or twelve times per K block of 512 cycles (8192^3: 268 us against
// 202 with E8M0_32, 363 against 218 with E4M3_16).
// A buffer is written again once the multiplies that read it have been committed.

template <int kFormat>
struct Fp4Pair {
    static constexpr int kScaleTiles = kFormat == MCD_FP4_E8M0_32 ? 2 : 4;
    static constexpr int kRowBytes = 128 * 128;
    static constexpr int kColBytes = 128 * 128;
    static constexpr int kRowScaleBytes = kScaleTiles * kFp4TileBytes;
    static constexpr int kColScaleBytes = 2 * kRowScaleBytes;
    static constexpr int kStageBytes = kRowBytes + kColBytes + kRowScaleBytes + kColScaleBytes;
    static constexpr int kTileBytes = kRowBytes + kColBytes;
    static constexpr int kStages = 5;
    static constexpr int kScaleBuffers = 3;  // K blocks whose scales TMEM holds
    static constexpr int kStagingPerWarp = 4096;
    static constexpr int kBarrierBytes = 1024;
    static constexpr int kSmem = kStages * kStageBytes + 1024 + kBarrierBytes + 8 * kStagingPerWarp;
    static constexpr int kOverlapChunks = kFormat == MCD_FP4_E8M0_32 ? 3 : 5;  // of 32 columns
    static constexpr int kOverlap = 32 * kOverlapChunks;
    static constexpr int kScaleBase = 512 - kOverlap;
    static constexpr int kRowScaleColumns = kScaleTiles * 4;
    static constexpr int kScaleColumns = 3 * kRowScaleColumns;  // rows, then columns: 8 per scale tile
    static_assert(kScaleBuffers * kScaleColumns <= kOverlap, "TMEM columns");
};

// A lane's 32 values, the row `lane` of a box of 32 x 32, to shared memory as a TMA store wants them: rows of 128 bytes (f32,
// 128-byte swizzle) or of 64 (16 bits, 64-byte swizzle). kBoth: times both factors of alpha, otherwise the second is 1.
template <bool kBoth>
__device__ __forceinline__ void stage_row(unsigned at, const unsigned (&v)[32], const TwoFactors& alpha, int type) {
    unsigned lane = threadIdx.x & 31;
    asm volatile("" : "+r"(lane));  // addresses made here and not kept: nothing of this is worth registers between tiles
    float f[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) f[j] = kBoth ? alpha.times(__uint_as_float(v[j])) : __uint_as_float(v[j]) * alpha.first;
    if (type == MCD_TYPE_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at + lane * 128 + ((j ^ (lane & 7)) << 4)), "f"(f[4 * j]), "f"(f[4 * j + 1]),
                         "f"(f[4 * j + 2]), "f"(f[4 * j + 3])
                         : "memory");
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)),
                         "r"(pack_half2(f[8 * j], f[8 * j + 1], type)), "r"(pack_half2(f[8 * j + 2], f[8 * j + 3], type)),
                         "r"(pack_half2(f[8 * j + 4], f[8 * j + 5], type)), "r"(pack_half2(f[8 * j + 6], f[8 * j + 7], type))
                         : "memory");
        }
    }
}

// Such a box to rows of C that start anywhere: a warp writes a row, or, where all 16-bit rows start on words, two of them.
// `rows` and `cols` of the box exist. Instructions are what this costs, so eight rows are read ahead of their stores, and
// the addresses in shared memory are constants beside two of the lane's (37728 x 1883 of bf16, K 128, 142 MB of C: 60 us,
// 51 for 1884 columns; TMA takes 38 for 1888).
__device__ __forceinline__ void store_box(unsigned at, void* c, int type, long long first, long long ldc, int rows, int cols) {
    int lane = static_cast<int>(threadIdx.x & 31);
    asm volatile("" : "+r"(lane));  // addresses made here and not kept: nothing of this is worth registers between tiles
    if (type == MCD_TYPE_F32) {
        float* to = static_cast<float*>(c) + first + lane;
        const int mine = lane < cols ? rows : 0;
#pragma unroll
        for (int r = 0; r < 32; r += 8) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[j]) : "r"(at + ((((lane >> 2) ^ j) << 4) + (lane & 3) * 4) + (r + j) * 128) : "memory");
            }
#pragma unroll
            for (int j = 0; j < 8; ++j, to += ldc) {
                if (r + j < mine) *to = v[j];
            }
        }
        return;
    }
    unsigned short* to = static_cast<unsigned short*>(c) + first;
    if (cols >= 32 && ((reinterpret_cast<unsigned long long>(to) >> 1 | static_cast<unsigned long long>(ldc)) & 1) == 0) {
        const int i = lane & 15, mine = rows - (lane >> 4);
        to += (lane >> 4) * ldc + 2 * i;
#pragma unroll
        for (int k = 0; k < 16; k += 8) {
            unsigned v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[j]) : "r"(at + (lane >> 4) * 64 + (((i >> 2) ^ (j & 3)) << 4) + (i & 3) * 4 + (k + j) * 128) : "memory");
            }
#pragma unroll
            for (int j = 0; j < 8; ++j, to += 2 * ldc) {
                if (2 * (k + j) < mine) *reinterpret_cast<unsigned*>(to) = v[j];
            }
        }
        return;
    }
    to += lane;
    const int mine = lane < cols ? rows : 0;
#pragma unroll
    for (int r = 0; r < 32; r += 8) {
        unsigned short v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v[j]) : "r"(at + (((lane >> 3) ^ ((j >> 1) & 3)) << 4) + (lane & 7) * 2 + (r + j) * 64) : "memory");
        }
#pragma unroll
        for (int j = 0; j < 8; ++j, to += ldc) {
            if (r + j < mine) *to = v[j];
        }
    }
}

constexpr int kPairThreads = 64 + 8 * 32 + 4 * 32;
constexpr int kPairTile = 256;
constexpr int kMaxPairSplits = 4;
constexpr int kSlicePitch = 1040;  // 256 sums of a row, and 16 bytes that spread rows over the banks

struct Fp4PairParams {
    const float* row_scale;
    const float* col_scale;
    void* c;
    unsigned* status;
    long long ldc;
    int c_type;
    int m, n, k_blocks;
    int splits, k_blocks_per_split;
    int by_tma;  // C leaves as TMA boxes; otherwise (alignment) row by row
};

template <int kFormat, bool kSplit>
__global__ void __launch_bounds__(kPairThreads, 1)
mc_fp4_gemm_pair(const __grid_constant__ McTensorMap map_rows, const __grid_constant__ McTensorMap map_cols,
                 const __grid_constant__ McTensorMap map_row_scales, const __grid_constant__ McTensorMap map_col_scales,
                 const __grid_constant__ McTensorMap map_c, const Fp4PairParams p) {
    using Pair = Fp4Pair<kFormat>;
    constexpr int stages = Pair::kStages;
    extern __shared__ unsigned char smem_raw[];
    const unsigned tiles_base = (mc_smem_addr(smem_raw) + 1023u) & ~1023u;
    const unsigned staging = tiles_base + stages * Pair::kStageBytes;
    const unsigned bars = staging + 8 * Pair::kStagingPerWarp;
    // full: the leader's, counts both CTAs' tiles. scales: one in each CTA, counts its own. empty: one in each CTA.
    // ready: the leader's, the scale warps of both CTAs. acc_full: one in each CTA; acc_empty: the leader's.
    const unsigned bar_full = bars, bar_empty = bars + 8 * stages, bar_scales = bars + 16 * stages, bar_ready = bars + 24 * stages;
    const unsigned bar_acc_full = bar_ready + 8 * Pair::kScaleBuffers, bar_acc_empty = bar_acc_full + 8;
    __shared__ unsigned tmem_slot;
    __shared__ int abort_storage;
    volatile int* abort_flag = &abort_storage;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    unsigned cluster_rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(cluster_rank));
    const unsigned rank = cluster_rank & 1u, pair_first = kSplit ? cluster_rank & ~1u : 0u;
    const bool leader = rank == 0;
    // Split: a cluster has one tile, its pairs a slice of K each.
    const int pairs = kSplit ? 2 * p.splits : 2;
    const int cluster = blockIdx.x / pairs, clusters = gridDim.x / pairs;
    const int kb_begin = kSplit ? static_cast<int>(cluster_rank >> 1) * p.k_blocks_per_split : 0;
    const int kb_end = kSplit ? min(p.k_blocks, kb_begin + p.k_blocks_per_split) : p.k_blocks;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tiles_r = (p.m + kPairTile - 1) / kPairTile;
    const int tiles_c = (p.n + kPairTile - 1) / kPairTile;
    const int items = tiles_r * tiles_c;

    if (threadIdx.x == 0) {
        abort_storage = 0;
        for (int s = 0; s < stages; ++s) {
            mc_mbar_init(bar_full + 8 * s, 1);
            mc_mbar_init(bar_empty + 8 * s, 1);
            mc_mbar_init(bar_scales + 8 * s, 1);
        }
        for (int b = 0; b < Pair::kScaleBuffers; ++b) mc_mbar_init(bar_ready + 8 * b, 8);
        mc_mbar_init(bar_acc_full, 1);
        mc_mbar_init(bar_acc_empty, 16);  // the epilogue warps of both CTAs
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mc_smem_addr(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0, issued = 0;
            unsigned phase = 0;
            bool ok = true;
            for (int item = cluster; ok && item < items; item += clusters) {
                int rb, cb, split;
                fp4_decode_item(item, tiles_r, tiles_c, 1, rb, cb, split);
                const int row_tile = 2 * rb + static_cast<int>(rank);
                for (int kb = kb_begin; kb < kb_end; ++kb) {
                    ok = mc_mbar_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, p.status, MC_FP4_ERR_PRODUCER);
                    if (!ok) break;
                    const unsigned full = cluster_address(bar_full + 8 * stage, pair_first);
                    const unsigned rows_dst = tiles_base + stage * Pair::kStageBytes;
                    const unsigned cols_dst = rows_dst + Pair::kRowBytes;
                    const unsigned row_scales_dst = cols_dst + Pair::kColBytes;
                    const unsigned col_scales_dst = row_scales_dst + Pair::kRowScaleBytes;
                    // Boxes count whole, what lies outside their tensor arrives as zeros: scales behind the last column too.
                    if (leader) mc_mbar_expect_tx(bar_full + 8 * stage, 2 * Pair::kTileBytes);
                    const unsigned scales = bar_scales + 8 * stage;
                    mc_mbar_expect_tx(scales, Pair::kRowScaleBytes + Pair::kColScaleBytes);
                    tma_load_3d(row_scales_dst, &map_row_scales, scales, 0, kb * Pair::kScaleTiles, row_tile);
                    tma_load_3d(col_scales_dst, &map_col_scales, scales, 0, kb * Pair::kScaleTiles, 2 * cb);
                    tma_load_2d_pair(rows_dst, &map_rows, full, kb * 128, row_tile * 128);
                    tma_load_2d_pair(cols_dst, &map_cols, full, kb * 128, cb * kPairTile + static_cast<int>(rank) * 128);
                    ++issued;
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (!ok) {
                // The copies in flight land before shared memory is given up: each CTA sees its own scales, the leader the
                // tiles of both.
                const int pending = min(issued, stages);
                for (int i = 0; i < pending; ++i) {
                    if (stage == 0) {
                        stage = stages;
                        phase ^= 1u;
                    }
                    --stage;
                    const unsigned long long t0 = mc_globaltimer();
                    while (!mc_mbar_try_wait(bar_scales + 8 * stage, phase) || (leader && !mc_mbar_try_wait(bar_full + 8 * stage, phase))) {
                        if (mc_globaltimer() - t0 > MC_WAIT_NS / 4) {
                            if (p.status != nullptr) atomicOr(p.status, MC_FP4_ERR_DRAIN);
                            break;
                        }
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            constexpr unsigned idesc = fp4_instruction<kFormat>(kPairTile, kPairTile);
            int stage = 0, acc = 0;
            unsigned phase = 0;
            bool seen = false;  // the next K block was seen to be ready while the one before it was being issued
            int ready = 0;
            unsigned ready_phase = 0;
            unsigned empty_phase = 1;  // the first tile waits for nothing
            bool ok = true;
            for (int item = cluster; ok && item < items; item += clusters) {
                ok = mc_mbar_wait(bar_acc_empty, empty_phase, abort_flag, p.status, MC_FP4_ERR_MMA);
                if (!ok) break;
                empty_phase ^= 1u;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned tmem_d = tmem + (acc ? static_cast<unsigned>(256 - Pair::kOverlap) : 0u);
                for (int kb = kb_begin; kb < kb_end; ++kb) {
                    if (!seen) {
                        ok = mc_mbar_wait(bar_full + 8 * stage, phase, abort_flag, p.status, MC_FP4_ERR_MMA) &&
                             mc_mbar_wait(bar_ready + 8 * ready, ready_phase, abort_flag, p.status, MC_FP4_ERR_MMA);
                        if (!ok) break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned rows_src = tiles_base + stage * Pair::kStageBytes;
                    const unsigned cols_src = rows_src + Pair::kRowBytes;
                    const unsigned scale_r = tmem + Pair::kScaleBase + static_cast<unsigned>(ready * Pair::kScaleColumns);
                    const unsigned scale_c = scale_r + Pair::kRowScaleColumns;
                    const unsigned long long desc_r = fp4_tile_desc(rows_src, 1024);
                    const unsigned long long desc_c = fp4_tile_desc(cols_src, 1024);
                    const int this_stage = stage;
                    if (++ready == Pair::kScaleBuffers) {
                        ready = 0;
                        ready_phase ^= 1u;
                    }
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
#pragma unroll
                    for (int ks = 0; ks < kFp4BlockK / kFp4MmaK; ++ks) {
                        // The answers of these tests are needed only behind the last multiply: their latency (some 80 cycles
                        // each, in which a queue of one or two multiplies runs dry) passes while they are being issued.
                        if (ks == 2) seen = mbar_test(bar_full + 8 * stage, phase) & mbar_test(bar_ready + 8 * ready, ready_phase);
                        const int t = kFormat == MCD_FP4_E8M0_32 ? ks >> 1 : ks;
                        const unsigned which = kFormat == MCD_FP4_E8M0_32 && (ks & 1) ? kFp4UpperScales : 0u;
                        fp4_mma<kFormat, 2>(tmem_d, desc_r + 2 * ks, desc_c + 2 * ks, idesc | which, scale_r + 4 * t, scale_c + 8 * t,
                                            (kb > kb_begin || ks > 0) ? 1u : 0u);
                    }
                    fp4_commit_pair(bar_empty + 8 * this_stage, pair_first);
                }
                if (!ok) break;
                fp4_commit_pair(bar_acc_full, pair_first);
                acc ^= 1;
            }
        }
    } else if (warp >= 10) {
        // Scales from shared memory to the 32 TMEM lanes of this warp, the same in every quarter: lane r takes the 16 bytes
        // of rows r, r + 32, r + 64, r + 96 of a tile as four columns.
        const unsigned tmem_lanes = tmem + (static_cast<unsigned>((warp & 3) * 32) << 16) + Pair::kScaleBase;
        const unsigned bar_leader = cluster_address(bar_ready, pair_first);
        int stage = 0, done_stage = 0, ready = 0, number = 0;
        unsigned phase = 0, done_phase = 0;
        bool ok = true;
        for (int item = cluster; ok && item < items; item += clusters) {
            for (int kb = kb_begin; kb < kb_end; ++kb) {
                ok = mc_mbar_wait(bar_scales + 8 * stage, phase, abort_flag, p.status, MC_FP4_ERR_SCALES);
                const unsigned src = tiles_base + stage * Pair::kStageBytes + Pair::kTileBytes + static_cast<unsigned>(lane * 16);
                const unsigned dst = tmem_lanes + static_cast<unsigned>(ready * Pair::kScaleColumns);
                unsigned v[Pair::kScaleColumns];
#pragma unroll
                for (int t = 0; t < Pair::kScaleTiles; ++t) {
                    load_shared_v4(src + t * kFp4TileBytes, v + 4 * t);
                    load_shared_v4(src + Pair::kRowScaleBytes + t * kFp4TileBytes, v + Pair::kRowScaleColumns + 8 * t);
                    load_shared_v4(src + Pair::kRowScaleBytes + (Pair::kScaleTiles + t) * kFp4TileBytes, v + Pair::kRowScaleColumns + 8 * t + 4);
                }
                if (ok && number >= Pair::kScaleBuffers) {  // the K block that used this buffer has been multiplied
                    ok = mc_mbar_wait(bar_empty + 8 * done_stage, done_phase, abort_flag, p.status, MC_FP4_ERR_SCALES);
                    if (++done_stage == stages) {
                        done_stage = 0;
                        done_phase ^= 1u;
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int c = 0; c < Pair::kScaleColumns; c += 8) tmem_store8(dst + c, v + c);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(bar_leader + 8 * ready);
                ++number;
                if (++ready == Pair::kScaleBuffers) ready = 0;
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else {
        const int quarter = warp & 3;
        const int half = (warp - 2) >> 2;
        const unsigned buffer = staging + static_cast<unsigned>(warp - 2) * Pair::kStagingPerWarp;
        const TwoFactors alpha = product_scale(p.row_scale, p.col_scale);
        const unsigned acc_empty = cluster_address(bar_acc_empty, pair_first);
        // Written once for each number of factors: 32 multiplications more per row of a chunk are felt where K is short (65536 x
        // 2048 x 256: 61 us instead of 56), and so is a branch around them (59).
        auto epilogue = [&](auto two) {
            constexpr bool kBoth = decltype(two)::value;
            int acc = 0;
            unsigned full_phase = 0, turn = 0;
            bool ok = true;
            for (int item = cluster; ok && item < items; item += clusters) {
                int rb, cb, split;
                fp4_decode_item(item, tiles_r, tiles_c, 1, rb, cb, split);
                ok = mc_mbar_wait(bar_acc_full, full_phase, abort_flag, p.status, MC_FP4_ERR_EPILOGUE);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                full_phase ^= 1u;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned lanes = tmem + (static_cast<unsigned>(quarter * 32) << 16) + (acc ? static_cast<unsigned>(256 - Pair::kOverlap) : 0u);
                if constexpr (kSplit) {
                    // The multiplies of this slice are done, and with them the ring: the slice goes there, row by row.
    #pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
                        const int chunk = 4 * half + i;
                        unsigned w[32];
                        tmem_load32(lanes + static_cast<unsigned>(chunk * 32), w);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        const unsigned to = tiles_base + static_cast<unsigned>((quarter * 32 + lane) * kSlicePitch + chunk * 128);
    #pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + 16 * j), "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]),
                                         "r"(w[4 * j + 3])
                                         : "memory");
                        }
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    break;
                }
                const int row0 = rb * kPairTile + static_cast<int>(rank) * 128 + quarter * 32;
                // Chunks of 32 columns in the order in which they are wanted back: the shared ones lie at the end of the first
                // accumulator and at the beginning of the second. The two warps of a lane quarter take turns.
                auto chunk_at = [&](int i) { return acc ? i : 7 - i; };
                // Boxes that reach over the last column are not left to TMA, which cuts rows off at 16 bytes: what lies behind C's
                // columns inside ldc is not ours.
                if (!p.by_tma || (p.n % 32 != 0 && (cb + 1) * kPairTile > p.n)) {
                    if (lane == 0) tma_store_wait_read<0>();
    #pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
                        const int chunk = chunk_at(2 * i + half), col0 = cb * kPairTile + chunk * 32;
                        unsigned w[32];
                        tmem_load32(lanes + static_cast<unsigned>(chunk * 32), w);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (i == 3 && lane == 0) mbar_arrive_cluster(acc_empty);
                        if (col0 >= p.n || row0 >= p.m) continue;  // warp-uniform
                        stage_row<kBoth>(buffer, w, alpha, p.c_type);
                        __syncwarp();
                        store_box(buffer, p.c, p.c_type, static_cast<long long>(row0) * p.ldc + col0, p.ldc, p.m - row0, p.n - col0);
                        __syncwarp();
                    }
                    acc ^= 1;
                    continue;
                }
                auto finish = [&](const unsigned (&v)[32], int chunk) {
                    const int col0 = cb * kPairTile + chunk * 32;
                    if (col0 >= p.n) return;  // warp-uniform
                    // boxes of 16 bits take turns in the halves of this warp's buffer
                    unsigned at = buffer;
                    if (p.c_type == MCD_TYPE_F32) {
                        if (lane == 0) tma_store_wait_read<0>();
                    } else {
                        at += (turn & 1u) * 2048u;
                        ++turn;
                        if (lane == 0) tma_store_wait_read<1>();
                    }
                    __syncwarp();
                    stage_row<kBoth>(at, v, alpha, p.c_type);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tma_store_2d(&map_c, at, col0, row0);
                };
                // The shared chunks are read before anything else; where a warp has three of them, the first leaves meanwhile (three
                // in registers spill).
                constexpr int kFirst = (Pair::kOverlapChunks + 1) / 2;  // shared chunks of the warps with half == 0
                unsigned v[2][32];
    #pragma unroll
                for (int i = 0; i < kFirst; ++i) {
                    if (i == 2) {
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        finish(v[0], chunk_at(half));
                    }
                    if (2 * i + half < Pair::kOverlapChunks) tmem_load32(lanes + static_cast<unsigned>(chunk_at(2 * i + half) * 32), v[i & 1]);
                }
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(acc_empty);
    #pragma unroll
                for (int i = kFirst == 3 ? 1 : 0; i < 4; ++i) {
                    const int order = 2 * i + half;
                    if (order >= Pair::kOverlapChunks) {
                        tmem_load32(lanes + static_cast<unsigned>(chunk_at(order) * 32), v[i & 1]);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    }
                    finish(v[i & 1], chunk_at(order));
                }
                acc ^= 1;
            }
        };
        if (alpha.second == 1.0f) {
            epilogue(std::false_type{});
        } else {
            epilogue(std::true_type{});
        }
        if (lane == 0) tma_store_wait_read<0>();
    }

    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (kSplit) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        // Every CTA finishes its share of the columns of its 128 rows, four neighbours per thread: slices in their order.
        int rb, cb, split;
        fp4_decode_item(cluster, tiles_r, tiles_c, 1, rb, cb, split);
        const TwoFactors alpha = product_scale(p.row_scale, p.col_scale);
        const int share = kPairTile / p.splits, first = static_cast<int>(cluster_rank >> 1) * share;
        const int per_row = share / 4;
        const int bytes = p.c_type == MCD_TYPE_F32 ? 4 : 2;
        const bool vec = ((reinterpret_cast<unsigned long long>(p.c) | static_cast<unsigned long long>(p.ldc * bytes)) & (4 * bytes - 1)) == 0;
        constexpr int kAtOnce = 2;  // quads per thread and turn
        for (int base = threadIdx.x; base < 128 * per_row; base += kAtOnce * kPairThreads) {
            float4 part[kAtOnce][kMaxPairSplits];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int q = min(base + u * kPairThreads, 128 * per_row - 1);
                const unsigned at = tiles_base + static_cast<unsigned>(q / per_row * kSlicePitch + (first + q % per_row * 4) * 4);
#pragma unroll
                for (int z = 0; z < kMaxPairSplits; ++z) {
                    if (z < p.splits) {
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(part[u][z].x), "=f"(part[u][z].y), "=f"(part[u][z].z), "=f"(part[u][z].w)
                                     : "r"(cluster_address(at, 2u * static_cast<unsigned>(z) + rank))
                                     : "memory");
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int q = base + u * kPairThreads;
                const int row = rb * kPairTile + static_cast<int>(rank) * 128 + q / per_row, col = cb * kPairTile + first + q % per_row * 4;
                if (q >= 128 * per_row || row >= p.m || col >= p.n) continue;
                float sum[4] = {part[u][0].x, part[u][0].y, part[u][0].z, part[u][0].w};
#pragma unroll
                for (int z = 1; z < kMaxPairSplits; ++z) {
                    if (z < p.splits) sum[0] += part[u][z].x, sum[1] += part[u][z].y, sum[2] += part[u][z].z, sum[3] += part[u][z].w;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = alpha.times(sum[j]);
                store_quad(p.c, p.c_type, static_cast<long long>(row) * p.ldc + col, 1, sum, vec, p.n - col);
            }
        }
    }
    // neither CTA gives up its shared memory or TMEM while the other may still use it
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// The K slices of every element in slice order, times the tensor scales. kVec neighbours of a row per thread.
template <int kVec>
__global__ void __launch_bounds__(256) mc_fp4_join(const float* __restrict__ parts, int splits, long long m, long long n, const float* scale_a,
                                                   const float* scale_b, void* c, int c_type, long long ldc) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const TwoFactors alpha = product_scale(scale_a, scale_b);
    const long long count = m * n;
    const unsigned per_row = static_cast<unsigned>(n / kVec);
    const long long r = blockIdx.y + static_cast<long long>(blockIdx.z) * gridDim.y;
    if (r >= m) return;
    for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < per_row; i += gridDim.x * 256) {
        const float* from = parts + r * n + static_cast<long long>(i) * kVec;
        float sum[kVec];
        if constexpr (kVec == 4) {
            float4 v = *reinterpret_cast<const float4*>(from);
#pragma unroll 4
            for (int z = 1; z < splits; ++z) {
                const float4 w = *reinterpret_cast<const float4*>(from + z * count);
                v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
            }
            sum[0] = v.x, sum[1] = v.y, sum[2] = v.z, sum[3] = v.w;
        } else {
            sum[0] = *from;
            for (int z = 1; z < splits; ++z) sum[0] += from[z * count];
        }
        const long long at = r * ldc + static_cast<long long>(i) * kVec;
#pragma unroll
        for (int j = 0; j < kVec; ++j) store_c(c, c_type, at + j, alpha.times(sum[j]));
    }
}

// ---------------------------------------------------------------------------------------------------------- host side

struct Plan {
    bool pairs = false;  // 256 x 256 tiles on SM pairs; the rest describes the one-CTA kernel
    bool swapped = false;
    int tile_cols = 128;
    int splits = 1;
    int k_blocks = 1;
    int per_split = 1;
    bool clustered = false;  // the slices of a tile meet in a cluster's shared memory
};

// Up to 128 rows or columns of C: the one-CTA kernel, the shorter side as accumulator columns, so that the longer one fills
// the 128 lanes and is read once. Anything larger: SM pairs, however few their tiles (256 x 8192 x 8192 unsplit: 18 us, 36 in
// tiles of 128 x 128; 1024^3: 12 against 23).
//
// K is split where the tiles leave half of the SMs without work, and their loads out of those in flight. The slices of a tile are
// CTAs, or pairs, of one cluster, which adds them up from shared memory, as many as find SMs all at once: eight CTAs for 14
// tiles, four for 32, three for 42.
//   One CTA per slice: one token, 8192 x 8192: 11 us, 14 whole; 128 tokens: 14, 18 through a workspace and a second launch;
//     2048 x 2048: 8 and 10.5. A second wave costs more than the slices give (32 tokens, 8192 columns of K, 16 tiles:
//     8.7 us in clusters of four, 14 in clusters of eight; 34 tiles: 10.8 in threes, 16 in fours). A long K with few tiles
//     has too few CTAs that way and goes through the workspace (128 rows, one token, K 131072: 21 us, 24 in a cluster; two
//     to four times 128 rows: 16, 25; up to 65536 the cluster takes as long or less).
//   Pairs: 512 x 512 x 8192, four slices: 12 us, 16 whole; 256 x 8192 x 8192, two: 16 against 18; x 16384: 24 against 32. At
//     K 4096 joining takes what the slices give.
Plan plan_for(long long m, long long n, long long k) {
    Plan plan;
    plan.k_blocks = static_cast<int>((k + kFp4BlockK - 1) / kFp4BlockK);
    plan.per_split = plan.k_blocks;
    plan.pairs = m > 128 && n > 128;
    if (plan.pairs) {
        const long long pair_tiles = ((m + 255) / 256) * ((n + 255) / 256);
        if (plan.k_blocks >= 24) plan.splits = pair_tiles <= 14 ? 4 : pair_tiles <= 32 ? 2 : 1;
        plan.per_split = (plan.k_blocks + plan.splits - 1) / plan.splits;
        plan.clustered = plan.splits > 1;
        return plan;
    }
    plan.swapped = m <= n;
    const long long rows = plan.swapped ? n : m;
    const long long cols = plan.swapped ? m : n;
    plan.tile_cols = cols <= 16 ? 16 : cols <= 32 ? 32 : cols <= 64 ? 64 : 128;
    const long long tiles = (rows + 127) / 128;
    constexpr int kSms = 148;
    const int stage = plan.tile_cols <= 32 ? 4 : 2;  // K blocks of a stage
    auto split = [&](int splits) {
        plan.per_split = ((plan.k_blocks + splits - 1) / splits + stage - 1) / stage * stage;
        plan.splits = (plan.k_blocks + plan.per_split - 1) / plan.per_split;
    };
    const int most = static_cast<int>(std::max<long long>(1, std::min<long long>(kSms / tiles, plan.k_blocks / 4)));
    if (tiles <= 6 && plan.k_blocks > 256) {
        split(most);
        return plan;
    }
    auto fits = [&](int slices, int sms) { return slices <= most && tiles * slices <= sms; };
    const int splits = fits(8, 112) ? 8 : fits(4, 128) ? 4 : fits(3, 128) ? 3 : fits(2, kSms) ? 2 : 1;
    split(splits);
    plan.clustered = plan.splits > 1;
    return plan;
}

int encode_codes(McTensorMap* map, const mcd_fp4_tensor& t, unsigned box_rows) {
    static_assert(sizeof(McTensorMap) == sizeof(CUtensorMap), "tensor map size");
    const DriverApi* drv = driver_api();
    if (drv == nullptr) return fail("the CUDA driver API is unavailable");
    const auto pitch = static_cast<cuuint64_t>(mcd_fp4_code_pitch(t.cols));
    const cuuint64_t dims[2] = {pitch, static_cast<cuuint64_t>(t.rows)};
    const cuuint64_t strides[1] = {pitch};
    const cuuint32_t box[2] = {128, box_rows};
    const cuuint32_t elem_strides[2] = {1, 1};
    return check_drv(drv->TensorMapEncodeTiled(reinterpret_cast<CUtensorMap*>(map), CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, t.codes, dims, strides,
                                               box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
                     "cuTensorMapEncodeTiled");
}

// Codes in atoms of 8 rows x 128 bytes; a box takes 16 such groups of rows and `blocks` neighbouring atoms of each, in the
// order atom, neighbour, next group. Rows a multiple of 8, pitch one of 128: the box then never leaves the matrix unseen.
bool can_be_wide(const mcd_fp4_tensor& t) { return t.rows % 8 == 0 && mcd_fp4_code_pitch(t.cols) % 128 == 0; }

int encode_wide_codes(McTensorMap* map, const mcd_fp4_tensor& t, unsigned blocks) {
    const DriverApi* drv = driver_api();
    if (drv == nullptr) return fail("the CUDA driver API is unavailable");
    const auto pitch = static_cast<cuuint64_t>(mcd_fp4_code_pitch(t.cols));
    const cuuint64_t dims[4] = {128, 8, pitch / 128, static_cast<cuuint64_t>(t.rows / 8)};
    const cuuint64_t strides[3] = {pitch, 128, 8 * pitch};
    const cuuint32_t box[4] = {128, 8, blocks, kTileRows / 8};
    const cuuint32_t elem_strides[4] = {1, 1, 1, 1};
    return check_drv(drv->TensorMapEncodeTiled(reinterpret_cast<CUtensorMap*>(map), CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, t.codes, dims, strides,
                                               box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
                     "cuTensorMapEncodeTiled");
}

// Scales as a tensor of 512-byte tiles [row tiles, k tiles]; a box takes `k_tiles` tiles of `row_tiles` rows of them.
int encode_scales(McTensorMap* map, const mcd_fp4_tensor& t, unsigned box_k_tiles, unsigned box_row_tiles) {
    const DriverApi* drv = driver_api();
    if (drv == nullptr) return fail("the CUDA driver API is unavailable");
    const Fp4Geometry geo = fp4_geometry(t.format, t.rows, t.cols);
    const cuuint64_t dims[3] = {kFp4TileBytes / 4, static_cast<cuuint64_t>(geo.k_tiles), static_cast<cuuint64_t>(geo.row_tiles)};
    const cuuint64_t strides[2] = {kFp4TileBytes, static_cast<cuuint64_t>(geo.k_tiles * kFp4TileBytes)};
    const cuuint32_t box[3] = {kFp4TileBytes / 4, box_k_tiles, box_row_tiles};
    const cuuint32_t elem_strides[3] = {1, 1, 1};
    return check_drv(drv->TensorMapEncodeTiled(reinterpret_cast<CUtensorMap*>(map), CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, t.scales, dims, strides,
                                               box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
                     "cuTensorMapEncodeTiled");
}

// C in boxes of 32 x 32.
int encode_c(McTensorMap* map, void* c, int type, long long m, long long n, long long ldc) {
    const DriverApi* drv = driver_api();
    if (drv == nullptr) return fail("the CUDA driver API is unavailable");
    const bool f32 = type == MCD_TYPE_F32;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(m)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ldc) * (f32 ? 4 : 2)};
    const cuuint32_t box[2] = {32, 32};
    const cuuint32_t elem_strides[2] = {1, 1};
    return check_drv(drv->TensorMapEncodeTiled(reinterpret_cast<CUtensorMap*>(map), f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                                               2, c, dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                               f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
                     "cuTensorMapEncodeTiled");
}

template <typename... Params, typename... Args>
int launch_dependent(void (*kernel)(Params...), dim3 grid, unsigned cluster, unsigned threads, size_t smem, cudaStream_t s, const char* what, Args... args) {
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return check_rt(cudaLaunchKernelEx(&config, kernel, args...), what);
}

template <int kFormat, int kCols>
int launch_one_cta(const McTensorMap& rows, const McTensorMap& cols, const Fp4GemmParams& p, unsigned grid, cudaStream_t s) {
    using Tile = Fp4Tile<kFormat, kCols>;
    static_assert(Tile::kSmem + 64 <= 227 * 1024, "shared memory");
    static SharedMemoryOnce once;
    if (int rc = once.allow(mc_fp4_gemm<kFormat, kCols>, Tile::kSmem)) return rc;
    return launch_dependent(mc_fp4_gemm<kFormat, kCols>, grid, p.clustered ? p.splits : 1, kOneCtaThreads, Tile::kSmem, s, "mc_fp4_gemm", rows, cols, p);
}

template <int kFormat>
int launch_format(int tile_cols, const McTensorMap& rows, const McTensorMap& cols, const Fp4GemmParams& p, unsigned grid, cudaStream_t s) {
    switch (tile_cols) {
        case 16: return launch_one_cta<kFormat, 16>(rows, cols, p, grid, s);
        case 32: return launch_one_cta<kFormat, 32>(rows, cols, p, grid, s);
        case 64: return launch_one_cta<kFormat, 64>(rows, cols, p, grid, s);
        default: return launch_one_cta<kFormat, 128>(rows, cols, p, grid, s);
    }
}

template <int kFormat, bool kSplit>
int launch_pairs(const mcd_fp4_gemm_args* args, const Plan& plan, cudaStream_t s) {
    using Pair = Fp4Pair<kFormat>;
    static_assert(Pair::kSmem + 64 <= 227 * 1024, "shared memory");
    static_assert(128 * kSlicePitch <= Pair::kStages * Pair::kStageBytes, "a slice fits into the ring");
    static SharedMemoryOnce once;
    if (int rc = once.allow(mc_fp4_gemm_pair<kFormat, kSplit>, Pair::kSmem)) return rc;
    McTensorMap rows, cols, row_scales, col_scales, c = {};
    if (int rc = encode_codes(&rows, args->a, 128)) return rc;
    if (int rc = encode_codes(&cols, args->b, 128)) return rc;
    if (int rc = encode_scales(&row_scales, args->a, Pair::kScaleTiles, 1)) return rc;
    if (int rc = encode_scales(&col_scales, args->b, Pair::kScaleTiles, 2)) return rc;
    Fp4PairParams p;
    p.row_scale = args->a.tensor_scale;
    p.col_scale = args->b.tensor_scale;
    p.c = args->c;
    p.status = args->status;
    p.ldc = args->ldc;
    p.c_type = args->c_type;
    p.m = static_cast<int>(args->a.rows);
    p.n = static_cast<int>(args->b.rows);
    p.k_blocks = plan.k_blocks;
    p.splits = plan.splits;
    p.k_blocks_per_split = plan.per_split;
    p.by_tma = is_aligned(args->c, 16) && args->ldc % (args->c_type == MCD_TYPE_F32 ? 4 : 8) == 0;
    if (p.by_tma) {
        if (int rc = encode_c(&c, args->c, args->c_type, p.m, p.n, args->ldc)) return rc;
    }
    const long long tiles = ((args->a.rows + kPairTile - 1) / kPairTile) * ((args->b.rows + kPairTile - 1) / kPairTile);
    const unsigned cluster = 2 * static_cast<unsigned>(plan.splits);
    const auto grid = cluster * static_cast<unsigned>(kSplit ? tiles : std::min<long long>(tiles, sm_count() / 2));
    return launch_dependent(mc_fp4_gemm_pair<kFormat, kSplit>, grid, cluster, kPairThreads, Pair::kSmem, s, "mc_fp4_gemm_pair", rows, cols, row_scales, col_scales, c, p);
}

size_t plan_workspace(const Plan& plan, long long m, long long n) {
    return plan.splits > 1 && !plan.clustered ? static_cast<size_t>(plan.splits) * static_cast<size_t>(m) * static_cast<size_t>(n) * sizeof(float) : 0;
}

bool sized(const mcd_fp4_gemm_args* a) {
    constexpr long long most = 2147483647LL;
    return a != nullptr && a->a.rows > 0 && a->b.rows > 0 && a->a.cols > 0 && a->a.rows <= most && a->b.rows <= most && a->a.cols <= most;
}

}  // namespace

extern "C" size_t mcd_fp4_gemm_workspace(const mcd_fp4_gemm_args* args) {
    if (!sized(args)) return 0;
    return plan_workspace(plan_for(args->a.rows, args->b.rows, args->a.cols), args->a.rows, args->b.rows);
}

extern "C" int mcd_fp4_gemm_launches(const mcd_fp4_gemm_args* args) {
    if (!sized(args)) return 0;
    const Plan plan = plan_for(args->a.rows, args->b.rows, args->a.cols);
    return plan.splits > 1 && !plan.clustered ? 2 : 1;
}

extern "C" int mcd_fp4_gemm(const mcd_fp4_gemm_args* args, void* stream) {
    const char* who = "mcd_fp4_gemm";
    if (args == nullptr) return fail("mcd_fp4_gemm: null arguments");
    if (int rc = check_fp4(who, &args->a)) return rc;
    if (int rc = check_fp4(who, &args->b)) return rc;
    if (args->a.batch != 1 || args->b.batch != 1) return fail("mcd_fp4_gemm: operands are single matrices (batch 1)");
    if (args->a.format != args->b.format) return fail("mcd_fp4_gemm: the operands' formats differ");
    if (args->a.cols != args->b.cols) return fail("mcd_fp4_gemm: the operands' columns (k) differ");
    const int type = args->c_type;
    if (type != MCD_TYPE_F32 && type != MCD_HALF_BF16 && type != MCD_HALF_F16) return fail("mcd_fp4_gemm: unknown type of c");
    if (args->c == nullptr) return fail("mcd_fp4_gemm: no output buffer");
    if (!is_aligned(args->c, type == MCD_TYPE_F32 ? 4 : 2)) return fail("mcd_fp4_gemm: c is not aligned to its type");
    const long long m = args->a.rows, n = args->b.rows, k = args->a.cols;
    if (args->ldc < n) return fail("mcd_fp4_gemm: ldc is less than a row of c");
    if (!fits(1, m, args->ldc, 1LL << 46)) return fail("mcd_fp4_gemm: c is too large");
    if (!is_aligned(args->status, 4)) return fail("mcd_fp4_gemm: unaligned status word");
    const Plan plan = plan_for(m, n, k);
    const long long rows = plan.swapped ? n : m, cols = plan.swapped ? m : n;
    const long long items = ((rows + 127) / 128) * ((cols + plan.tile_cols - 1) / plan.tile_cols) * plan.splits;
    if (items > 2000000000LL) return fail("mcd_fp4_gemm: too many tiles");
    const size_t need = plan_workspace(plan, m, n);
    if (need > 0 && (args->workspace == nullptr || args->workspace_bytes < need)) {
        return fail("mcd_fp4_gemm: this problem needs " + std::to_string(need) + " bytes of workspace");
    }
    if (need > 0 && !is_aligned(args->workspace, 16)) return fail("mcd_fp4_gemm: the workspace needs 16-byte alignment");
    if (int rc = check_device_pointers(who, {args->a.codes, args->a.scales, args->a.tensor_scale, args->b.codes, args->b.scales, args->b.tensor_scale,
                                             args->c, need > 0 ? args->workspace : nullptr, args->status})) {
        return rc;
    }
    if (plan.pairs) {
        auto on = static_cast<cudaStream_t>(stream);
        if (args->a.format == MCD_FP4_E8M0_32) {
            return plan.splits > 1 ? launch_pairs<MCD_FP4_E8M0_32, true>(args, plan, on) : launch_pairs<MCD_FP4_E8M0_32, false>(args, plan, on);
        }
        return plan.splits > 1 ? launch_pairs<MCD_FP4_E4M3_16, true>(args, plan, on) : launch_pairs<MCD_FP4_E4M3_16, false>(args, plan, on);
    }
    const mcd_fp4_tensor& on_rows = plan.swapped ? args->b : args->a;
    const mcd_fp4_tensor& on_cols = plan.swapped ? args->a : args->b;
    McTensorMap map_rows, map_cols;
    const bool wide = can_be_wide(on_rows);
    if (int rc = wide ? encode_wide_codes(&map_rows, on_rows, plan.tile_cols <= 32 ? 4 : 2) : encode_codes(&map_rows, on_rows, kTileRows)) return rc;
    if (int rc = encode_codes(&map_cols, on_cols, static_cast<unsigned>(plan.tile_cols))) return rc;
    Fp4GemmParams p;
    p.row_scales = static_cast<const unsigned char*>(on_rows.scales);
    p.col_scales = static_cast<const unsigned char*>(on_cols.scales);
    p.k_tiles = fp4_geometry(args->a.format, 1, k).k_tiles;
    p.row_scale = on_rows.tensor_scale;
    p.col_scale = on_cols.tensor_scale;
    p.c = args->c;
    p.workspace = static_cast<float*>(args->workspace);
    p.status = args->status;
    p.ldc = args->ldc;
    p.c_type = type;
    p.rows = static_cast<int>(rows);
    p.cols = static_cast<int>(cols);
    p.k = static_cast<int>(k);
    p.k_blocks = plan.k_blocks;
    p.k_blocks_per_split = plan.per_split;
    p.splits = plan.splits;
    p.swapped = plan.swapped ? 1 : 0;
    p.wide = wide ? 1 : 0;
    p.clustered = plan.clustered ? 1 : 0;
    auto s = static_cast<cudaStream_t>(stream);
    const auto grid = static_cast<unsigned>(plan.clustered ? items : std::min<long long>(items, sm_count()));
    if (int rc = args->a.format == MCD_FP4_E8M0_32 ? launch_format<MCD_FP4_E8M0_32>(plan.tile_cols, map_rows, map_cols, p, grid, s)
                                                   : launch_format<MCD_FP4_E4M3_16>(plan.tile_cols, map_rows, map_cols, p, grid, s)) {
        return rc;
    }
    if (plan.splits == 1 || plan.clustered) return 0;
    const bool vec = n % 4 == 0;
    const long long per_row = vec ? n / 4 : n;
    const auto join_rows = static_cast<unsigned>(std::min<long long>(m, 32768));
    const dim3 join_grid(static_cast<unsigned>(std::min<long long>((per_row + 255) / 256, 1024)), join_rows, static_cast<unsigned>((m + join_rows - 1) / join_rows));
    return launch_dependent(vec ? mc_fp4_join<4> : mc_fp4_join<1>, join_grid, 1, 256, 0, s, "mc_fp4_join", static_cast<const float*>(p.workspace), plan.splits, m, n,
                            args->a.tensor_scale, args->b.tensor_scale, p.c, p.c_type, p.ldc);
}
