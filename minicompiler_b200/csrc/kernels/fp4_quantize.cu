// mcd_fp4_quantize, mcd_fp4_dequantize, mcd_fp4_tensor_scale: values to and from the microscaled 4-bit formats.
//
// All three move bytes: a value is read once and 0.53 (E8M0_32) or 0.56 (E4M3_16) bytes are written for it, or the
// other way round; a dozen instructions per value lie between. A thread takes 16 consecutive columns - one E4M3 block, or
// half an E8M0 block whose two halves meet through one shuffle - and several rows, so that enough loads are under way.

#include "minicompiler_b200_device.h"

#include "device/driver_api.hpp"
#include "kernels/fp4_format.cuh"
#include "kernels/fp4_host.hpp"

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

using namespace mcd;

namespace {

constexpr int kUnit = 16;     // columns per thread
constexpr int kThreads = 256;

struct F32 {
    using type = float;
    static constexpr int kind = MCD_TYPE_F32;
};
struct Bf16 {
    using type = unsigned short;
    static constexpr int kind = MCD_HALF_BF16;
};
struct F16 {
    using type = unsigned short;
    static constexpr int kind = MCD_HALF_F16;
};

template <typename T>
__device__ __forceinline__ float to_f32(typename T::type v) {
    if constexpr (T::kind == MCD_TYPE_F32) {
        return v;
    } else if constexpr (T::kind == MCD_HALF_BF16) {
        return __uint_as_float(static_cast<unsigned>(v) << 16);
    } else {
        return f16_lo(v);
    }
}

template <typename T>
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
    unsigned d;
    if constexpr (T::kind == MCD_HALF_BF16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    }
    return d;
}

// How the rows of dense values lie: 32 (16) - every row starts on such a boundary and values move in accesses of that many
// bytes; 0 - one by one. An access of 32 bytes is a whole sector of a lane's own: 65536 x 2048 values take 51 us from codes
// to bf16 that way (268 MB written, 71 MB read: 6.6 TB/s) and 68 us in halves of it; the way to codes takes 73 us.
//
// The 16 values from column c0 on as they lie in memory; zeros behind `cols`.
template <typename T>
struct Raw {
    static constexpr int kWords = T::kind == MCD_TYPE_F32 ? 16 : 8;
    unsigned w[kWords];

    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    template <int kVec>
    __device__ __forceinline__ void load(const typename T::type* row, long long c0, long long cols) {
        const auto* from = row + c0;
        if (kVec != 0 && c0 + kUnit <= cols) {
            if constexpr (kVec == 32) {
#pragma unroll
                for (int i = 0; i < kWords; i += 8) {
                    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                                 : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]), "=r"(w[i + 7])
                                 : "l"(reinterpret_cast<const unsigned*>(from) + i));
                }
            } else {
#pragma unroll
                for (int i = 0; i < kWords; i += 4) {
                    const uint4 q = __ldcs(reinterpret_cast<const uint4*>(from) + i / 4);
                    w[i] = q.x, w[i + 1] = q.y, w[i + 2] = q.z, w[i + 3] = q.w;
                }
            }
            return;
        }
        const int left = static_cast<int>(min(static_cast<long long>(kUnit), cols - c0));
        if constexpr (T::kind == MCD_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) w[i] = i < left ? __float_as_uint(from[i]) : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < kUnit; i += 2) {
                const unsigned lo = i < left ? from[i] : 0u, hi = i + 1 < left ? from[i + 1] : 0u;
                w[i / 2] = lo | hi << 16;
            }
        }
    }
    // The largest magnitude as bits of f32: an integer maximum, in which infinity and NaN come out on top. Without their
    // signs 16-bit values compare as integers, two at a time.
    __device__ __forceinline__ unsigned amax() const {
        unsigned most = 0;
        if constexpr (T::kind == MCD_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) most = max(most, w[i] & 0x7fffffffu);
            return most;
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(most) : "r"(w[i] & 0x7fff7fffu));
            return __float_as_uint(to_f32<T>(static_cast<unsigned short>(max(most & 0xffffu, most >> 16))));
        }
    }
    __device__ __forceinline__ void values(float (&v)[kUnit]) const {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            if constexpr (T::kind == MCD_TYPE_F32) {
                v[i] = __uint_as_float(w[i]);
            } else {
                v[i] = to_f32<T>(static_cast<unsigned short>(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
            }
        }
    }
};

struct QuantizeParams {
    const void* src;
    unsigned char* codes;
    unsigned char* scales;
    const float* tensor_scale;
    long long rows, cols, pitch_elems;
    long long code_pitch, k_tiles, padded_rows;
    long long batch;
    int units;      // per row, whole scale tiles
    int unit_bits;  // a row takes 1 << unit_bits threads of a block (at most 256), several trips where that is less than units
};

// Which matrix a row belongs to (rows of all matrices in a row, `per_matrix` each) and its number there.
__device__ __forceinline__ long long matrix_of(long long& row, long long per_matrix, long long batch) {
    if (batch == 1) return 0;
    const long long m = row / per_matrix;
    row -= m * per_matrix;
    return m;
}

// A thread takes the same unit of kRows rows: their loads are under way together.
template <typename T, int kFormat, int kVec, int kRows>
__global__ void __launch_bounds__(kThreads) mc_fp4_quantize(const QuantizeParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the launch before this one
    const int lanes = 1 << p.unit_bits;
    const int rows_per_block = kThreads >> p.unit_bits;
    const int lane = static_cast<int>(threadIdx.x) & (lanes - 1);
    const long long all_rows = p.batch * p.padded_rows;
    const long long first_row = static_cast<long long>(blockIdx.x) * (rows_per_block * kRows) + (threadIdx.x >> p.unit_bits);
    // whole warps run every trip: the halves of a block meet in a shuffle
    for (int first = 0; first < p.units; first += lanes) {
        const int unit = first + lane;
        const bool live = unit < p.units;
        const long long c0 = static_cast<long long>(unit) * kUnit;
        Raw<T> raw[kRows];
        float g[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            long long r = first_row + i * rows_per_block;
            raw[i].zero();
            g[i] = 1.0f;
            if (r < all_rows) {
                const long long m = matrix_of(r, p.padded_rows, p.batch);
                if (r < p.rows && live && c0 < p.cols) {
                    raw[i].template load<kVec>(static_cast<const typename T::type*>(p.src) + (m * p.rows + r) * p.pitch_elems, c0, p.cols);
                }
                if (kFormat == MCD_FP4_E4M3_16 && p.tensor_scale != nullptr) g[i] = p.tensor_scale[m];
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            long long r = first_row + i * rows_per_block;
            const bool inside = r < all_rows;
            const long long m = inside ? matrix_of(r, p.padded_rows, p.batch) : 0;
            const bool real = inside && r < p.rows;
            float v[kUnit];
            raw[i].values(v);
            unsigned amax = raw[i].amax();
            unsigned byte;
            float inverse;
            if (kFormat == MCD_FP4_E8M0_32) {
                amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                const int e = static_cast<int>(amax >> 23) - 2;  // floor(log2 amax) - 2, biased by 127
                byte = amax >= 0x7f800000u ? 255u : static_cast<unsigned>(max(e, 0));
                inverse = __uint_as_float((254u - min(byte, 252u)) << 23);  // 2^-(byte - 127)
            } else {
                const bool g_ok = g[i] > 0.0f && g[i] <= 3.402823466e38f;
                byte = (amax >= 0x7f800000u || !g_ok) ? 0x7fu : e4m3_encode(__fdiv_rn(__uint_as_float(amax), __fmul_rn(6.0f, g[i])));
                const float s_g = __fmul_rn(e4m3_decode(byte), g[i]);
                inverse = s_g == 0.0f ? 0.0f : fminf(__fdiv_rn(1.0f, s_g), 3.402823466e38f);
            }
            const bool bad = byte == (kFormat == MCD_FP4_E8M0_32 ? 255u : 0x7fu);  // the NaN scales; no rounding gives them
#pragma unroll
            for (int j = 0; j < kUnit; ++j) v[j] = __fmul_rn(v[j], inverse);
            unsigned lo = fp4_encode8(v), hi = fp4_encode8(v + 8);
            if (bad) lo = hi = 0;
            if (real && live && c0 / 2 < p.code_pitch) {
                *reinterpret_cast<uint2*>(p.codes + (m * p.rows + r) * p.code_pitch + c0 / 2) = make_uint2(lo, hi);
            }
            if (inside && live) {
                unsigned char* scales = p.scales + m * (p.padded_rows >> 7) * p.k_tiles * kFp4TileBytes;
                const unsigned char stored = static_cast<unsigned char>(c0 < p.cols && real ? byte : 0u);
                if (kFormat == MCD_FP4_E8M0_32) {
                    if ((unit & 1) == 0) scales[fp4_scale_offset(r, unit >> 1, p.k_tiles)] = stored;
                } else {
                    scales[fp4_scale_offset(r, unit, p.k_tiles)] = stored;
                }
            }
        }
    }
}

struct DequantizeParams {
    const unsigned char* codes;
    const unsigned char* scales;
    const float* tensor_scale;
    void* dst;
    long long rows, cols, pitch_elems;
    long long code_pitch, k_tiles, matrix_scales;
    long long batch;
    int units;
    int unit_bits;
};

// a * g in f32, rounded to odd: cut off, and the last bit set where something was cut off. Rounding that to 16 bits gives what
// rounding the product itself does: f32 has two bits and more than those types, and they tell a tie from what lies beside
// it. `a` has at most 6 significant bits, from 2^-10 up. What is cut off is found exactly by an fma, 2^64 times larger where
// g is so small that f32 would not hold it.
__device__ __forceinline__ float times_to_odd(float a, float g) {
    const float larger = fabsf(g) < 0x1p-40f ? 0x1p64f : 1.0f;
    const float v = __fmul_rz(a, g);
    const float left = fmaf(a, g * larger, -(v * larger));
    return fabsf(left) > 0.0f ? __uint_as_float(__float_as_uint(v) | 1u) : v;
}

// The 16 values of an E4M3 block with a tensor scale, code * scale * g rounded once to 16 bits. A block has eight magnitudes:
// they are rounded once each, and every code picks the two bytes of its own. Value by value the rounding costs nine
// instructions more than two roundings (65536 x 2048 bf16 values with their scale there and back: 211 us, this way 187).
template <typename T>
__device__ __forceinline__ void e4m3_values16(const uint2& codes, float scale, float g, unsigned (&w)[8]) {
    float m[8];
    if (fabsf(g) >= 0x1p-100f && fabsf(g) <= 0x1p100f) {  // far from the ends of f32 powers of two come for nothing
        const float one = times_to_odd(scale, g), three = times_to_odd(1.5f * scale, g);
        m[0] = 0.0f * one, m[1] = 0.5f * one, m[2] = one, m[3] = three, m[4] = 2.0f * one, m[5] = 2.0f * three, m[6] = 4.0f * one, m[7] = 4.0f * three;
    } else {
        constexpr float magnitudes[8] = {0.0f, 0.5f, 1.0f, 1.5f, 2.0f, 3.0f, 4.0f, 6.0f};
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = times_to_odd(magnitudes[i] * scale, g);
    }
    const unsigned r[4] = {pack2<T>(m[0], m[1]), pack2<T>(m[2], m[3]), pack2<T>(m[4], m[5]), pack2<T>(m[6], m[7])};
    const unsigned low[2] = {__byte_perm(r[0], r[1], 0x6420), __byte_perm(r[2], r[3], 0x6420)};
    const unsigned high[2] = {__byte_perm(r[0], r[1], 0x7531), __byte_perm(r[2], r[3], 0x7531)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // four codes: 16 bits of them are four selectors, three bits a magnitude, the fourth the sign
        const unsigned four = (i < 2 ? codes.x : codes.y) >> (16 * (i & 1));
        unsigned signs, lo, hi;
        asm("prmt.b32 %0, %1, %1, %2;" : "=r"(signs) : "r"(0x80808080u), "r"(four));  // the fourth bit copies a byte's first to all: 0x80 or 0xff
        asm("prmt.b32 %0, %1, %2, %3;" : "=r"(lo) : "r"(low[0]), "r"(low[1]), "r"(four & 0x7777u));
        asm("prmt.b32 %0, %1, %2, %3;" : "=r"(hi) : "r"(high[0]), "r"(high[1]), "r"(four & 0x7777u));
        hi ^= (signs << 7) & 0x80808080u;
        w[2 * i] = __byte_perm(lo, hi, 0x5140);
        w[2 * i + 1] = __byte_perm(lo, hi, 0x7362);
    }
}

// The j-th of a thread's values.
template <typename T>
__device__ __forceinline__ typename T::type value_of(const unsigned (&w)[Raw<T>::kWords], int j) {
    if constexpr (T::kind == MCD_TYPE_F32) {
        return __uint_as_float(w[j]);
    } else {
        return static_cast<unsigned short>(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu);
    }
}

// Codes are few bytes: a thread asks for those of kRows rows before it unpacks any.
template <typename T, int kFormat, int kVec, int kRows>
__global__ void __launch_bounds__(kThreads) mc_fp4_dequantize(const DequantizeParams p) {
    __shared__ __align__(16) typename T::type tile[kVec == 0 ? kThreads * kUnit : 16];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lanes = 1 << p.unit_bits;
    const int rows_per_block = kThreads >> p.unit_bits;
    const int lane = static_cast<int>(threadIdx.x) & (lanes - 1);
    const long long all_rows = p.batch * p.rows;
    const long long first_row = static_cast<long long>(blockIdx.x) * (rows_per_block * kRows) + (threadIdx.x >> p.unit_bits);
    for (int first = 0; first < p.units; first += lanes) {
        const int unit = first + lane;
        const bool live = unit < p.units;
        const long long c0 = static_cast<long long>(unit) * kUnit;
        uint2 word[kRows];
        unsigned byte[kRows];
        float g[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const long long at = first_row + i * rows_per_block;
            g[i] = 1.0f;
            word[i] = make_uint2(0, 0);
            byte[i] = 0;
            if (at < all_rows && live) {
                long long r = at;
                const long long m = matrix_of(r, p.rows, p.batch);
                word[i] = __ldcs(reinterpret_cast<const uint2*>(p.codes + at * p.code_pitch + c0 / 2));
                byte[i] = p.scales[m * p.matrix_scales + fp4_scale_offset(r, kFormat == MCD_FP4_E8M0_32 ? unit >> 1 : unit, p.k_tiles)];
                if (kFormat == MCD_FP4_E4M3_16 && p.tensor_scale != nullptr) g[i] = p.tensor_scale[m];
            }
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const long long at = first_row + i * rows_per_block;
            if (kVec != 0 && (at >= all_rows || !live)) continue;
            const float scale = kFormat == MCD_FP4_E8M0_32 ? e8m0_decode(byte[i]) : e4m3_decode(byte[i]);
            unsigned w[Raw<T>::kWords];
            if constexpr (kFormat == MCD_FP4_E4M3_16 && T::kind != MCD_TYPE_F32) {
                e4m3_values16<T>(word[i], scale, g[i], w);
            } else {
                float v[kUnit];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    unsigned pairs[4];
                    fp4_decode8(h == 0 ? word[i].x : word[i].y, pairs);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[8 * h + 2 * j] = f16_lo(pairs[j]) * scale;  // exact: at most 6 significant bits
                        v[8 * h + 2 * j + 1] = f16_hi(pairs[j]) * scale;
                    }
                }
#pragma unroll
                for (int j = 0; j < Raw<T>::kWords; ++j) {
                    if constexpr (T::kind == MCD_TYPE_F32) {
                        w[j] = __float_as_uint(kFormat == MCD_FP4_E4M3_16 ? v[j] * g[i] : v[j]);
                    } else {
                        w[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
                    }
                }
            }
            auto* to = static_cast<typename T::type*>(p.dst) + at * p.pitch_elems + c0;
            if (kVec != 0 && c0 + kUnit <= p.cols) {
                if constexpr (kVec == 32) {
#pragma unroll
                    for (int j = 0; j < Raw<T>::kWords; j += 8) {
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<unsigned*>(to) + j), "r"(w[j]),
                                     "r"(w[j + 1]), "r"(w[j + 2]), "r"(w[j + 3]), "r"(w[j + 4]), "r"(w[j + 5]), "r"(w[j + 6]), "r"(w[j + 7])
                                     : "memory");
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < Raw<T>::kWords; j += 4) __stcs(reinterpret_cast<uint4*>(to) + j / 4, make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]));
                }
            } else if (kVec != 0) {
#pragma unroll
                for (int j = 0; j < kUnit; ++j) {
                    if (c0 + j < p.cols) to[j] = value_of<T>(w, j);
                }
            } else {
                // Rows that start anywhere: neighbouring values leave together (8191 x 8191 f16 values to codes and back: 129 us,
                // 439 with a thread's 16 values one after the other; for loads the caches make up for it).
                typename T::type* mine = tile + (threadIdx.x - lane) * kUnit;
#pragma unroll
                for (int j = 0; j < kUnit; ++j) mine[lane * kUnit + j] = value_of<T>(w, j);
                __syncthreads();
                auto* row = static_cast<typename T::type*>(p.dst) + at * p.pitch_elems;
#pragma unroll
                for (int j = 0; j < kUnit; ++j) {
                    const long long c = static_cast<long long>(first) * kUnit + lane + j * lanes;
                    if (at < all_rows && c < p.cols) row[c] = mine[lane + j * lanes];
                }
                __syncthreads();
            }
        }
    }
}

// ---- the tensor scale: maxima of bit patterns (order does not matter), then one division.

// The largest finite magnitude among this thread's share, as bits.
template <typename T, int kVec>
__device__ __forceinline__ unsigned amax_share(const typename T::type* src, long long rows, long long cols, long long pitch, long long first,
                                               long long stride) {
    const long long units = (cols + kUnit - 1) / kUnit;
    long long r = first / units, u = first - r * units;
    const long long skip_r = stride / units, skip_u = stride - skip_r * units;
    unsigned amax = 0;
    while (r < rows) {
        Raw<T> raw;
        raw.template load<kVec>(src + r * pitch, u * kUnit, cols);
        float v[kUnit];
        raw.values(v);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            const unsigned bits = __float_as_uint(v[i]) & 0x7fffffffu;
            amax = max(amax, bits >= 0x7f800000u ? 0u : bits);
        }
        r += skip_r;
        u += skip_u;
        if (u >= units) u -= units, ++r;
    }
    return amax;
}

__device__ __forceinline__ float scale_of(unsigned amax_bits) {
    if (amax_bits == 0) return 1.0f;
    return fmaxf(__fdiv_rn(__uint_as_float(amax_bits), 2688.0f), 7.52316384526264e-37f);  // 2^-120
}

// The maximum over the block, in thread 0.
__device__ __forceinline__ unsigned block_max(unsigned v) {
    __shared__ unsigned per_warp[32];
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) per_warp[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
        v = threadIdx.x < blockDim.x / 32 ? per_warp[threadIdx.x] : 0u;
        v = __reduce_max_sync(0xffffffffu, v);
    }
    return v;
}

// A matrix per cluster of 8 CTAs, in one launch.
template <typename T, int kVec>
__global__ void __cluster_dims__(8, 1, 1) __launch_bounds__(1024)
mc_fp4_amax_one(const typename T::type* src, long long rows, long long cols, long long pitch, float* out) {
    __shared__ unsigned parts[8];  // of the cluster's first CTA
    unsigned rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const long long matrix = blockIdx.x / 8;
    const unsigned v = block_max(amax_share<T, kVec>(src + matrix * rows * pitch, rows, cols, pitch, rank * 1024 + threadIdx.x, 8 * 1024));
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the first CTA runs
    if (threadIdx.x == 0) {
        unsigned to;
        const auto mine = static_cast<unsigned>(__cvta_generic_to_shared(parts + rank));
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(mine), "r"(0u));
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(v) : "memory");
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0 && threadIdx.x == 0) {
        unsigned all = 0;
        for (int i = 0; i < 8; ++i) all = max(all, parts[i]);
        out[matrix] = scale_of(all);
    }
}

template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) mc_fp4_amax_many(const typename T::type* src, long long rows, long long cols, long long pitch, unsigned* out) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const typename T::type* matrix = src + static_cast<long long>(blockIdx.y) * rows * pitch;
    const unsigned v = block_max(amax_share<T, kVec>(matrix, rows, cols, pitch, static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x,
                                                     static_cast<long long>(gridDim.x) * kThreads));
    if (threadIdx.x == 0 && v != 0) atomicMax(out + blockIdx.y, v);
}

__global__ void mc_fp4_amax_finish(float* out, int batch) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int i = static_cast<int>(blockIdx.x * blockDim.x + threadIdx.x);
    if (i < batch) out[i] = scale_of(__float_as_uint(out[i]));
}

// How a block of threads takes rows of `units`: a power of two of threads per row, at least one warp-even pair.
int unit_bits(long long units) {
    int bits = 1;
    while (bits < 8 && (1LL << bits) < units) ++bits;
    return bits;
}

long long blocks_for(long long rows, int bits, int rows_per_thread) {
    const long long per_block = static_cast<long long>(kThreads >> bits) * rows_per_thread;
    return (rows + per_block - 1) / per_block;
}

// 32, 16 or 0, see Raw.
int rows_aligned(int type, const void* p, long long pitch) {
    const long long row = pitch * (type == MCD_TYPE_F32 ? 4 : 2);
    return is_aligned(p, 32) && row % 32 == 0 ? 32 : is_aligned(p, 16) && row % 16 == 0 ? 16 : 0;
}

// Every launch is a programmatic dependent of what precedes it (each kernel says griddepcontrol.wait before its first
// access): a matrix of 8192 x 4096 f32 values and its scale, there and back, takes 87 us instead of 93; a row of 2048
// values, there and back and waited for, 8.2 instead of 10.3.
template <typename... Params, typename... Args>
int launch(void (*kernel)(Params...), long long grid, unsigned threads, cudaStream_t s, const char* what, Args... args) {
    if (grid > 2147483647LL) return fail(std::string(what) + ": too many rows");
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
    config.blockDim = dim3(threads, 1, 1);
    config.stream = s;
    config.attrs = &attribute;
    config.numAttrs = 1;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return check_rt(cudaLaunchKernelEx(&config, kernel, args...), what);
}

// Several rows per thread only where that leaves every SM 16 blocks.
bool many_blocks(long long blocks) { return blocks >= 16LL * sm_count(); }

template <typename T, int kFormat, int kRows>
int quantize_rows(const QuantizeParams& p, int vec, cudaStream_t s) {
    auto* kernel = vec == 32 ? mc_fp4_quantize<T, kFormat, 32, kRows> : vec == 16 ? mc_fp4_quantize<T, kFormat, 16, kRows> : mc_fp4_quantize<T, kFormat, 0, kRows>;
    return launch(kernel, blocks_for(p.batch * p.padded_rows, p.unit_bits, kRows), kThreads, s, "mc_fp4_quantize", p);
}

template <typename T, int kFormat>
int quantize_launch(const QuantizeParams& p, int vec, cudaStream_t s) {
    constexpr int kRows = T::kind == MCD_TYPE_F32 ? 2 : 4;
    return many_blocks(blocks_for(p.batch * p.padded_rows, p.unit_bits, kRows)) ? quantize_rows<T, kFormat, kRows>(p, vec, s)
                                                                                : quantize_rows<T, kFormat, 1>(p, vec, s);
}

template <typename T, int kFormat, int kRows>
int dequantize_rows(const DequantizeParams& p, int vec, cudaStream_t s) {
    auto* kernel =
        vec == 32 ? mc_fp4_dequantize<T, kFormat, 32, kRows> : vec == 16 ? mc_fp4_dequantize<T, kFormat, 16, kRows> : mc_fp4_dequantize<T, kFormat, 0, kRows>;
    return launch(kernel, blocks_for(p.batch * p.rows, p.unit_bits, kRows), kThreads, s, "mc_fp4_dequantize", p);
}

template <typename T, int kFormat>
int dequantize_launch(const DequantizeParams& p, int vec, cudaStream_t s) {
    return many_blocks(blocks_for(p.batch * p.rows, p.unit_bits, 4)) ? dequantize_rows<T, kFormat, 4>(p, vec, s) : dequantize_rows<T, kFormat, 1>(p, vec, s);
}

template <typename T>
int tensor_scale_launch(const void* src, long long rows, long long cols, long long pitch, int batch, float* out, int vec, cudaStream_t s) {
    const auto* in = static_cast<const typename T::type*>(src);
    if (pitch == cols && batch == 1) {  // one run of values, whatever their rows' alignment
        cols *= rows;
        rows = 1;
        pitch = cols;
        vec = is_aligned(src, 32) ? 32 : is_aligned(src, 16) ? 16 : 0;
    }
    const long long units = rows * ((cols + kUnit - 1) / kUnit);
    if (units <= 8192) {  // one per thread of a cluster; at four per thread (9 us) three launches on all SMs are as quick
        auto* kernel = vec == 32 ? mc_fp4_amax_one<T, 32> : vec == 16 ? mc_fp4_amax_one<T, 16> : mc_fp4_amax_one<T, 0>;
        return launch(kernel, 8LL * batch, 1024, s, "mc_fp4_amax_one", in, rows, cols, pitch, out);
    }
    if (int rc = check_rt(cudaMemsetAsync(out, 0, sizeof(float) * static_cast<std::size_t>(batch), s), "cudaMemsetAsync(tensor scale)")) return rc;
    const long long want = (units + kThreads - 1) / kThreads;
    auto* kernel = vec == 32 ? mc_fp4_amax_many<T, 32> : vec == 16 ? mc_fp4_amax_many<T, 16> : mc_fp4_amax_many<T, 0>;
    for (int first = 0; first < batch; first += 65535) {
        const int some = std::min(65535, batch - first);
        const dim3 grid(static_cast<unsigned>(std::min<long long>(want, std::max(1, 8 * sm_count() / some))), static_cast<unsigned>(some));
        kernel<<<grid, kThreads, 0, s>>>(in + static_cast<long long>(first) * rows * pitch, rows, cols, pitch, reinterpret_cast<unsigned*>(out) + first);
        if (int rc = launched("mc_fp4_amax_many")) return rc;
    }
    return launch(mc_fp4_amax_finish, (batch + 255) / 256, 256, s, "mc_fp4_amax_finish", out, batch);
}

int check_dense(const char* who, int type, const void* p, long long rows, long long cols, long long pitch, int batch) {
    if (type != MCD_TYPE_F32 && type != MCD_HALF_BF16 && type != MCD_HALF_F16) return fail(std::string(who) + ": unknown type");
    if (p == nullptr) return fail(std::string(who) + ": null values");
    const std::uintptr_t size = type == MCD_TYPE_F32 ? 4 : 2;
    if ((reinterpret_cast<std::uintptr_t>(p) & (size - 1)) != 0) return fail(std::string(who) + ": values not aligned to their type");
    if (pitch < cols) return fail(std::string(who) + ": the pitch is less than a row");
    if (!fits(batch, rows, pitch, 1LL << 46)) return fail(std::string(who) + ": too many values");
    return 0;
}

}  // namespace

extern "C" long long mcd_fp4_code_pitch(long long cols) { return cols <= 0 ? 0 : (cols + 31) / 32 * 16; }

extern "C" size_t mcd_fp4_codes_bytes(long long rows, long long cols, int batch) {
    if (rows <= 0 || cols <= 0 || batch <= 0) return 0;
    return static_cast<size_t>(batch) * static_cast<size_t>(rows) * static_cast<size_t>(mcd_fp4_code_pitch(cols));
}

extern "C" size_t mcd_fp4_scales_bytes(int format, long long rows, long long cols, int batch) {
    if (rows <= 0 || cols <= 0 || batch <= 0 || (format != MCD_FP4_E8M0_32 && format != MCD_FP4_E4M3_16)) return 0;
    return static_cast<size_t>(batch) * static_cast<size_t>(fp4_geometry(format, rows, cols).matrix_scales);
}

extern "C" int mcd_fp4_tensor_scale(int type, const void* src, long long rows, long long cols, long long pitch, int batch, float* out,
                                    void* stream) {
    const char* who = "mcd_fp4_tensor_scale";
    if (batch < 1) return fail("mcd_fp4_tensor_scale: no matrices");
    if (rows < 1 || cols < 1) return fail("mcd_fp4_tensor_scale: empty matrix");
    if (int rc = check_dense(who, type, src, rows, cols, pitch, batch)) return rc;
    if (out == nullptr || (reinterpret_cast<std::uintptr_t>(out) & 3) != 0) return fail("mcd_fp4_tensor_scale: null or unaligned result");
    if (int rc = check_device_pointers(who, {src, out})) return rc;
    const int vec = rows_aligned(type, src, pitch);
    auto s = static_cast<cudaStream_t>(stream);
    if (type == MCD_TYPE_F32) return tensor_scale_launch<F32>(src, rows, cols, pitch, batch, out, vec, s);
    if (type == MCD_HALF_BF16) return tensor_scale_launch<Bf16>(src, rows, cols, pitch, batch, out, vec, s);
    return tensor_scale_launch<F16>(src, rows, cols, pitch, batch, out, vec, s);
}

extern "C" int mcd_fp4_quantize(int type, const void* src, long long pitch, const mcd_fp4_tensor* dst, void* stream) {
    const char* who = "mcd_fp4_quantize";
    if (int rc = check_fp4(who, dst)) return rc;
    if (int rc = check_dense(who, type, src, dst->rows, dst->cols, pitch, dst->batch)) return rc;
    if (int rc = check_device_pointers(who, {src, dst->codes, dst->scales, dst->tensor_scale})) return rc;
    const Fp4Geometry geo = fp4_geometry(dst->format, dst->rows, dst->cols);
    QuantizeParams p;
    p.src = src;
    p.codes = static_cast<unsigned char*>(dst->codes);
    p.scales = static_cast<unsigned char*>(dst->scales);
    p.tensor_scale = dst->tensor_scale;
    p.rows = dst->rows;
    p.cols = dst->cols;
    p.pitch_elems = pitch;
    p.code_pitch = geo.pitch;
    p.k_tiles = geo.k_tiles;
    p.padded_rows = geo.row_tiles * 128;
    p.batch = dst->batch;
    p.units = static_cast<int>(geo.k_tiles * 4 * geo.block / kUnit);
    p.unit_bits = unit_bits(p.units);
    const int vec = rows_aligned(type, src, pitch);
    auto s = static_cast<cudaStream_t>(stream);
    const bool e8m0 = dst->format == MCD_FP4_E8M0_32;
    if (type == MCD_TYPE_F32) return e8m0 ? quantize_launch<F32, MCD_FP4_E8M0_32>(p, vec, s) : quantize_launch<F32, MCD_FP4_E4M3_16>(p, vec, s);
    if (type == MCD_HALF_BF16) return e8m0 ? quantize_launch<Bf16, MCD_FP4_E8M0_32>(p, vec, s) : quantize_launch<Bf16, MCD_FP4_E4M3_16>(p, vec, s);
    return e8m0 ? quantize_launch<F16, MCD_FP4_E8M0_32>(p, vec, s) : quantize_launch<F16, MCD_FP4_E4M3_16>(p, vec, s);
}

extern "C" int mcd_fp4_dequantize(const mcd_fp4_tensor* src, int type, void* dst, long long pitch, void* stream) {
    const char* who = "mcd_fp4_dequantize";
    if (int rc = check_fp4(who, src)) return rc;
    if (int rc = check_dense(who, type, dst, src->rows, src->cols, pitch, src->batch)) return rc;
    if (int rc = check_device_pointers(who, {dst, src->codes, src->scales, src->tensor_scale})) return rc;
    const Fp4Geometry geo = fp4_geometry(src->format, src->rows, src->cols);
    DequantizeParams p;
    p.codes = static_cast<const unsigned char*>(src->codes);
    p.scales = static_cast<const unsigned char*>(src->scales);
    p.tensor_scale = src->tensor_scale;
    p.dst = dst;
    p.rows = src->rows;
    p.cols = src->cols;
    p.pitch_elems = pitch;
    p.code_pitch = geo.pitch;
    p.k_tiles = geo.k_tiles;
    p.matrix_scales = geo.matrix_scales;
    p.batch = src->batch;
    p.units = static_cast<int>((src->cols + kUnit - 1) / kUnit);
    p.unit_bits = unit_bits(p.units);
    const int vec = rows_aligned(type, dst, pitch);
    auto s = static_cast<cudaStream_t>(stream);
    const bool e8m0 = src->format == MCD_FP4_E8M0_32;
    if (type == MCD_TYPE_F32) return e8m0 ? dequantize_launch<F32, MCD_FP4_E8M0_32>(p, vec, s) : dequantize_launch<F32, MCD_FP4_E4M3_16>(p, vec, s);
    if (type == MCD_HALF_BF16) return e8m0 ? dequantize_launch<Bf16, MCD_FP4_E8M0_32>(p, vec, s) : dequantize_launch<Bf16, MCD_FP4_E4M3_16>(p, vec, s);
    return e8m0 ? dequantize_launch<F16, MCD_FP4_E8M0_32>(p, vec, s) : dequantize_launch<F16, MCD_FP4_E4M3_16>(p, vec, s);
}
