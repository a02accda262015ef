// mcd_fp4_quantize, mcd_fp4_dequantize, mcd_fp4_tensor_scale: values to and from the microscaled 4-bit formats.
//
// All three move bytes: a value is read once and 0.53 (E8M0_32) or 0.56 (E4M3_16) bytes are written for it, or the
// other way round; a dozen instructions per value lie between. A thread takes 16 consecutive columns - one E4M3 block, or
// half an E8M0 block whose two halves meet through one shuffle - so that codes leave as 8-byte stores and 16-bit
// values arrive as two 16-byte loads.

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
__device__ __forceinline__ typename T::type from_f32(float v) {
    if constexpr (T::kind == MCD_TYPE_F32) {
        return v;
    } else {
        unsigned short h;
        if constexpr (T::kind == MCD_HALF_BF16) {
            asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(h) : "f"(v));
        } else {
            asm("cvt.rn.f16.f32 %0, %1;" : "=h"(h) : "f"(v));
        }
        return h;
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

// The 16 values from column c0 on; zeros behind `cols`. kVec: rows start on 16-byte boundaries.
template <typename T, bool kVec>
__device__ __forceinline__ void load16(const typename T::type* row, long long c0, long long cols, float (&v)[kUnit]) {
    if (kVec && c0 + kUnit <= cols) {
        if constexpr (T::kind == MCD_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 q = __ldcs(reinterpret_cast<const float4*>(row + c0) + i);
                v[4 * i] = q.x, v[4 * i + 1] = q.y, v[4 * i + 2] = q.z, v[4 * i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 q = __ldcs(reinterpret_cast<const uint4*>(row + c0) + i);
                const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[8 * i + 2 * j] = to_f32<T>(static_cast<unsigned short>(w[j] & 0xffffu));
                    v[8 * i + 2 * j + 1] = to_f32<T>(static_cast<unsigned short>(w[j] >> 16));
                }
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i) v[i] = c0 + i < cols ? to_f32<T>(row[c0 + i]) : 0.0f;
}

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

template <typename T, int kFormat, bool kVec>
__global__ void __launch_bounds__(kThreads) mc_fp4_quantize(const QuantizeParams p) {
    const int lanes = 1 << p.unit_bits;
    const int rows_per_block = kThreads >> p.unit_bits;
    const int lane = static_cast<int>(threadIdx.x) & (lanes - 1);
    const long long all_rows = p.batch * p.padded_rows;
    const long long step = static_cast<long long>(gridDim.x) * rows_per_block;
    for (long long base = static_cast<long long>(blockIdx.x) * rows_per_block; base < all_rows; base += step) {
        const long long at = base + (threadIdx.x >> p.unit_bits);
        const bool inside = at < all_rows;
        const long long matrix = inside ? at / p.padded_rows : 0;
        const long long r = inside ? at - matrix * p.padded_rows : 0;
        const bool real = inside && r < p.rows;
        const auto* row = static_cast<const typename T::type*>(p.src) + (matrix * p.rows + r) * p.pitch_elems;
        unsigned char* codes = p.codes + (matrix * p.rows + r) * p.code_pitch;
        unsigned char* scales = p.scales + matrix * (p.padded_rows >> 7) * p.k_tiles * kFp4TileBytes;
        float g = 1.0f;
        if (kFormat == MCD_FP4_E4M3_16 && p.tensor_scale != nullptr) g = p.tensor_scale[matrix];
        // whole warps run every trip: the halves of a block meet in a shuffle
        for (int first = 0; first < p.units; first += lanes) {
            const int unit = first + lane;
            const bool live = unit < p.units;
            const long long c0 = static_cast<long long>(unit) * kUnit;
            float v[kUnit];
            if (real && live && c0 < p.cols) {
                load16<T, kVec>(row, c0, p.cols, v);
            } else {
#pragma unroll
                for (int i = 0; i < kUnit; ++i) v[i] = 0.0f;
            }
            // the largest magnitude as bits: an integer maximum, in which infinity and NaN come out on top
            unsigned amax = 0;
#pragma unroll
            for (int i = 0; i < kUnit; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
            unsigned byte;
            float inverse;
            if (kFormat == MCD_FP4_E8M0_32) {
                amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                const int e = static_cast<int>(amax >> 23) - 2;  // floor(log2 amax) - 2, biased by 127
                byte = amax >= 0x7f800000u ? 255u : static_cast<unsigned>(max(e, 0));
                inverse = __uint_as_float((254u - min(byte, 252u)) << 23);  // 2^-(byte - 127)
            } else {
                const bool g_ok = g > 0.0f && g <= 3.402823466e38f;
                byte = (amax >= 0x7f800000u || !g_ok) ? 0x7fu : e4m3_encode(__fdiv_rn(__uint_as_float(amax), __fmul_rn(6.0f, g)));
                const float s_g = __fmul_rn(e4m3_decode(byte), g);
                inverse = s_g == 0.0f ? 0.0f : fminf(__fdiv_rn(1.0f, s_g), 3.402823466e38f);
            }
            const bool bad = byte == (kFormat == MCD_FP4_E8M0_32 ? 255u : 0x7fu);  // the NaN scales; no rounding gives them
#pragma unroll
            for (int i = 0; i < kUnit; ++i) v[i] = __fmul_rn(v[i], inverse);
            unsigned lo = fp4_encode8(v), hi = fp4_encode8(v + 8);
            if (bad) lo = hi = 0;
            if (real && live && c0 / 2 < p.code_pitch) *reinterpret_cast<uint2*>(codes + c0 / 2) = make_uint2(lo, hi);
            if (inside && live) {
                if (kFormat == MCD_FP4_E8M0_32) {
                    if ((unit & 1) == 0) scales[fp4_scale_offset(r, unit >> 1, p.k_tiles)] = static_cast<unsigned char>(c0 < p.cols && real ? byte : 0u);
                } else {
                    scales[fp4_scale_offset(r, unit, p.k_tiles)] = static_cast<unsigned char>(c0 < p.cols && real ? byte : 0u);
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

template <typename T, int kFormat, bool kVec>
__global__ void __launch_bounds__(kThreads) mc_fp4_dequantize(const DequantizeParams p) {
    const int lanes = 1 << p.unit_bits;
    const int rows_per_block = kThreads >> p.unit_bits;
    const int lane = static_cast<int>(threadIdx.x) & (lanes - 1);
    const long long all_rows = p.batch * p.rows;
    const long long step = static_cast<long long>(gridDim.x) * rows_per_block;
    for (long long at = static_cast<long long>(blockIdx.x) * rows_per_block + (threadIdx.x >> p.unit_bits); at < all_rows; at += step) {
        const long long matrix = at / p.rows;
        const long long r = at - matrix * p.rows;
        const unsigned char* codes = p.codes + at * p.code_pitch;
        const unsigned char* scales = p.scales + matrix * p.matrix_scales;
        auto* row = static_cast<typename T::type*>(p.dst) + at * p.pitch_elems;
        float g = 1.0f;
        if (kFormat == MCD_FP4_E4M3_16 && p.tensor_scale != nullptr) g = p.tensor_scale[matrix];
        for (int unit = lane; unit < p.units; unit += lanes) {
            const long long c0 = static_cast<long long>(unit) * kUnit;
            const uint2 w = __ldcs(reinterpret_cast<const uint2*>(codes + c0 / 2));
            float scale;
            if (kFormat == MCD_FP4_E8M0_32) {
                scale = e8m0_decode(scales[fp4_scale_offset(r, unit >> 1, p.k_tiles)]);
            } else {
                const unsigned byte = scales[fp4_scale_offset(r, unit, p.k_tiles)];
                scale = e4m3_decode(byte);
            }
            float v[kUnit];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                unsigned pairs[4];
                fp4_decode8(i == 0 ? w.x : w.y, pairs);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[8 * i + 2 * j] = f16_lo(pairs[j]) * scale;  // exact: at most 6 significant bits
                    v[8 * i + 2 * j + 1] = f16_hi(pairs[j]) * scale;
                }
            }
            if (kFormat == MCD_FP4_E4M3_16) {
#pragma unroll
                for (int i = 0; i < kUnit; ++i) v[i] *= g;
            }
            if (kVec && c0 + kUnit <= p.cols) {
                if constexpr (T::kind == MCD_TYPE_F32) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        __stcs(reinterpret_cast<float4*>(row + c0) + i, make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float* q = v + 8 * i;
                        __stcs(reinterpret_cast<uint4*>(row + c0) + i,
                               make_uint4(pack2<T>(q[0], q[1]), pack2<T>(q[2], q[3]), pack2<T>(q[4], q[5]), pack2<T>(q[6], q[7])));
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < kUnit; ++i) {
                    if (c0 + i < p.cols) row[c0 + i] = from_f32<T>(v[i]);
                }
            }
        }
    }
}

// ---- the tensor scale: maxima of bit patterns (order does not matter), then one division.

// The largest finite magnitude among this thread's share, as bits.
template <typename T, bool kVec>
__device__ __forceinline__ unsigned amax_share(const typename T::type* src, long long rows, long long cols, long long pitch,
                                               long long first, long long stride) {
    const long long units = (cols + kUnit - 1) / kUnit;
    unsigned amax = 0;
    for (long long u = first; u < rows * units; u += stride) {
        const long long r = u / units;
        float v[kUnit];
        load16<T, kVec>(src + r * pitch, (u - r * units) * kUnit, cols, v);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            const unsigned bits = __float_as_uint(v[i]) & 0x7fffffffu;
            amax = max(amax, bits >= 0x7f800000u ? 0u : bits);
        }
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

template <typename T, bool kVec>
__global__ void __launch_bounds__(1024) mc_fp4_amax_one(const typename T::type* src, long long rows, long long cols, long long pitch, float* out) {
    const typename T::type* matrix = src + static_cast<long long>(blockIdx.x) * rows * pitch;
    const unsigned v = block_max(amax_share<T, kVec>(matrix, rows, cols, pitch, threadIdx.x, blockDim.x));
    if (threadIdx.x == 0) out[blockIdx.x] = scale_of(v);
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) mc_fp4_amax_many(const typename T::type* src, long long rows, long long cols, long long pitch,
                                                             unsigned* out) {
    const typename T::type* matrix = src + static_cast<long long>(blockIdx.y) * rows * pitch;
    const unsigned v = block_max(amax_share<T, kVec>(matrix, rows, cols, pitch, static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x,
                                                     static_cast<long long>(gridDim.x) * kThreads));
    if (threadIdx.x == 0 && v != 0) atomicMax(out + blockIdx.y, v);
}

__global__ void mc_fp4_amax_finish(float* out, int batch) {
    const int i = static_cast<int>(blockIdx.x * blockDim.x + threadIdx.x);
    if (i < batch) out[i] = scale_of(__float_as_uint(out[i]));
}

// How a block of threads takes rows of `units`: a power of two of threads per row, at least one warp-even pair.
int unit_bits(long long units) {
    int bits = 1;
    while (bits < 8 && (1LL << bits) < units) ++bits;
    return bits;
}

unsigned grid_for(long long rows, int bits) {
    const long long rows_per_block = kThreads >> bits;
    const long long blocks = (rows + rows_per_block - 1) / rows_per_block;
    return static_cast<unsigned>(std::max<long long>(1, std::min<long long>(blocks, 1 << 20)));
}

bool rows_aligned(int type, const void* p, long long pitch) {
    return (reinterpret_cast<std::uintptr_t>(p) & 15) == 0 && (pitch * (type == MCD_TYPE_F32 ? 4 : 2)) % 16 == 0;
}

template <typename T, int kFormat>
void quantize_launch(const QuantizeParams& p, bool vec, cudaStream_t s) {
    const unsigned grid = grid_for(p.batch * p.padded_rows, p.unit_bits);
    if (vec) {
        mc_fp4_quantize<T, kFormat, true><<<grid, kThreads, 0, s>>>(p);
    } else {
        mc_fp4_quantize<T, kFormat, false><<<grid, kThreads, 0, s>>>(p);
    }
}

template <typename T, int kFormat>
void dequantize_launch(const DequantizeParams& p, bool vec, cudaStream_t s) {
    const unsigned grid = grid_for(p.batch * p.rows, p.unit_bits);
    if (vec) {
        mc_fp4_dequantize<T, kFormat, true><<<grid, kThreads, 0, s>>>(p);
    } else {
        mc_fp4_dequantize<T, kFormat, false><<<grid, kThreads, 0, s>>>(p);
    }
}

template <typename T>
int tensor_scale_launch(const void* src, long long rows, long long cols, long long pitch, int batch, float* out, bool vec, cudaStream_t s) {
    const auto* in = static_cast<const typename T::type*>(src);
    const long long units = rows * ((cols + kUnit - 1) / kUnit);
    if (units <= 4096) {
        if (vec) {
            mc_fp4_amax_one<T, true><<<batch, 1024, 0, s>>>(in, rows, cols, pitch, out);
        } else {
            mc_fp4_amax_one<T, false><<<batch, 1024, 0, s>>>(in, rows, cols, pitch, out);
        }
        return launched("mc_fp4_amax_one");
    }
    if (int rc = check_rt(cudaMemsetAsync(out, 0, sizeof(float) * static_cast<std::size_t>(batch), s), "cudaMemsetAsync(tensor scale)")) return rc;
    const long long want = std::max<long long>(1, (units + kThreads * 4 - 1) / (kThreads * 4));
    for (int first = 0; first < batch; first += 65535) {
        const int some = std::min(65535, batch - first);
        const dim3 grid(static_cast<unsigned>(std::min<long long>(want, std::max(1, 8 * sm_count() / some))), static_cast<unsigned>(some));
        const auto* part = in + static_cast<long long>(first) * rows * pitch;
        auto* bits = reinterpret_cast<unsigned*>(out) + first;
        if (vec) {
            mc_fp4_amax_many<T, true><<<grid, kThreads, 0, s>>>(part, rows, cols, pitch, bits);
        } else {
            mc_fp4_amax_many<T, false><<<grid, kThreads, 0, s>>>(part, rows, cols, pitch, bits);
        }
        if (int rc = launched("mc_fp4_amax_many")) return rc;
    }
    mc_fp4_amax_finish<<<(batch + 255) / 256, 256, 0, s>>>(out, batch);
    return launched("mc_fp4_amax_finish");
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
    const bool vec = rows_aligned(type, src, pitch);
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
    const bool vec = rows_aligned(type, src, pitch);
    auto s = static_cast<cudaStream_t>(stream);
    const bool e8m0 = dst->format == MCD_FP4_E8M0_32;
    if (type == MCD_TYPE_F32) {
        e8m0 ? quantize_launch<F32, MCD_FP4_E8M0_32>(p, vec, s) : quantize_launch<F32, MCD_FP4_E4M3_16>(p, vec, s);
    } else if (type == MCD_HALF_BF16) {
        e8m0 ? quantize_launch<Bf16, MCD_FP4_E8M0_32>(p, vec, s) : quantize_launch<Bf16, MCD_FP4_E4M3_16>(p, vec, s);
    } else {
        e8m0 ? quantize_launch<F16, MCD_FP4_E8M0_32>(p, vec, s) : quantize_launch<F16, MCD_FP4_E4M3_16>(p, vec, s);
    }
    return launched("mc_fp4_quantize");
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
    const bool vec = rows_aligned(type, dst, pitch);
    auto s = static_cast<cudaStream_t>(stream);
    const bool e8m0 = src->format == MCD_FP4_E8M0_32;
    if (type == MCD_TYPE_F32) {
        e8m0 ? dequantize_launch<F32, MCD_FP4_E8M0_32>(p, vec, s) : dequantize_launch<F32, MCD_FP4_E4M3_16>(p, vec, s);
    } else if (type == MCD_HALF_BF16) {
        e8m0 ? dequantize_launch<Bf16, MCD_FP4_E8M0_32>(p, vec, s) : dequantize_launch<Bf16, MCD_FP4_E4M3_16>(p, vec, s);
    } else {
        e8m0 ? dequantize_launch<F16, MCD_FP4_E8M0_32>(p, vec, s) : dequantize_launch<F16, MCD_FP4_E4M3_16>(p, vec, s);
    }
    return launched("mc_fp4_dequantize");
}
