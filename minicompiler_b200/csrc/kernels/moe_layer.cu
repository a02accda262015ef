// mcd_moe_layer: router, gate and up projection, down projection and combination of a mixture-of-experts layer for up to
// 64 tokens, the experts' weights in a microscaled 4-bit format.
//
//   l = R x;  p = softmax(l);  y = sum over the top_k experts e of w_e * D_e (silu(G_e x) * (U_e x))
//
// Few tokens meet many weights: every weight is used for the handful of tokens that chose its expert, so the time is
// that of reading the chosen experts' weights once. Three launches, each a programmatic dependent of the one before it:
//
//   mc_moe_router  one cluster of 8 CTAs per token: logits in 64-bit sums, softmax, the top_k experts
//   mc_moe_up      4-warp CTAs take (expert, 32 rows of G and the same 32 of U): h = silu(G x) * (U x), f32
//   mc_moe_down    a cluster of up to 8 CTAs takes 64 rows of y, its CTAs share the experts and add up what they found
//
// The products: codes are small numbers that f16 holds exactly, so a warp turns 16 rows of codes into f16 fragments
// (one conversion for two codes) and multiplies them with 8 tokens' values by mma.sync m16n8k16, f32 sums. That
// instruction is far from the tensor cores' peak and does not have to be near it: a byte of weights costs 32 multiply-adds
// here. The order of k within a product does not matter, so a lane takes the 8 codes of one 32-bit word and the 8
// matching values of a token, instead of the interleaved order of the fragment's definition.
// Scales: E8M0_32 - 32 columns (one block) are two multiplies into a fresh sum, which then counts scale times; E4M3_16 -
// code * scale is exact in f16 (6 bits, 2^-10 .. 2688), so the codes are scaled before the multiply.
// x and h come to f16 as well, after a power of two per token (x) or per token and expert (h) that takes the largest
// magnitude to [2^14, 2^15): 11 bits are kept of values down to 2^-29 of the largest. bf16 and f16 inputs lose nothing
// above that, h is rounded to 11 bits.

#include "minicompiler_b200_device.h"

#include "device/driver_api.hpp"
#include "device/per_device.hpp"
#include "kernels/fp4_format.cuh"
#include "kernels/fp4_host.hpp"

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

using namespace mcd;

namespace {

constexpr int kTokenTile = 8;        // columns of one mma
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStageK = 256;         // codes per row and stage: 128 bytes
constexpr int kStages = 6;
constexpr int kChunkK = 1024;        // values of a token in shared memory at a time
constexpr int kValuePitch = 2 * (kChunkK + 32);  // bytes; 16 words past a multiple of 32: the four lanes of two tokens cover all banks
constexpr int kMaxSlots = MCD_MOE_MAX_TOKENS * MCD_MOE_MAX_TOP_K;
constexpr int kDownRows = 64;
constexpr int kDownPitch = kDownRows + 4;
constexpr int kRouterCluster = 8;
constexpr int kRouterThreads = 256;

template <int kFormat>
struct Stage {
    static constexpr int kScaleWords = kFormat == MCD_FP4_E8M0_32 ? 2 : 4;  // per row: one for 4 blocks
    static constexpr int kCodeBytes = 16 * 128;
    static constexpr int kBytes = kCodeBytes + kScaleWords * 16 * 4;
};

struct Matrix4 {
    const unsigned char* codes;
    const unsigned char* scales;
    const float* tensor_scale;
    long long matrix_codes, matrix_scales, pitch;
    int k_tiles, stages;  // per row
};

struct MoeParams {
    const unsigned short* x;
    const unsigned short* router;
    unsigned short* y;
    long long ldx, ld_router, ldy;
    int type, tokens, top_k, renormalize, experts;
    int d, f;
    int x_vec;       // rows of x start on 16-byte boundaries
    int router_vec;  // rows of x and of the router do
    Matrix4 gate_up, down;
    int* chosen_out;
    float* weights_out;
    // workspace
    int* chosen;           // [tokens * top_k]
    float* weights;        // [tokens * top_k]
    float* x_shift;        // [tokens]: the power of two that x is multiplied with
    unsigned* h_max;       // [tokens * top_k]: bits of the largest |h|
    float* h;              // [tokens * top_k][f]
};

__device__ __forceinline__ float value16(unsigned short v, int type) {
    return type == MCD_HALF_BF16 ? __uint_as_float(static_cast<unsigned>(v) << 16) : f16_lo(v);
}

__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
    unsigned d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// The power of two that takes a largest magnitude (as bits) to [2^14, 2^15). Zero, infinity and NaN are left alone; the
// exponent stops where the factor or its inverse would leave f32.
__device__ __forceinline__ float shift_for(unsigned max_bits) {
    if (max_bits == 0 || max_bits >= 0x7f800000u) return 1.0f;
    const int e = max(-113, min(120, 14 - (static_cast<int>(max_bits >> 23) - 127)));
    return __uint_as_float(static_cast<unsigned>(e + 127) << 23);
}
__device__ __forceinline__ float inverse_power(float p) { return __uint_as_float((254u << 23) - __float_as_uint(p)); }

__device__ __forceinline__ unsigned smem_u32(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned peer_address(unsigned addr, unsigned rank) {
    unsigned out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
    return out;
}

// ------------------------------------------------------------------------------------------------------------- router

// True when (a, i) comes before (b, j): the larger logit, ties to the lower index, NaN behind every number.
__device__ __forceinline__ bool before(double a, int i, double b, int j) {
    const bool a_nan = a != a, b_nan = b != b;
    if (a_nan != b_nan) return b_nan;
    if (!a_nan && a != b) return a > b;
    return i < j;
}

__global__ void __cluster_dims__(kRouterCluster, 1, 1) __launch_bounds__(kRouterThreads) mc_moe_router(const MoeParams p) {
    __shared__ double logits[MCD_MOE_MAX_EXPERTS];  // of the cluster's first CTA
    __shared__ unsigned warp_max[kRouterThreads / 32];
    const int token = blockIdx.x / kRouterCluster;
    const unsigned rank = cluster_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned short* x = p.x + token * p.ldx;
    const unsigned logits_first = peer_address(smem_u32(logits), 0);
    cluster_sync_all();  // every CTA of the cluster runs before its shared memory is written

    for (int e = static_cast<int>(rank) * (kRouterThreads / 32) + warp; e < p.experts; e += kRouterCluster * (kRouterThreads / 32)) {
        const unsigned short* r = p.router + e * p.ld_router;
        double sum = 0.0;
        if (p.router_vec) {
            for (int c = lane * 8; c + 8 <= p.d; c += 256) {
                const uint4 a = *reinterpret_cast<const uint4*>(x + c), b = *reinterpret_cast<const uint4*>(r + c);
                const unsigned aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // products of 16-bit values are exact in f32
                    sum += static_cast<double>(value16(aw[i] & 0xffffu, p.type) * value16(bw[i] & 0xffffu, p.type));
                    sum += static_cast<double>(value16(aw[i] >> 16, p.type) * value16(bw[i] >> 16, p.type));
                }
            }
        }
        for (int c = (p.router_vec ? p.d / 8 * 8 : 0) + lane; c < p.d; c += 32) sum += static_cast<double>(value16(x[c], p.type)) * value16(r[c], p.type);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(logits_first + 8u * static_cast<unsigned>(e)), "d"(sum) : "memory");
    }
    unsigned largest = 0;
    if (rank == 0) {
        for (int c = threadIdx.x; c < p.d; c += kRouterThreads) largest = max(largest, __float_as_uint(value16(x[c], p.type)) & 0x7fffffffu);
        largest = __reduce_max_sync(0xffffffffu, largest);
        if (lane == 0) warp_max[warp] = largest;
    }
    cluster_sync_all();
    if (rank != 0) return;
    if (threadIdx.x < p.top_k) p.h_max[token * p.top_k + threadIdx.x] = 0u;
    if (warp != 0) return;
    largest = __reduce_max_sync(0xffffffffu, lane < kRouterThreads / 32 ? warp_max[lane] : 0u);
    if (lane == 0) p.x_shift[token] = shift_for(largest);

    // best logit first; then the softmax's sum, one lane's share after the other's in a fixed tree
    constexpr int kPerLane = MCD_MOE_MAX_EXPERTS / 32;
    double top = 0.0;
    float total = 0.0f, kept = 0.0f;
    float mine = 0.0f;  // lane j keeps the weight of the j-th choice
    int my_choice = 0;
    unsigned taken = 0;
    for (int j = 0; j < p.top_k; ++j) {
        double best = 0.0;
        int at = 0x7fffffff;
        bool any = false;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int e = i * 32 + lane;
            if (e < p.experts && !((taken >> i) & 1u)) {
                const double l = logits[e];
                if (!any || before(l, e, best, at)) best = l, at = e, any = true;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double other = __shfl_xor_sync(0xffffffffu, best, o);
            const int other_at = __shfl_xor_sync(0xffffffffu, at, o);
            const bool other_any = __shfl_xor_sync(0xffffffffu, static_cast<int>(any), o) != 0;
            if (other_any && (!any || before(other, other_at, best, at))) best = other, at = other_at, any = true;
        }
        if ((at & 31) == lane) taken |= 1u << (at >> 5);
        if (j == 0) {
            top = best;
            for (int e = lane; e < p.experts; e += 32) total += expf(static_cast<float>(logits[e] - top));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        }
        const float w = expf(static_cast<float>(best - top)) / total;
        kept += w;
        if (lane == j) mine = w, my_choice = at;
    }
    if (lane < p.top_k) {
        const float w = p.renormalize ? mine / kept : mine;
        const int slot = token * p.top_k + lane;
        p.chosen[slot] = my_choice;
        p.weights[slot] = w;
        if (p.chosen_out != nullptr) p.chosen_out[slot] = my_choice;
        if (p.weights_out != nullptr) p.weights_out[slot] = w;
    }
}

// ------------------------------------------------------------------------------------------- rows of codes times tokens

// Experts that somebody chose, in order of their index.
struct Routing {
    int chosen[kMaxSlots];
    short active[MCD_MOE_MAX_EXPERTS];
    int count[MCD_MOE_MAX_EXPERTS];
    int num_active;
    int slots[MCD_MOE_MAX_TOKENS];  // of the expert at work: token * top_k + rank, in that order (a token names it once)
    int num_slots;
};

__device__ __forceinline__ void load_routing(Routing& r, const MoeParams& p) {
    const int all = p.tokens * p.top_k;
    for (int e = threadIdx.x; e < p.experts; e += kThreads) r.count[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < all; i += kThreads) {
        const int e = p.chosen[i];
        r.chosen[i] = e;
        atomicAdd(&r.count[e], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        int n = 0;
        for (int base = 0; base < p.experts; base += 32) {
            const int e = base + static_cast<int>(threadIdx.x);
            const bool used = e < p.experts && r.count[e] > 0;
            const unsigned mask = __ballot_sync(0xffffffffu, used);
            if (used) r.active[n + __popc(mask & ((1u << threadIdx.x) - 1u))] = static_cast<short>(e);
            n += __popc(mask);
        }
        if (threadIdx.x == 0) r.num_active = n;
    }
    __syncthreads();
}

// Slots of expert e into r.slots. The caller has a barrier before (nobody reads the old ones) and after.
__device__ __forceinline__ void list_slots(Routing& r, int e, int all) {
    if (threadIdx.x < 32) {
        int n = 0;
        for (int base = 0; base < all; base += 32) {
            const int i = base + static_cast<int>(threadIdx.x);
            const bool mine = i < all && r.chosen[i] == e;
            const unsigned mask = __ballot_sync(0xffffffffu, mine);
            if (mine) r.slots[n + __popc(mask & ((1u << threadIdx.x) - 1u))] = i;
            n += __popc(mask);
        }
        if (threadIdx.x == 0) r.num_slots = n;
    }
}

// The 16 rows of a warp's tile as it streams them: row[i] of the lane's four 16-byte copies per stage (rows i * 4 + lane / 8)
// and the rows of its scale words.
template <int kFormat>
struct RowStream {
    const unsigned char* codes[4];   // nullptr: no such row
    const unsigned char* scales;     // of row lane % 16: its word in the first scale tile of its row group
    long long pitch;
    int k_tiles;
    unsigned ring;                   // this warp's stages in shared memory

    __device__ __forceinline__ void issue(int s) const {
        const int lane = threadIdx.x & 31;
        const unsigned base = ring + static_cast<unsigned>(s % kStages) * Stage<kFormat>::kBytes;
        const int c = lane & 7;
        const long long at = static_cast<long long>(s) * 128 + c * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 4 + (lane >> 3);
            const bool there = codes[i] != nullptr && at < pitch;
            const unsigned dst = base + row * 128 + ((c ^ (row & 7)) << 4);
            const void* src = there ? codes[i] + at : static_cast<const void*>(scales);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
        }
        const int row = lane & 15;
#pragma unroll
        for (int i = 0; i < Stage<kFormat>::kScaleWords / 2; ++i) {
            const int word = i * 2 + (lane >> 4);
            const int tile = s * Stage<kFormat>::kScaleWords + word;
            const bool there = tile < k_tiles;
            const unsigned dst = base + Stage<kFormat>::kCodeBytes + (word * 16 + row) * 4;
            const void* src = there ? scales + static_cast<long long>(tile) * kFp4TileBytes : scales;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
        }
    }
};

__device__ __forceinline__ void copies_done_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

__device__ __forceinline__ unsigned lds32(unsigned a) {
    unsigned v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint4 lds128(unsigned a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma16816(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned mul_f16x2(unsigned a, unsigned b) {
    unsigned d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Two e8m0 bytes -> two f32 (bf16 holds every power of two they stand for, and NaN).
__device__ __forceinline__ void e8m0x2(unsigned two, float& lo, float& hi) {
    unsigned d;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, t;\n\t}" : "=r"(d) : "r"(two));
    lo = __uint_as_float(d << 16);
    hi = __uint_as_float(d & 0xffff0000u);
}

// One stage: 16 rows x 256 codes of the ring slot at `base`, times the values at `values` (f16, token rows kValuePitch apart).
template <int kFormat>
__device__ __forceinline__ void multiply_stage(unsigned base, unsigned values, float (&acc)[4]) {
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const unsigned scales = base + Stage<kFormat>::kCodeBytes;
    const unsigned v_at = values + static_cast<unsigned>(g * kValuePitch + t * 16);
    const unsigned sel = static_cast<unsigned>(t >> 1) * 0x11u;
    float scale_lo[4], scale_hi[4];
    unsigned word_lo = 0, word_hi = 0;
#pragma unroll
    for (int b = 0; b < kStageK / 32; ++b) {
        const unsigned at = base + static_cast<unsigned>(g * 128 + ((b ^ g) << 4) + t * 4);
        const unsigned lo = lds32(at), hi = lds32(at + 8 * 128);
        const uint4 v = lds128(v_at + b * 64);
        unsigned a[4], c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = fp4_decode2((lo >> (8 * i)) & 0xffu);
            c[i] = fp4_decode2((hi >> (8 * i)) & 0xffu);
        }
        if constexpr (kFormat == MCD_FP4_E8M0_32) {
            if ((b & 3) == 0) {
                word_lo = lds32(scales + (b >> 2) * 64 + g * 4), word_hi = lds32(scales + (b >> 2) * 64 + (g + 8) * 4);
                e8m0x2(word_lo & 0xffffu, scale_lo[0], scale_lo[1]);
                e8m0x2(word_lo >> 16, scale_lo[2], scale_lo[3]);
                e8m0x2(word_hi & 0xffffu, scale_hi[0], scale_hi[1]);
                e8m0x2(word_hi >> 16, scale_hi[2], scale_hi[3]);
            }
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma16816(s, a[0], c[0], a[1], c[1], v.x, v.y);
            mma16816(s, a[2], c[2], a[3], c[3], v.z, v.w);
            acc[0] = fmaf(s[0], scale_lo[b & 3], acc[0]);
            acc[1] = fmaf(s[1], scale_lo[b & 3], acc[1]);
            acc[2] = fmaf(s[2], scale_hi[b & 3], acc[2]);
            acc[3] = fmaf(s[3], scale_hi[b & 3], acc[3]);
        } else {
            if ((b & 1) == 0) word_lo = lds32(scales + (b >> 1) * 64 + g * 4), word_hi = lds32(scales + (b >> 1) * 64 + (g + 8) * 4);
            const unsigned which = sel + (b & 1 ? 0x22u : 0u);
            unsigned s_lo, s_hi;
            asm("{\n\t.reg .b32 w;\n\t.reg .b16 t;\n\tprmt.b32 w, %1, 0, %2;\n\tcvt.u16.u32 t, w;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(s_lo) : "r"(word_lo), "r"(which));
            asm("{\n\t.reg .b32 w;\n\t.reg .b16 t;\n\tprmt.b32 w, %1, 0, %2;\n\tcvt.u16.u32 t, w;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(s_hi) : "r"(word_hi), "r"(which));
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = mul_f16x2(a[i], s_lo), c[i] = mul_f16x2(c[i], s_hi);
            mma16816(acc, a[0], c[0], a[1], c[1], v.x, v.y);
            mma16816(acc, a[2], c[2], a[3], c[3], v.z, v.w);
        }
    }
}

// acc = 16 rows (this warp's) x 8 tokens over the whole of k. `stage_values(first, count)` has the CTA's threads bring values
// first .. first + count of the current tokens to shared memory.
template <int kFormat, typename Values>
__device__ __forceinline__ void multiply_rows(const RowStream<kFormat>& rows, int stages, unsigned values, float (&acc)[4], Values&& stage_values) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = 0.0f;
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        if (s < stages) rows.issue(s);
        copies_done_group();
    }
    constexpr int kPerChunk = kChunkK / kStageK;
    for (int s = 0; s < stages; ++s) {
        if (s % kPerChunk == 0) {
            __syncthreads();  // the chunk before has been read
            stage_values(s * kStageK, min(kChunkK, (stages - s) * kStageK));
            __syncthreads();
        }
        copies_wait<kStages - 2>();
        __syncwarp();
        multiply_stage<kFormat>(rows.ring + static_cast<unsigned>(s % kStages) * Stage<kFormat>::kBytes,
                                values + static_cast<unsigned>(s % kPerChunk) * kStageK * 2, acc);
        __syncwarp();
        if (s + kStages - 1 < stages) rows.issue(s + kStages - 1);
        copies_done_group();
    }
    copies_wait<0>();
    __syncwarp();
}

// Rows of a warp's tile: row_of(i) for i = 0 .. 15, negative where there is none.
template <int kFormat, typename RowOf>
__device__ __forceinline__ void aim(RowStream<kFormat>& s, const Matrix4& m, int expert, unsigned ring, RowOf&& row_of) {
    const int lane = threadIdx.x & 31;
    const unsigned char* codes = m.codes + expert * m.matrix_codes;
    const unsigned char* scales = m.scales + expert * m.matrix_scales;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = row_of(i * 4 + (lane >> 3));
        s.codes[i] = r < 0 ? nullptr : codes + r * m.pitch;
    }
    const int r = max(0, row_of(lane & 15));  // a row that is not there: its codes are 0, any scale of this matrix but NaN would do
    s.scales = scales + fp4_scale_offset(r, 0, m.k_tiles);
    s.pitch = m.pitch;
    s.k_tiles = m.k_tiles;
    s.ring = ring;
}

__device__ __forceinline__ void store_values(unsigned values, int token, int k, const float (&v)[8]) {
    const unsigned a = values + static_cast<unsigned>(token * kValuePitch + k * 2);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(pack_f16(v[0], v[1])), "r"(pack_f16(v[2], v[3])),
                 "r"(pack_f16(v[4], v[5])), "r"(pack_f16(v[6], v[7]))
                 : "memory");
}

template <int kFormat>
constexpr int kRingBytes = kWarps * kStages * Stage<kFormat>::kBytes;
constexpr int kValueBytes = kTokenTile * kValuePitch;

template <int kFormat>
__global__ void __launch_bounds__(kThreads) mc_moe_up(const MoeParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Routing routing;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned values = smem_u32(smem);
    const unsigned ring = values + kValueBytes + static_cast<unsigned>(warp * kStages * Stage<kFormat>::kBytes);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    load_routing(routing, p);
    const int groups = (p.f + 127) / 128 * 4;  // 32 rows of G each
    const int items = routing.num_active * groups;
    const int all = p.tokens * p.top_k;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int expert = routing.active[item / groups];
        const int group = item % groups;
        // Rows of a 128-row scale tile that share 32 bytes of scales: two neighbours in each of the four groups of 32.
        auto row_in_f = [&](int g) { return (group >> 2) * 128 + 32 * (g >> 1) + 8 * (group & 3) + 2 * warp + (g & 1); };
        RowStream<kFormat> rows;
        aim(rows, p.gate_up, expert, ring, [&](int i) {
            const int r = row_in_f(i & 7);
            return r >= p.f ? -1 : i < 8 ? r : p.f + r;
        });
        __syncthreads();
        list_slots(routing, expert, all);
        __syncthreads();
        const float scale = p.gate_up.tensor_scale != nullptr ? p.gate_up.tensor_scale[expert] : 1.0f;
        for (int first = 0; first < routing.num_slots; first += kTokenTile) {
            const int here = min(kTokenTile, routing.num_slots - first);
            float acc[4];
            multiply_rows<kFormat>(rows, p.gate_up.stages, values, acc, [&](int k0, int count) {
                for (int i = threadIdx.x; i < here * (count / 8); i += kThreads) {
                    const int n = i / (count / 8), k = (i - n * (count / 8)) * 8;
                    const int token = routing.slots[first + n] / p.top_k;
                    const unsigned short* x = p.x + token * p.ldx;
                    const float shift = p.x_shift[token];
                    float v[8];
                    const int c = k0 + k;
                    if (p.x_vec && c + 8 <= p.d) {
                        const uint4 q = *reinterpret_cast<const uint4*>(x + c);
                        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[2 * j] = value16(w[j] & 0xffffu, p.type) * shift, v[2 * j + 1] = value16(w[j] >> 16, p.type) * shift;
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = c + j < p.d ? value16(x[c + j], p.type) * shift : 0.0f;
                    }
                    store_values(values, n, k, v);
                }
            });
            const int g = lane >> 2, t = lane & 3;
            const int r = row_in_f(g);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = 2 * t + j;
                unsigned largest = 0;
                if (n < here && r < p.f) {
                    const int slot = routing.slots[first + n];
                    const float back = inverse_power(p.x_shift[slot / p.top_k]) * scale;
                    const float gate = acc[j] * back, up = acc[2 + j] * back;
                    const float h = gate / (1.0f + expf(-gate)) * up;
                    p.h[static_cast<long long>(slot) * p.f + r] = h;
                    largest = __float_as_uint(h) & 0x7fffffffu;
                }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
                if (g == 0 && n < here && largest != 0) atomicMax(p.h_max + routing.slots[first + n], largest);
            }
        }
    }
}

template <int kFormat>
__global__ void __launch_bounds__(kThreads) mc_moe_down(const MoeParams p, int cluster) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Routing routing;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* sums = reinterpret_cast<float*>(smem);  // [tokens][kDownPitch]
    const unsigned values = smem_u32(smem) + static_cast<unsigned>(MCD_MOE_MAX_TOKENS * kDownPitch * 4);
    const unsigned ring = values + kValueBytes + static_cast<unsigned>(warp * kStages * Stage<kFormat>::kBytes);
    const int rank = cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int group = blockIdx.x / cluster;  // 64 rows of y: one half of the 16 rows in each group of 32 of a 128-row tile
    asm volatile("griddepcontrol.wait;" ::: "memory");
    load_routing(routing, p);
    for (int i = threadIdx.x; i < p.tokens * kDownPitch; i += kThreads) sums[i] = 0.0f;
    const int all = p.tokens * p.top_k;
    auto row_in_y = [&](int i) { return (group >> 1) * 128 + 32 * (i >> 2) + 16 * (group & 1) + 4 * warp + (i & 3); };
    for (int a = rank; a < routing.num_active; a += cluster) {
        const int expert = routing.active[a];
        RowStream<kFormat> rows;
        aim(rows, p.down, expert, ring, [&](int i) {
            const int r = row_in_y(i);
            return r < p.d ? r : -1;
        });
        __syncthreads();
        list_slots(routing, expert, all);
        __syncthreads();
        const float scale = p.down.tensor_scale != nullptr ? p.down.tensor_scale[expert] : 1.0f;
        for (int first = 0; first < routing.num_slots; first += kTokenTile) {
            const int here = min(kTokenTile, routing.num_slots - first);
            float acc[4];
            multiply_rows<kFormat>(rows, p.down.stages, values, acc, [&](int k0, int count) {
                for (int i = threadIdx.x; i < here * (count / 8); i += kThreads) {
                    const int n = i / (count / 8), k = (i - n * (count / 8)) * 8;
                    const int slot = routing.slots[first + n];
                    const float* h = p.h + static_cast<long long>(slot) * p.f;
                    const float shift = shift_for(p.h_max[slot]);
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = k0 + k + j < p.f ? h[k0 + k + j] * shift : 0.0f;
                    store_values(values, n, k, v);
                }
            });
            const int g = lane >> 2, t = lane & 3;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = 2 * t + j;
                if (n < here) {
                    const int slot = routing.slots[first + n];
                    const float back = inverse_power(shift_for(p.h_max[slot])) * scale;
                    const float w = p.weights[slot];
                    // this warp's 16 columns; nobody else adds to them
                    float* sum = sums + slot / p.top_k * kDownPitch + warp * 16;
                    sum[g] += w * (acc[j] * back);
                    sum[g + 8] += w * (acc[2 + j] * back);
                }
            }
        }
    }
    __syncthreads();
    if (cluster > 1) cluster_sync_all();
    // Every CTA of the cluster finishes its share of the elements: the partial sums in rank order.
    const unsigned mine = smem_u32(sums);
    const int count = p.tokens * kDownRows;
    for (int i = rank * kThreads + static_cast<int>(threadIdx.x); i < count; i += cluster * kThreads) {
        const int token = i / kDownRows, c = i - token * kDownRows;
        const unsigned at = mine + static_cast<unsigned>(token * kDownPitch + c) * 4u;
        float v = 0.0f;
        for (int z = 0; z < cluster; ++z) {
            float part;
            if (cluster > 1) {
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(peer_address(at, static_cast<unsigned>(z))) : "memory");
            } else {
                part = sums[token * kDownPitch + c];
            }
            v += part;
        }
        const int w = c >> 4, k = c & 15;
        const int r = (group >> 1) * 128 + 32 * (k >> 2) + 16 * (group & 1) + 4 * w + (k & 3);
        if (r < p.d) {
            unsigned short out;
            if (p.type == MCD_HALF_BF16) {
                asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(out) : "f"(v));
            } else {
                asm("cvt.rn.f16.f32 %0, %1;" : "=h"(out) : "f"(v));
            }
            p.y[token * p.ldy + r] = out;
        }
    }
    if (cluster > 1) cluster_sync_all();  // shared memory stays until the last peer has read it
}

template <int kFormat>
constexpr int kUpSmem = kValueBytes + kRingBytes<kFormat>;
template <int kFormat>
constexpr int kDownSmem = MCD_MOE_MAX_TOKENS * kDownPitch * 4 + kValueBytes + kRingBytes<kFormat>;

// ---------------------------------------------------------------------------------------------------------- host side

template <typename... Params, typename... Args>
int launch(void (*kernel)(Params...), unsigned grid, unsigned cluster, unsigned threads, size_t smem, cudaStream_t s, const char* what, Args... args) {
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid, 1, 1);
    config.blockDim = dim3(threads, 1, 1);
    config.dynamicSmemBytes = smem;
    config.stream = s;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return check_rt(cudaLaunchKernelEx(&config, kernel, args...), what);
}

template <int kFormat>
int launch_layer(const MoeParams& p, cudaStream_t s) {
    static PerDeviceOnce configured;
    int device = 0;
    if (int rc = check_rt(cudaGetDevice(&device), "cudaGetDevice")) return rc;
    if (configured.first_use(device)) {
        cudaError_t err = cudaFuncSetAttribute(mc_moe_up<kFormat>, cudaFuncAttributeMaxDynamicSharedMemorySize, kUpSmem<kFormat>);
        if (err == cudaSuccess) err = cudaFuncSetAttribute(mc_moe_down<kFormat>, cudaFuncAttributeMaxDynamicSharedMemorySize, kDownSmem<kFormat>);
        if (int rc = check_rt(err, "cudaFuncSetAttribute(max dynamic shared memory)")) {
            configured.forget(device);
            return rc;
        }
    }
    // The router's clusters are declared with the kernel.
    if (int rc = launch(mc_moe_router, static_cast<unsigned>(p.tokens * kRouterCluster), 1, kRouterThreads, 0, s, "mc_moe_router", p)) return rc;
    const int reached = std::min(p.experts, p.tokens * p.top_k);
    const long long most = static_cast<long long>(reached) * ((p.f + 127) / 128 * 4);
    const auto up_grid = static_cast<unsigned>(std::min<long long>(most, 2LL * sm_count()));
    if (int rc = launch(mc_moe_up<kFormat>, up_grid, 1, kThreads, kUpSmem<kFormat>, s, "mc_moe_up", p)) return rc;
    int cluster = 8;
    while (cluster > reached) cluster /= 2;
    const auto down_grid = static_cast<unsigned>((p.d + 127) / 128 * 2 * cluster);
    return launch(mc_moe_down<kFormat>, down_grid, static_cast<unsigned>(cluster), kThreads, kDownSmem<kFormat>, s, "mc_moe_down", p, cluster);
}

size_t rounded(size_t bytes) { return (bytes + 15) / 16 * 16; }

Matrix4 matrix_of(const mcd_fp4_tensor& t) {
    const Fp4Geometry geo = fp4_geometry(t.format, t.rows, t.cols);
    Matrix4 m;
    m.codes = static_cast<const unsigned char*>(t.codes);
    m.scales = static_cast<const unsigned char*>(t.scales);
    m.tensor_scale = t.tensor_scale;
    m.matrix_codes = geo.matrix_codes;
    m.matrix_scales = geo.matrix_scales;
    m.pitch = geo.pitch;
    m.k_tiles = static_cast<int>(geo.k_tiles);
    m.stages = static_cast<int>((t.cols + kStageK - 1) / kStageK);
    return m;
}

}  // namespace

extern "C" size_t mcd_moe_workspace(int tokens, int experts, int top_k, long long d, long long f) {
    if (tokens < 1 || tokens > MCD_MOE_MAX_TOKENS || experts < 1 || top_k < 1 || top_k > MCD_MOE_MAX_TOP_K || d < 1 || f < 1) return 0;
    const size_t slots = static_cast<size_t>(tokens) * static_cast<size_t>(top_k);
    return 3 * rounded(slots * 4) + rounded(static_cast<size_t>(tokens) * 4) + rounded(slots * static_cast<size_t>(f) * 4);
}

extern "C" int mcd_moe_layer(const mcd_moe_args* args, void* stream) {
    const char* who = "mcd_moe_layer";
    if (args == nullptr) return fail("mcd_moe_layer: null arguments");
    if (args->type != MCD_HALF_BF16 && args->type != MCD_HALF_F16) return fail("mcd_moe_layer: x, router and y are bf16 or f16");
    if (args->tokens < 1 || args->tokens > MCD_MOE_MAX_TOKENS) {
        return fail("mcd_moe_layer: 1 to " + std::to_string(MCD_MOE_MAX_TOKENS) + " tokens per call, got " + std::to_string(args->tokens));
    }
    if (int rc = check_fp4(who, &args->gate_up)) return rc;
    if (int rc = check_fp4(who, &args->down)) return rc;
    const mcd_fp4_tensor &gu = args->gate_up, &dn = args->down;
    const int experts = gu.batch;
    if (experts > MCD_MOE_MAX_EXPERTS) return fail("mcd_moe_layer: at most " + std::to_string(MCD_MOE_MAX_EXPERTS) + " experts");
    if (dn.batch != experts) return fail("mcd_moe_layer: gate_up and down have different numbers of experts");
    if (gu.format != dn.format) return fail("mcd_moe_layer: gate_up and down differ in format");
    if (gu.rows % 2 != 0 || gu.rows / 2 != dn.cols) return fail("mcd_moe_layer: gate_up has 2f rows where down has f columns");
    if (gu.cols != dn.rows) return fail("mcd_moe_layer: gate_up's columns are down's rows (d)");
    if (gu.cols > (1 << 24) || dn.cols > (1 << 24)) return fail("mcd_moe_layer: d and f are at most 2^24");
    if (args->top_k < 1 || args->top_k > MCD_MOE_MAX_TOP_K || args->top_k > experts) {
        return fail("mcd_moe_layer: top_k is 1 to " + std::to_string(std::min(MCD_MOE_MAX_TOP_K, experts)) + ", got " + std::to_string(args->top_k));
    }
    if (args->x == nullptr || args->router == nullptr || args->y == nullptr) return fail("mcd_moe_layer: null x, router or y");
    if (!is_aligned(args->x, 2) || !is_aligned(args->router, 2) || !is_aligned(args->y, 2)) return fail("mcd_moe_layer: x, router or y is not aligned to its type");
    const long long d = gu.cols, f = dn.cols;
    if (args->ldx < d || args->ld_router < d || args->ldy < d) return fail("mcd_moe_layer: a leading dimension is less than d");
    if (!fits(MCD_MOE_MAX_EXPERTS, args->ldx, 1, 1LL << 46) || !fits(MCD_MOE_MAX_EXPERTS, args->ld_router, 1, 1LL << 46) ||
        !fits(MCD_MOE_MAX_EXPERTS, args->ldy, 1, 1LL << 46)) {
        return fail("mcd_moe_layer: a leading dimension is too large");
    }
    if (!is_aligned(args->chosen, 4) || !is_aligned(args->weights, 4)) return fail("mcd_moe_layer: unaligned chosen or weights");
    const size_t need = mcd_moe_workspace(args->tokens, experts, args->top_k, d, f);
    if (args->workspace == nullptr || args->workspace_bytes < need) return fail("mcd_moe_layer: needs " + std::to_string(need) + " bytes of workspace");
    if (!is_aligned(args->workspace, 16)) return fail("mcd_moe_layer: the workspace needs 16-byte alignment");
    if (int rc = check_device_pointers(who, {args->x, args->router, gu.codes, gu.scales, gu.tensor_scale, dn.codes, dn.scales, dn.tensor_scale, args->y,
                                             args->chosen, args->weights, args->workspace})) {
        return rc;
    }
    MoeParams p;
    p.x = static_cast<const unsigned short*>(args->x);
    p.router = static_cast<const unsigned short*>(args->router);
    p.y = static_cast<unsigned short*>(args->y);
    p.ldx = args->ldx;
    p.ld_router = args->ld_router;
    p.ldy = args->ldy;
    p.type = args->type;
    p.tokens = args->tokens;
    p.top_k = args->top_k;
    p.renormalize = args->renormalize;
    p.experts = experts;
    p.d = static_cast<int>(d);
    p.f = static_cast<int>(f);
    p.x_vec = is_aligned(args->x, 16) && args->ldx % 8 == 0;
    p.router_vec = p.x_vec && is_aligned(args->router, 16) && args->ld_router % 8 == 0;
    p.gate_up = matrix_of(gu);
    p.down = matrix_of(dn);
    p.chosen_out = args->chosen;
    p.weights_out = args->weights;
    const size_t slots = static_cast<size_t>(args->tokens) * static_cast<size_t>(args->top_k);
    auto* at = static_cast<unsigned char*>(args->workspace);
    p.chosen = reinterpret_cast<int*>(at);
    p.weights = reinterpret_cast<float*>(at += rounded(slots * 4));
    p.h_max = reinterpret_cast<unsigned*>(at += rounded(slots * 4));
    p.x_shift = reinterpret_cast<float*>(at += rounded(slots * 4));
    p.h = reinterpret_cast<float*>(at += rounded(static_cast<size_t>(args->tokens) * 4));
    auto s = static_cast<cudaStream_t>(stream);
    return gu.format == MCD_FP4_E8M0_32 ? launch_layer<MCD_FP4_E8M0_32>(p, s) : launch_layer<MCD_FP4_E4M3_16>(p, s);
}
