// mcd_moe_layer: router, gate and up projection, down projection and combination of a mixture-of-experts layer for up to
// 64 tokens, the experts' weights in a microscaled 4-bit format.
//
//   l = R x;  p = softmax(l);  y = sum over the top_k experts e of w_e * D_e (silu(G_e x) * (U_e x))
//
// Few tokens meet many weights: every weight is used for the handful of tokens that chose its expert, so the floor is the
// time of reading the chosen experts' weights once. Three launches, or four, each a programmatic dependent of the one
// before it:
//
//   mc_moe_router  one cluster of 8 CTAs per token: logits in double-length sums, softmax, the top_k experts; x to f16
//   mc_moe_up      8-warp CTAs take (expert, 32 or 64 rows of G and the same of U): h = silu(G x) * (U x), f32
//   mc_moe_level   (where many CTAs read it) h to the two f16 numbers that the down projection multiplies
//   mc_moe_down    a cluster of up to 8 CTAs takes 64 or 32 rows of y, its CTAs share the experts and add up what they found
//
// Where the time goes: for one token and 8 of 64 experts (26.7 MB of weights, 4 us to read) 24 us are the latencies of
// three dependent launches - routing, first copies, one round of multiplies, joining, each a microsecond or two. For 32
// tokens and 128 experts of 2048 x 768 (294 MB, 46 us) 106 to 110 us: 49 up, 44 down. Nothing is full then: instructions are
// issued on 2.3 and 1.8 of 4 slots, DRAM is at 47 and 26 %, the tensor pipe at 20 and 11 %. What is left is latency that 16
// warps per SM, a barrier per round and the chain of load, decode and multiply of a step do not cover.
//
// The products: codes are small numbers that f16 holds exactly, so a warp turns 16 rows of codes into f16 fragments
// (one conversion for two codes) and multiplies them with 8 tokens' values by mma.sync m16n8k16, f32 sums. That
// instruction is far from the tensor cores' peak and does not have to be near it: a byte of weights costs 32 multiply-adds
// here. The order of k within a product does not matter, so a lane takes the 8 codes of one 32-bit word and the 8
// matching values of a token, instead of the interleaved order of the fragment's definition.
// Scales: E8M0_32 - 32 columns (one block) are two multiplies into a fresh sum, which then counts scale times; E4M3_16 -
// code * scale is exact in f16 (6 bits, 2^-10 .. 2688), so the codes are scaled before the multiply.
//
// x and h come to f16 as well, after a power of two that takes the largest magnitude to [2^14, 2^15): one per token for x,
// one per token and expert for h. 11 bits are kept of x's values down to 2^-29 of the largest, so bf16 and f16 inputs lose
// nothing above that. h has the 24 bits of f32 and enters as two f16 numbers, hi and what it leaves times 2^11, which
// keep 22 of them: columns 2 s and 2 s + 1 of a multiply are those of slot s. A multiply has 8 columns and an expert rarely
// more than four tokens, so the second number mostly takes columns that would be empty.
//
// How the weights stream: a CTA has 8 warps, four tiles of 16 rows by two halves of k. Every warp keeps a ring of its own
// in shared memory filled by 16-byte cp.async, three steps of 256 columns ahead of the multiplies and across the ends of
// rows, tokens and experts; two CTAs per SM have some 100 KB in flight, which is what the memory's latency asks for. No
// barrier orders the weights: a warp waits for its own copies. The tokens' values are prefetched into registers one round
// (1024 columns) ahead and pass through two buffers that the CTA shares.

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

constexpr int kTokenTile = 8;        // columns of one mma
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStageK = 256;         // codes per row and step: 128 bytes
constexpr int kMaxSlots = MCD_MOE_MAX_TOKENS * MCD_MOE_MAX_TOP_K;

// How a CTA's warps divide their work: tiles of 16 rows, and halves of the columns of a round. With two halves there are
// twice as many, shorter passes: for a few tokens, which could not occupy the SMs otherwise. With one, what a pass costs
// beside its multiplies (as many instructions as they have, for 1024 columns) is spread over twice the columns. Groups of
// four or of two warps go through passes of their own, each with its barrier: the down projection's form of that, whose
// CTAs must not grow beyond 64 rows.
template <int kHalves, int kGroups, int kColumnTiles = 1>
struct Shape {
    static constexpr int kGroupWarps = kWarps / kGroups;
    static constexpr int kGroupThreads = kGroupWarps * 32;
    static constexpr int kTiles = kGroupWarps / kHalves;
    static constexpr int kColumns = kTokenTile * kColumnTiles;
    static constexpr int kRoundSteps = kHalves * kGroups == 1 ? 4 : kGroups == 4 || kColumnTiles == 2 ? 1 : 2;  // per warp
    static constexpr int kRoundK = kStageK * kRoundSteps * kHalves;
    static constexpr int kValuePitch = 2 * (kRoundK + 32);  // bytes; 16 words past a multiple of 32: the four lanes of two tokens cover all banks
    static constexpr int kValueBytes = kColumns * kValuePitch;
    static constexpr int kPieces = kColumns * kRoundK / 8 / kGroupThreads;  // of 8 values of a column, per thread and round
};

constexpr int kRouterCluster = 8;
constexpr int kRouterThreads = 256;
constexpr int kUpStages = 4;  // depth of a warp's ring

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
    int rounds;           // of a CTA's shape
};

struct MoeParams {
    const unsigned short* x;
    const unsigned short* router;
    unsigned short* y;
    long long ldx, ld_router, ldy;
    int type, tokens, top_k, renormalize, experts;
    int d, f;
    int d_pitch, f_pitch;  // in whole groups of 8
    int f_groups;    // tiles of 8 rows of h: 16 for every 128 rows begun
    int router_vec;  // rows of x and of the router start on 16-byte boundaries
    Matrix4 gate_up, down;
    int* chosen_out;
    float* weights_out;
    // workspace
    int* chosen;              // [tokens * top_k]
    float* weights;           // [tokens * top_k]
    int* h_max;               // [tokens * top_k]: f32 exponent of the largest |h|
    float* x_shift;           // [tokens]: the power of two that x is multiplied with
    unsigned short* x16;      // [tokens][d_pitch]: x in f16 after that
    uint4* h;                 // [tokens * top_k][f_pitch / 8][2]: 8 values in f32; mc_moe_level: 8 hi, then 8 lo in f16
};

__device__ __forceinline__ float value16(unsigned short v, int type) {
    return type == MCD_HALF_BF16 ? __uint_as_float(static_cast<unsigned>(v) << 16) : f16_lo(v);
}

__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
    unsigned d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// The exponent of the power of two that takes magnitudes of f32 exponent `e` (biased) to [2^14, 2^15). Zero, infinity and
// NaN are left alone; it stops where the factor or its inverse would leave f32.
__device__ __forceinline__ int shift_of(int e) { return e == 0 || e >= 255 ? 0 : max(-113, min(120, 14 - (e - 127))); }
__device__ __forceinline__ float power(int e) { return __uint_as_float(static_cast<unsigned>(e + 127) << 23); }
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

// A logit as an unsigned number of the same order; NaN below every number.
__device__ __forceinline__ unsigned long long sort_key(double l) {
    const auto bits = static_cast<unsigned long long>(__double_as_longlong(l));
    if (l != l) return 0ull;
    return bits >> 63 ? ~bits : bits | (1ull << 63);
}

// sum + c is the running sum to twice f32's precision: the exact error of each addition is collected.
__device__ __forceinline__ void add_exactly(float& sum, float& c, float v) {
    const float t = __fadd_rn(sum, v);
    const float b = __fsub_rn(t, sum);
    c = __fadd_rn(c, __fadd_rn(__fsub_rn(sum, __fsub_rn(t, b)), __fsub_rn(v, b)));
    sum = t;
}

__device__ __forceinline__ void add_products(float& sum, float& c, const uint4& a, const uint4& b, int type) {
    const unsigned aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // products of 16-bit values are exact in f32, see far_logit for the range
        add_exactly(sum, c, value16(aw[i] & 0xffffu, type) * value16(bw[i] & 0xffffu, type));
        add_exactly(sum, c, value16(aw[i] >> 16, type) * value16(bw[i] >> 16, type));
    }
}

// The larger ones of two magnitudes (16-bit values without their signs compare as integers) and those of eight values.
__device__ __forceinline__ unsigned packed_max(unsigned most, const uint4& v) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(most) : "r"(w[i] & 0x7fff7fffu));
    return most;
}

// The double-length sum of a warp's lanes.
__device__ __forceinline__ double lanes_sum(const float (&sum)[2], const float (&c)[2]) {
    const float whole = sum[0] + sum[1];
    const bool finite = fabsf(whole) <= 3.402823466e38f;  // an infinite or NaN sum has no error to speak of
    double total = finite ? (static_cast<double>(sum[0]) + sum[1]) + (static_cast<double>(c[0]) + c[1]) : static_cast<double>(whole);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    return total;
}

// Products of bf16 numbers reach from 2^-266 to 2^256. Where a logit leaves f32 above, its sum in f32 is not finite. Below, a
// product is off by 2^-150 at most and 2^24 of them by 2^-126: less than the 2^-48 of all the sum's terms that it is
// good for, if it is 2^-60 or more. All other logits are taken again in 64 bits, which hold every product.
__device__ __forceinline__ bool is_far(double logit) { return !(fabs(logit) >= 0x1p-60 && fabs(logit) <= 3.402823466e38); }

__device__ __noinline__ double far_logit(const unsigned short* x, const unsigned short* r, int d) {
    const int lane = threadIdx.x & 31;
    double sum = 0.0;
#pragma unroll 8
    for (int k = lane; k < d; k += 32) {
        sum = fma(static_cast<double>(value16(x[k], MCD_HALF_BF16)), static_cast<double>(value16(r[k], MCD_HALF_BF16)), sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// exp(d) for d <= 0. A difference of logits has more bits than f32: what is left of it counts as exp(rest) = 1 + rest. Below
// -200 it is 0.
__device__ __forceinline__ float exp_below(double d) {
    d = d < -200.0 ? -200.0 : d;
    const float near = static_cast<float>(d);
    const float e = expf(near);
    return fmaf(e, static_cast<float>(d - near), e);
}

__global__ void __cluster_dims__(kRouterCluster, 1, 1) __launch_bounds__(kRouterThreads) mc_moe_router(const MoeParams p) {
    // used in the cluster's first CTA
    __shared__ double logits[MCD_MOE_MAX_EXPERTS];
    __shared__ unsigned long long keys[MCD_MOE_MAX_EXPERTS];
    __shared__ int order[MCD_MOE_MAX_EXPERTS];
    __shared__ int best[MCD_MOE_MAX_TOP_K];
    __shared__ float warp_sum[kRouterThreads / 32];
    const int token = blockIdx.x / kRouterCluster;
    const unsigned rank = cluster_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const unsigned short* x = p.x + token * p.ldx;
    const unsigned logits_first = peer_address(smem_u32(logits), 0);
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    unsigned largest = 0;  // |x| as bits, packed 16-bit pairs: every warp sees all of x on its first expert
    bool started = false;
    for (int e = static_cast<int>(rank) * (kRouterThreads / 32) + warp; e < p.experts || !started; e += kRouterCluster * (kRouterThreads / 32)) {
        const unsigned short* r = p.router + min(e, p.experts - 1) * p.ld_router;
        float sum[2] = {0.0f, 0.0f}, c[2] = {0.0f, 0.0f};
        int at = lane * 8;
        if (p.router_vec) {
            for (; at + 768 + 8 <= p.d; at += 1024) {  // four loads of each row in flight
                uint4 a[4], b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i] = *reinterpret_cast<const uint4*>(x + at + 256 * i);
                    b[i] = *reinterpret_cast<const uint4*>(r + at + 256 * i);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    add_products(sum[i & 1], c[i & 1], a[i], b[i], p.type);
                    largest = packed_max(largest, a[i]);
                }
            }
            for (; at + 8 <= p.d; at += 256) {
                const uint4 a = *reinterpret_cast<const uint4*>(x + at);
                add_products(sum[0], c[0], a, *reinterpret_cast<const uint4*>(r + at), p.type);
                largest = packed_max(largest, a);
            }
        }
        // Rows that start anywhere: eight loads of each in flight (one token, 1282 columns: the layer takes 24 us, one by one 35).
        for (int base = p.router_vec ? p.d / 8 * 8 : 0; base < p.d; base += 256) {
            unsigned short a[8], b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k = base + 32 * i + lane;
                a[i] = k < p.d ? x[k] : static_cast<unsigned short>(0);
                b[i] = k < p.d ? r[k] : static_cast<unsigned short>(0);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                add_exactly(sum[i & 1], c[i & 1], value16(a[i], p.type) * value16(b[i], p.type));
                largest = packed_max(largest, make_uint4(a[i], 0, 0, 0));
            }
        }
        double total = lanes_sum(sum, c);
        // `largest` speaks for all of x from the first expert on; a token of zeros (padding) needs no second look
        if (p.type == MCD_HALF_BF16 && is_far(total) && (total != 0.0 || __any_sync(0xffffffffu, largest != 0))) total = far_logit(x, r, p.d);
        if (!started) {  // the first CTA of the cluster runs before its shared memory is written
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            started = true;
        }
        if (e < p.experts && lane == 0) {
            asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(logits_first + 8u * static_cast<unsigned>(e)), "d"(total) : "memory");
        }
    }
    // Every CTA of the cluster knows the token's largest magnitude and brings its share of x to f16.
    largest = __reduce_max_sync(0xffffffffu, max(largest & 0xffffu, largest >> 16));
    const float shift = power(shift_of(static_cast<int>(__float_as_uint(value16(static_cast<unsigned short>(largest), p.type)) >> 23)));
    for (int c = static_cast<int>(rank) * kRouterThreads + static_cast<int>(threadIdx.x); c < p.d_pitch; c += kRouterCluster * kRouterThreads) {
        const float v = c < p.d ? value16(x[c], p.type) * shift : 0.0f;
        p.x16[token * static_cast<long long>(p.d_pitch) + c] = static_cast<unsigned short>(pack_f16(v, 0.0f) & 0xffffu);
    }
    if (rank == 0) {
        if (threadIdx.x == 0) p.x_shift[token] = shift;
        for (int e = threadIdx.x; e < p.experts; e += kRouterThreads) order[e] = 0;
        if (threadIdx.x < p.top_k) p.h_max[token * p.top_k + threadIdx.x] = 0;
    }
    cluster_sync_all();
    if (rank != 0) return;

    for (int e = threadIdx.x; e < p.experts; e += kRouterThreads) keys[e] = sort_key(logits[e]);
    __syncthreads();
    // An expert's place is the number of experts that come before it: the larger logit, ties to the lower index. Where there
    // are fewer experts than threads, several share the comparisons of one.
    int spread = 32 - __clz(p.experts - 1);  // experts in a power of two
    if (p.experts == 1) spread = 0;
    const int shares = max(1, kRouterThreads >> spread);
    for (int i = threadIdx.x; (i & ((1 << spread) - 1)) < p.experts && i < (shares << spread); i += kRouterThreads) {
        const int e = i & ((1 << spread) - 1), share = i >> spread;
        const unsigned long long key = keys[e];
        int before = 0;
#pragma unroll 8
        for (int j = share; j < p.experts; j += shares) {
            const unsigned long long other = keys[j];
            before += other > key || (other == key && j < e) ? 1 : 0;
        }
        if (before != 0) atomicAdd(&order[e], before);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.experts; e += kRouterThreads) {
        if (order[e] < p.top_k) best[order[e]] = e;
    }
    __syncthreads();
    const double top = logits[best[0]];
    float total = 0.0f;
    for (int e = threadIdx.x; e < p.experts; e += kRouterThreads) total += exp_below(logits[e] - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) warp_sum[warp] = total;
    __syncthreads();
    if (warp != 0) return;
    total = 0.0f;
    for (int w = 0; w < kRouterThreads / 32; ++w) total += warp_sum[w];
    float weight = 0.0f, kept = 0.0f;
    if (lane < p.top_k) weight = exp_below(logits[best[lane]] - top) / total;
    for (int j = 0; j < p.top_k; ++j) kept += __shfl_sync(0xffffffffu, weight, j);
    if (lane < p.top_k) {
        if (p.renormalize) weight /= kept;
        const int slot = token * p.top_k + lane;
        p.chosen[slot] = best[lane];
        p.weights[slot] = weight;
        if (p.chosen_out != nullptr) p.chosen_out[slot] = best[lane];
        if (p.weights_out != nullptr) p.weights_out[slot] = weight;
    }
}

// ------------------------------------------------------------------------------------------- rows of codes times tokens

// The experts that somebody chose, in order of their index, and who chose them. The order of an expert's slots is left to
// the atomics: each is a column of its own, and nothing is added up over an expert's columns.
struct Routing {
    short active[MCD_MOE_MAX_EXPERTS];
    short start[MCD_MOE_MAX_EXPERTS + 1];  // of each active expert's slots
    short slots[kMaxSlots];                // token * top_k + rank
    unsigned char tokens[kMaxSlots];       // of each of them
    int num_active;
};

// `scratch`: an int per expert. Waits for the launch before this one; ends with a barrier.
__device__ __forceinline__ void load_routing(Routing& r, int* scratch, const MoeParams& p) {
    const int all = p.tokens * p.top_k;
    if (all <= 32) {
        // One warp, without counting: a lane per slot, equal experts found by a vote.
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x;
            const int e = lane < all ? p.chosen[lane] : 0x7fffffff;
            const unsigned mine = __match_any_sync(0xffffffffu, e);
            const bool first = lane < all && (mine & ((1u << lane) - 1u)) == 0;
            const unsigned firsts = __ballot_sync(0xffffffffu, first);
            int experts_before = 0, slots_before = 0;
            for (unsigned left = firsts; left != 0; left &= left - 1) {
                const int at = __ffs(left) - 1;
                const int other = __shfl_sync(0xffffffffu, e, at);
                const int count = __popc(__shfl_sync(0xffffffffu, mine, at));
                if (other < e) ++experts_before, slots_before += count;
            }
            if (first) {
                r.active[experts_before] = static_cast<short>(e);
                r.start[experts_before] = static_cast<short>(slots_before);
            }
            if (lane < all) {
                const int at = slots_before + __popc(mine & ((1u << lane) - 1u));
                r.slots[at] = static_cast<short>(lane);
                r.tokens[at] = static_cast<unsigned char>(lane / p.top_k);
            }
            if (lane == 0) {
                r.num_active = __popc(firsts);
                r.start[__popc(firsts)] = static_cast<short>(all);
            }
        }
        __syncthreads();
        return;
    }
    for (int e = threadIdx.x; e < p.experts; e += kThreads) scratch[e] = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    constexpr int kMost = kMaxSlots / kThreads;
    int chosen[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int slot = i * kThreads + static_cast<int>(threadIdx.x);
        chosen[i] = slot < all ? p.chosen[slot] : -1;
    }
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        if (chosen[i] >= 0) atomicAdd(&scratch[chosen[i]], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        int n = 0, slots = 0;
        for (int base = 0; base < p.experts; base += 32) {
            const int e = base + static_cast<int>(threadIdx.x);
            const int count = e < p.experts ? scratch[e] : 0;
            const unsigned mask = __ballot_sync(0xffffffffu, count > 0);
            int sum = count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int below = __shfl_up_sync(0xffffffffu, sum, o);
                if (static_cast<int>(threadIdx.x) >= o) sum += below;
            }
            if (count > 0) {
                const int at = n + __popc(mask & ((1u << threadIdx.x) - 1u));
                r.active[at] = static_cast<short>(e);
                r.start[at] = static_cast<short>(slots + sum - count);
                scratch[e] = slots + sum - count;
            }
            n += __popc(mask);
            slots += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (threadIdx.x == 0) {
            r.num_active = n;
            r.start[n] = static_cast<short>(slots);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        if (chosen[i] < 0) continue;
        const int slot = i * kThreads + static_cast<int>(threadIdx.x);
        const int at = atomicAdd(&scratch[chosen[i]], 1);
        r.slots[at] = static_cast<short>(slot);
        r.tokens[at] = static_cast<unsigned char>(slot / p.top_k);
    }
    __syncthreads();
}

// What a CTA works through: rows of an expert against up to 8 of its slots, or 4 (down, two columns each, in one tile of them).
struct Pass {
    int active;  // which of the active experts
    int group;   // of rows (up only)
    int first;   // slot within the expert
};

// Where the 16-byte piece c of a row lies within the row's 128 bytes of a step, so that what lanes read together falls
// into different banks: E8M0_32 reads words of eight rows at a time, E4M3_16 whole pieces of two rows.
template <int kFormat>
__device__ __forceinline__ int piece_at(int row, int c) {
    return kFormat == MCD_FP4_E8M0_32 ? c ^ (row & 7) : c ^ ((row & 1) << 2);
}

// Copies of a warp's 16 rows: four 16-byte pieces per lane and step (rows i * 4 + lane / 8), and the scale words of row
// lane % 16. Nothing is tested on the way: behind the end of a row its last piece comes again, where the values it meets
// are 0 (and its scales are the row's own, so a NaN among them belongs to the row); for a row that is not there another
// one comes, whose sums go nowhere. The copies carry no memory clobber, so that their arithmetic is scheduled among that
// of the multiplies behind them; they write a slot of the ring that nothing else touches until the next wait.
template <int kFormat>
struct RowStream {
    const unsigned char* codes;      // this lane's first row
    const unsigned char* scales;     // of this lane's row, first tile
    long long offset[3];             // of its other rows
    int last_piece, last_tile;

    // `wanted` false: zeros instead, and nothing is read.
    __device__ __forceinline__ void issue(int s, unsigned base, bool wanted) const {
        const int lane = threadIdx.x & 31;
        const unsigned char* from = codes + min(s * 128 + (lane & 7) * 16, last_piece);
        const unsigned dst = base + (lane >> 3) * 128;
        // rows i * 4 + lane / 8: the swizzle goes by the row's low bits
        const unsigned even = dst + (piece_at<kFormat>(lane >> 3, lane & 7) << 4), odd = dst + (piece_at<kFormat>(4 + (lane >> 3), lane & 7) << 4);
        const int bytes = wanted ? 16 : 0;
        copy16(even, from, bytes);
        copy16(odd + 512, from + offset[0], bytes);
        copy16(even + 1024, from + offset[1], bytes);
        copy16(odd + 1536, from + offset[2], bytes);
        const unsigned scales_dst = base + Stage<kFormat>::kCodeBytes + lane * 4;
#pragma unroll
        for (int i = 0; i < Stage<kFormat>::kScaleWords / 2; ++i) {
            const int tile = min(s * Stage<kFormat>::kScaleWords + i * 2 + (lane >> 4), last_tile);
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(scales_dst + i * 128), "l"(scales + static_cast<long long>(tile) * kFp4TileBytes),
                         "r"(bytes >> 2));
        }
    }
    static __device__ __forceinline__ void copy16(unsigned dst, const void* src, int bytes) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes));
    }
};

__device__ __forceinline__ void mma16816(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned mul_f16x2(unsigned a, unsigned b) {
    unsigned d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Four e8m0 bytes -> four f32 (bf16 holds every power of two they stand for, and NaN).
__device__ __forceinline__ void e8m0x4(unsigned word, float (&s)[4]) {
    unsigned lo, hi;
    asm("{\n\t.reg .b16 t, u;\n\tmov.b32 {t, u}, %2;\n\tcvt.rn.bf16x2.ue8m0x2 %0, t;\n\tcvt.rn.bf16x2.ue8m0x2 %1, u;\n\t}" : "=r"(lo), "=r"(hi) : "r"(word));
    s[0] = __uint_as_float(lo << 16);
    s[1] = __uint_as_float(lo & 0xffff0000u);
    s[2] = __uint_as_float(hi << 16);
    s[3] = __uint_as_float(hi & 0xffff0000u);
}
// Two e4m3 bytes -> two f16 pairs, each of one scale twice.
__device__ __forceinline__ void e4m3_pairs(unsigned short two, unsigned& first, unsigned& second) {
    unsigned both;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(both) : "h"(two));
    first = __byte_perm(both, 0, 0x1010);
    second = __byte_perm(both, 0, 0x3232);
}

// Where the 8 values from column k on lie in a token's row (in pieces of 16 bytes), so that the pieces that the four
// lanes of a token read together are neighbours. E8M0_32: lane t takes columns 8 t of every block of 32, which is the
// columns' own order. E4M3_16: lane t takes 32 columns in a row, a quarter of them at a time.
template <int kFormat>
__device__ __forceinline__ int value_piece(int k) {
    const int i = k >> 3;
    return kFormat == MCD_FP4_E8M0_32 ? i : (i & ~15) | (i & 3) << 2 | (i >> 2 & 3);
}

// One step: 16 rows x 256 codes at `base` times the values at `values` (f16, columns kValuePitch apart).
template <int kFormat, int kValuePitch, int kColumnTiles>
__device__ __forceinline__ void multiply_step(const unsigned char* base, const unsigned char* values, float (&acc)[kColumnTiles][2][4]) {
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const unsigned char* v_at = values + g * kValuePitch + t * 16;
    if constexpr (kFormat == MCD_FP4_E8M0_32) {
        const unsigned char* scales = base + Stage<kFormat>::kCodeBytes + g * 4;
        const unsigned char* c_at = base + g * 128 + t * 4;
        float scale_lo[4], scale_hi[4];
#pragma unroll
        for (int b = 0; b < kStageK / 32; ++b) {
            const unsigned lo = *reinterpret_cast<const unsigned*>(c_at + ((b ^ g) << 4));
            const unsigned hi = *reinterpret_cast<const unsigned*>(c_at + ((b ^ g) << 4) + 8 * 128);
            if ((b & 3) == 0) {
                e8m0x4(*reinterpret_cast<const unsigned*>(scales + (b >> 2) * 64), scale_lo);
                e8m0x4(*reinterpret_cast<const unsigned*>(scales + (b >> 2) * 64 + 32), scale_hi);
            }
            unsigned a[4], c[4];
            fp4_decode8(lo, a);
            fp4_decode8(hi, c);
#pragma unroll
            for (int n = 0; n < kColumnTiles; ++n) {
                const uint4 v = *reinterpret_cast<const uint4*>(v_at + n * kTokenTile * kValuePitch + b * 64);
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma16816(s, a[0], c[0], a[1], c[1], v.x, v.y);
                mma16816(s, a[2], c[2], a[3], c[3], v.z, v.w);
                acc[n][b & 1][0] = fmaf(s[0], scale_lo[b & 3], acc[n][b & 1][0]);
                acc[n][b & 1][1] = fmaf(s[1], scale_lo[b & 3], acc[n][b & 1][1]);
                acc[n][b & 1][2] = fmaf(s[2], scale_hi[b & 3], acc[n][b & 1][2]);
                acc[n][b & 1][3] = fmaf(s[3], scale_hi[b & 3], acc[n][b & 1][3]);
            }
        }
    } else {
        // lane t: pieces t and t + 4 of a row, each two blocks of 16; their scales are one half of word (t + 4 q) / 2
        const unsigned char* scales = base + Stage<kFormat>::kCodeBytes + (t >> 1) * 64 + g * 4 + (t & 1) * 2;
        const int c_at = g * 128 + (piece_at<kFormat>(g, t) << 4);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const unsigned char* c_q = base + (c_at ^ (q << 6));  // piece t + 4 lies in the other half of the 128 bytes
            const uint4 lo = *reinterpret_cast<const uint4*>(c_q);
            const uint4 hi = *reinterpret_cast<const uint4*>(c_q + 8 * 128);
            unsigned s_lo[2], s_hi[2];
            e4m3_pairs(*reinterpret_cast<const unsigned short*>(scales + q * 128), s_lo[0], s_lo[1]);
            e4m3_pairs(*reinterpret_cast<const unsigned short*>(scales + q * 128 + 32), s_hi[0], s_hi[1]);
            const unsigned lo_w[4] = {lo.x, lo.y, lo.z, lo.w}, hi_w[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unsigned a[4], c[4];
                fp4_decode8(lo_w[i], a);
                fp4_decode8(hi_w[i], c);
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = mul_f16x2(a[j], s_lo[i >> 1]), c[j] = mul_f16x2(c[j], s_hi[i >> 1]);
#pragma unroll
                for (int n = 0; n < kColumnTiles; ++n) {
                    const uint4 v = *reinterpret_cast<const uint4*>(v_at + n * kTokenTile * kValuePitch + q * 256 + i * 64);
                    mma16816(acc[n][0], a[0], c[0], a[1], c[1], v.x, v.y);
                    mma16816(acc[n][1], a[2], c[2], a[3], c[3], v.z, v.w);
                }
            }
        }
    }
}

// The two projections differ in what a pass is, where values come from and what becomes of the sums; Work supplies these:
//   begin(pass), next(pass)   the CTA's first pass, the one after: false when there is none
//   aim(rows, pass, tile)     point the stream at the warp's rows
//   kParts                    columns of a multiply that a slot takes
//   load(piece, n, k)         8 values of slot n (of all slots) from column k on, as they lie in memory
//   finish(piece, columns)    the same in f16, for each of its columns
//   look(pass, here)          what a lane will need of its two columns, read before the multiplies
//   done(pass, here, tile, side, acc)  a warp's sums, both halves of k
template <int kFormat, int kHalves, int kGroups, int kColumnTiles, int kStages, typename Work>
__device__ __forceinline__ void run_passes(Work& work, const Matrix4& m, const Routing& routing, unsigned char* values, unsigned char* rings,
                                           float4* halves) {
    using S = Shape<kHalves, kGroups, kColumnTiles>;
    static_assert(kHalves == 1 || kColumnTiles == 1, "halves meet in one tile of columns");
    constexpr int kTiles = S::kTiles, kRoundSteps = S::kRoundSteps, kRoundK = S::kRoundK, kValuePitch = S::kValuePitch;
    constexpr int kParts = Work::kParts, kPieces = S::kPieces / kParts;
    const int lane = threadIdx.x & 31, group = threadIdx.x / S::kGroupThreads;
    const int thread = threadIdx.x % S::kGroupThreads;
    const int tile = (thread >> 5) % kTiles, half = (thread >> 5) / kTiles;
    unsigned char* ring = rings + (threadIdx.x >> 5) * kStages * Stage<kFormat>::kBytes;
    values += group * 2 * S::kValueBytes;
    auto sync = [&] {
        if constexpr (kGroups == 1) {
            __syncthreads();
        } else {
            asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(S::kGroupThreads) : "memory");
        }
    };
    const unsigned ring_at = smem_u32(ring);
    const int steps = m.rounds * kRoundSteps;

    // three walks over the same passes: the copies run ahead of the values, the values ahead of the multiplies
    Pass at;
    bool more = work.begin(at);
    if (!more) return;
    Pass ahead = at;
    bool ahead_more = true;
    int ahead_step = 0, ahead_slot = 0;
    RowStream<kFormat> rows;
    rows.last_piece = static_cast<int>(m.pitch) - 16;
    rows.last_tile = m.k_tiles - 1;
    work.aim(rows, ahead, tile);
    auto copy_next = [&] {
        const int s = (ahead_step / kRoundSteps) * (kRoundSteps * kHalves) + half * kRoundSteps + ahead_step % kRoundSteps;
        rows.issue(s, ring_at + static_cast<unsigned>(ahead_slot * Stage<kFormat>::kBytes), ahead_more && s < m.stages);
        if (++ahead_slot == kStages) ahead_slot = 0;
        if (++ahead_step == steps) {
            ahead_step = 0;
            if (ahead_more) ahead_more = work.next(ahead);
            if (ahead_more && ahead.first == 0) work.aim(rows, ahead, tile);
        }
    };
    auto copies_end = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    // One copy of the code for each of these: unrolled, the loop outgrows the instruction cache (a third of all stalls).
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) {
        copy_next();
        copies_end();
    }

    Pass value_pass = at;
    bool value_more = true;
    int value_round = 0;
    typename Work::Piece pieces[kPieces];
    auto slots_of = [&](const Pass& pass) { return min(Work::kSlots, routing.start[pass.active + 1] - routing.start[pass.active] - pass.first); };
    auto load_values = [&] {
        if (!value_more) return;
        const int here = slots_of(value_pass);
        const int first = routing.start[value_pass.active] + value_pass.first;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int piece = i * S::kGroupThreads + thread;
            const int n = piece / (kRoundK / 8);
            if (n < here) work.load(pieces[i], first + n, value_round * kRoundK + piece % (kRoundK / 8) * 8);
        }
    };
    auto store_values = [&](unsigned char* to) {
        if (!value_more) return;
        const int here = slots_of(value_pass);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int piece = i * S::kGroupThreads + thread;
            const int n = piece / (kRoundK / 8);
            unsigned char* slot = to + n * kParts * kValuePitch + value_piece<kFormat>(piece % (kRoundK / 8) * 8) * 16;
            if (n >= here) continue;
            uint4 columns[kParts];
            work.finish(pieces[i], columns);
#pragma unroll
            for (int c = 0; c < kParts; ++c) *reinterpret_cast<uint4*>(slot + c * kValuePitch) = columns[c];
        }
        if (++value_round == m.rounds) {
            value_round = 0;
            value_more = work.next(value_pass);
        }
    };
    int buffer = 1, slot = 0, round = -1;  // round -1: the first values only
    float sums[kColumnTiles][2][4] = {};   // two chains
    while (more) {
        const typename Work::Side side = work.look(at, slots_of(at));
#pragma unroll 1
        for (; round < m.rounds; ++round) {
            sync();  // this round's values are there, nobody reads the other buffer any more
            load_values();
            if (round >= 0) {
#pragma unroll 1
                for (int j = 0; j < kRoundSteps; ++j) {
                    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
                    __syncwarp();
                    copy_next();  // into the slot of the step before, which all lanes have left
                    const int s = round * (kRoundSteps * kHalves) + half * kRoundSteps + j;
                    if (s < m.stages) {
                        multiply_step<kFormat, kValuePitch, kColumnTiles>(ring + slot * Stage<kFormat>::kBytes,
                                                            values + buffer * S::kValueBytes + (half * kRoundSteps + j) * (kStageK * 2), sums);
                    }
                    copies_end();
                    if (++slot == kStages) slot = 0;
                }
            }
            buffer ^= 1;
            store_values(values + buffer * S::kValueBytes);
        }
        round = 0;
        float acc[kColumnTiles][4];
#pragma unroll
        for (int n = 0; n < kColumnTiles; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = sums[n][0][i] + sums[n][1][i], sums[n][0][i] = sums[n][1][i] = 0.0f;
        }
        if constexpr (kHalves == 2) {
            if (half == 1) halves[tile * 32 + lane] = make_float4(acc[0][0], acc[0][1], acc[0][2], acc[0][3]);
            sync();
            if (half == 0) {
                const float4 other = halves[tile * 32 + lane];
                acc[0][0] += other.x, acc[0][1] += other.y, acc[0][2] += other.z, acc[0][3] += other.w;
            }
        }
        if (half == 0) work.done(at, slots_of(at), tile, side, acc);
        more = work.next(at);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// -------------------------------------------------------------------------------------------------------- up and down

// v / (1 + exp(-v)) * up. With e = exp(-|v| / 2) that is v / (1 + e^2) * up, and for negative v times e^2, which is taken in two
// halves: nothing on the way leaves f32's range unless the result does, however large `up` is.
__device__ __forceinline__ float silu_times(float v, float up) {
    const float e = expf(-0.5f * fabsf(v));
    const float part = v < 0.0f ? e : 1.0f;
    return __fdividef(v * part, fmaf(e, e, 1.0f)) * (up * part);  // a divisor of 1 to 2
}

template <int kHalves>
struct UpWork {
    using S = Shape<kHalves, 1>;
    using Piece = uint4;
    static constexpr int kParts = 1, kSlots = kTokenTile;
    const MoeParams& p;
    const Routing& routing;
    static constexpr int kGroupsOf128 = 16 / S::kTiles;  // groups of rows of G (and of U) in 128
    int groups;                                          // of rows of an expert
    int skip_active, skip_groups;  // gridDim.x items further on

    __device__ __forceinline__ UpWork(const MoeParams& params, const Routing& r) : p(params), routing(r), groups(params.f_groups / S::kTiles) {
        skip_active = gridDim.x / groups;
        skip_groups = gridDim.x - skip_active * groups;
    }
    __device__ __forceinline__ bool begin(Pass& pass) const {
        pass.active = blockIdx.x / groups;
        pass.group = blockIdx.x - pass.active * groups;
        pass.first = 0;
        return pass.active < routing.num_active;
    }
    __device__ __forceinline__ bool next(Pass& pass) const {
        pass.first += kSlots;
        if (pass.first < routing.start[pass.active + 1] - routing.start[pass.active]) return true;
        pass.first = 0;
        pass.active += skip_active;
        pass.group += skip_groups;
        if (pass.group >= groups) pass.group -= groups, ++pass.active;
        return pass.active < routing.num_active;
    }
    // Rows that share 32 bytes of scales: two neighbours in each of the four groups of 32 of a 128-row tile.
    __device__ __forceinline__ int row_in_f(const Pass& pass, int tile, int g) const {
        return pass.group / kGroupsOf128 * 128 + 32 * (g >> 1) + 2 * S::kTiles * (pass.group % kGroupsOf128) + 2 * tile + (g & 1);
    }
    // Rows 0 .. 7 of a tile are G's, 8 .. 15 the same of U.
    template <typename Rows>
    __device__ __forceinline__ void aim(Rows& rows, const Pass& pass, int tile) const {
        const int lane = threadIdx.x & 31;
        const int expert = routing.active[pass.active];
        const int r = min(row_in_f(pass, tile, lane >> 3), p.f - 1);
        rows.codes = p.gate_up.codes + expert * p.gate_up.matrix_codes + r * p.gate_up.pitch;
        rows.offset[0] = r + 64 < p.f ? 64 * p.gate_up.pitch : 0;
        rows.offset[1] = p.f * p.gate_up.pitch;
        rows.offset[2] = rows.offset[0] + rows.offset[1];
        const int q = min(row_in_f(pass, tile, lane & 7), p.f - 1) + (lane & 8 ? p.f : 0);
        rows.scales = p.gate_up.scales + expert * p.gate_up.matrix_scales + fp4_scale_offset(q, 0, p.gate_up.k_tiles);
    }
    __device__ __forceinline__ void load(Piece& piece, int n, int k) const {
        piece = make_uint4(0, 0, 0, 0);
        if (k < p.d_pitch) piece = *reinterpret_cast<const uint4*>(p.x16 + routing.tokens[n] * static_cast<long long>(p.d_pitch) + k);
    }
    __device__ __forceinline__ void finish(const Piece& piece, uint4 (&columns)[1]) const { columns[0] = piece; }
    struct Side {
        float back[2];  // undoes x's shift, times the expert's tensor scale
        int slot[2];
    };
    __device__ __forceinline__ Side look(const Pass& pass, int here) const {
        Side side;
        const int first = routing.start[pass.active] + pass.first;
        const float scale = p.gate_up.tensor_scale != nullptr ? p.gate_up.tensor_scale[routing.active[pass.active]] : 1.0f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = min(static_cast<int>(threadIdx.x & 3) * 2 + j, here - 1);
            side.slot[j] = routing.slots[first + n];
            side.back[j] = inverse_power(p.x_shift[routing.tokens[first + n]]) * scale;
        }
        return side;
    }
    __device__ __forceinline__ void done(const Pass& pass, int here, int tile, const Side& side, const float (&acc)[1][4]) const {
        const int lane = threadIdx.x & 31;
        const int g = lane >> 2, t = lane & 3;
        const int r = row_in_f(pass, tile, g);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = 2 * t + j;
            const int slot = side.slot[j];
            float h = 0.0f;
            if (n < here && r < p.f) {
                const float gate = acc[0][j] * side.back[j], up = acc[0][2 + j] * side.back[j];
                h = silu_times(gate, up);
            }
            int e = static_cast<int>((__float_as_uint(h) >> 23) & 0xffu);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) e = max(e, __shfl_xor_sync(0xffffffffu, e, o));
            if (n < here) {
                if (r < p.f_pitch) reinterpret_cast<float*>(p.h)[static_cast<long long>(slot) * p.f_pitch + r] = h;
                if (g == 0) atomicMax(p.h_max + slot, e);
            }
        }
    }
};

template <int kFormat>
constexpr int ring_bytes(int stages) { return kWarps * stages * Stage<kFormat>::kBytes; }
template <int kFormat, int kHalves>
constexpr int kUpSmem = 2 * Shape<kHalves, 1>::kValueBytes + ring_bytes<kFormat>(kUpStages);
// The down projection in one of four forms. One group: the halves of a round, all warps on one expert after the other, h as
// mc_moe_up left it. Two groups on experts of their own, h levelled before by mc_moe_level. Four, of two warps and 32 rows
// of y, for few rows of y, which leave SMs without work otherwise (the layer, 4 tokens, 8 of 64 experts of 1024 x 1024: 36
// us against 39 in two groups; 40 tokens, 8 of 160 of 1024 x 512: 71 against 78; 16 tokens, 8 of 64 of 512 x 512: 31 against
// 32). And two groups with two tiles of columns, eight slots, in one pass: the codes are decoded once for both, in rounds
// half as long (64 tokens, 8 of 64 experts of 2048 x 768: 139 us against 160; 8 of 128: 143 against 156; 32 tokens, two slots
// per expert: 109 both ways; 64 tokens, 8 of 64 experts of 1024 x 1024: 109, 139 in four groups of one tile). Two CTAs have
// to fit on an SM: with room for one, 32 tokens, 8 of 128 experts of 1024 x 512 took 81 us instead of 59.
template <int kGroups, int kColumnTiles>
struct DownShape : Shape<kGroups == 1 ? 2 : 1, kGroups, kColumnTiles> {
    static constexpr int kRows = DownShape::kTiles * 16;
    static constexpr int kRowGroups = 128 / kRows;  // in 128 rows of y
    static constexpr int kPitch = kRows + 4;
};
template <int kFormat, int kGroups, int kColumnTiles, int kStages>
constexpr int down_smem(int tokens) {
    using S = DownShape<kGroups, kColumnTiles>;
    return kGroups * (tokens * S::kPitch * 4 + 2 * S::kValueBytes) + ring_bytes<kFormat>(kStages);
}

template <int kFormat, int kHalves>
__global__ void __launch_bounds__(kThreads, 2) mc_moe_up(const MoeParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Routing routing;
    __shared__ float4 halves[kWarps / 2 * 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    load_routing(routing, reinterpret_cast<int*>(smem), p);
    UpWork<kHalves> work(p, routing);
    run_passes<kFormat, kHalves, 1, 1, kUpStages>(work, p.gate_up, routing, smem, smem + 2 * Shape<kHalves, 1>::kValueBytes, halves);
}

// Eight values of h after the power of two of their slot's largest: hi, the nearest f16, and lo, 2^11 times what hi leaves, at
// most 2^14. An infinite hi (beside a value that is infinite or NaN nothing is shifted) leaves nothing.
__device__ __forceinline__ void split(const uint4& first, const uint4& second, int largest, uint4 (&columns)[2]) {
    const unsigned w[8] = {first.x, first.y, first.z, first.w, second.x, second.y, second.z, second.w};
    const float to = power(shift_of(largest));
    unsigned hi[4], lo[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = __uint_as_float(w[2 * j]) * to, b = __uint_as_float(w[2 * j + 1]) * to;
        hi[j] = pack_f16(a, b);
        const float ha = f16_lo(hi[j]), hb = f16_hi(hi[j]);
        lo[j] = pack_f16(fabsf(ha) <= 65504.0f ? (a - ha) * 2048.0f : 0.0f, fabsf(hb) <= 65504.0f ? (b - hb) * 2048.0f : 0.0f);
    }
    columns[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    columns[1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// All of h, in place.
__global__ void __launch_bounds__(128) mc_moe_level(const MoeParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int slot = blockIdx.x;
    const int largest = p.h_max[slot], eights = p.f_pitch / 8;
    for (int i = threadIdx.x; i < eights; i += 128) {
        uint4* at = p.h + 2 * (static_cast<long long>(slot) * eights + i);
        uint4 columns[2];
        split(at[0], at[1], largest, columns);
        at[0] = columns[0];
        at[1] = columns[1];
    }
}

// One group: h lies as mc_moe_up left it, in f32; several: as mc_moe_level did, as the two f16 numbers.
template <int kGroups, int kColumnTiles>
struct DownWork {
    using S = DownShape<kGroups, kColumnTiles>;
    static constexpr bool kLevel = kGroups > 1;
    static constexpr int kParts = 2, kSlots = S::kColumns / 2;
    struct Piece {
        uint4 raw[2];
        int largest;
    };
    const MoeParams& p;
    const Routing& routing;
    float* sums;  // [tokens][kPitch]
    int group;    // of rows of y: their share of each group of 32 of a 128-row tile
    int first, step;

    __device__ __forceinline__ bool begin(Pass& pass) const {
        pass.active = first;
        pass.group = 0;
        pass.first = 0;
        return pass.active < routing.num_active;
    }
    __device__ __forceinline__ bool next(Pass& pass) const {
        pass.first += kSlots;
        if (pass.first < routing.start[pass.active + 1] - routing.start[pass.active]) return true;
        pass.first = 0;
        pass.active += step;
        return pass.active < routing.num_active;
    }
    // Row i of a tile: four neighbours in each group of 32, so that a warp uses 64 of 128 bytes of scales, the tile beside it the rest.
    __device__ __forceinline__ int row_in_y(int tile, int i) const {
        return group / S::kRowGroups * 128 + 32 * (i >> 2) + 4 * S::kTiles * (group % S::kRowGroups) + 4 * tile + (i & 3);
    }
    template <typename Rows>
    __device__ __forceinline__ void aim(Rows& rows, const Pass& pass, int tile) const {
        const int lane = threadIdx.x & 31;
        const int expert = routing.active[pass.active];
        const int r = min(row_in_y(tile, lane >> 3), p.d - 1);
        rows.codes = p.down.codes + expert * p.down.matrix_codes + r * p.down.pitch;
#pragma unroll
        for (int i = 0; i < 3; ++i) rows.offset[i] = r + 32 * (i + 1) < p.d ? 32 * (i + 1) * p.down.pitch : 0;
        rows.scales = p.down.scales + expert * p.down.matrix_scales + fp4_scale_offset(min(row_in_y(tile, lane & 15), p.d - 1), 0, p.down.k_tiles);
    }
    __device__ __forceinline__ void load(Piece& piece, int n, int k) const {
        const int slot = routing.slots[n];
        piece.raw[0] = piece.raw[1] = make_uint4(0, 0, 0, 0);
        if (!kLevel) piece.largest = p.h_max[slot];
        if (k < p.f_pitch) {
            const uint4* at = p.h + 2 * (static_cast<long long>(slot) * (p.f_pitch / 8) + k / 8);
            piece.raw[0] = at[0];
            piece.raw[1] = at[1];
        }
    }
    __device__ __forceinline__ void finish(const Piece& piece, uint4 (&columns)[2]) const {
        if (kLevel) {
            columns[0] = piece.raw[0];
            columns[1] = piece.raw[1];
        } else {
            split(piece.raw[0], piece.raw[1], piece.largest, columns);
        }
    }
    struct Side {
        TwoFactors weight[kColumnTiles];  // the expert's for the token, times its tensor scale, and undoes h's shift
        int token[kColumnTiles];
    };
    // A lane's two columns of a tile are the two of one slot.
    __device__ __forceinline__ Side look(const Pass& pass, int here) const {
        const float scale = p.down.tensor_scale != nullptr ? p.down.tensor_scale[routing.active[pass.active]] : 1.0f;
        const int first_slot = routing.start[pass.active] + pass.first;
        Side side;
#pragma unroll
        for (int n = 0; n < kColumnTiles; ++n) {
            const int at = first_slot + min(n * 4 + static_cast<int>(threadIdx.x & 3), here - 1);
            const int slot = routing.slots[at];
            const float back = power(-shift_of(p.h_max[slot]));
            side.weight[n] = scale < back ? two_factors(scale, back) : two_factors(back, scale);
            side.weight[n].second *= p.weights[slot];  // the larger one, where there are two
            side.token[n] = routing.tokens[at];
        }
        return side;
    }
    __device__ __forceinline__ void done(const Pass& pass, int here, int tile, const Side& side, const float (&acc)[kColumnTiles][4]) const {
        const int lane = threadIdx.x & 31;
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < kColumnTiles; ++n) {
            if (n * 4 + t < here) {
                // this warp's 16 columns; nobody else adds to them
                float* sum = sums + side.token[n] * S::kPitch + tile * 16;
                sum[g] += side.weight[n].times(fmaf(acc[n][1], 0x1p-11f, acc[n][0]));
                sum[g + 8] += side.weight[n].times(fmaf(acc[n][3], 0x1p-11f, acc[n][2]));
            }
        }
    }
};

template <int kFormat, int groups, int kColumnTiles, int kStages>
__global__ void __launch_bounds__(kThreads, 2) mc_moe_down(const MoeParams p, int cluster) {
    using S = DownShape<groups, kColumnTiles>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ Routing routing;
    __shared__ float4 halves[groups == 1 ? kWarps / 2 * 32 : 1];
    unsigned char* values = smem;
    unsigned char* rings = values + groups * 2 * S::kValueBytes;
    float* sums = reinterpret_cast<float*>(rings + ring_bytes<kFormat>(kStages));  // [groups][tokens][kPitch]
    const int group_sums = p.tokens * S::kPitch;
    const int rank = cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int rows = blockIdx.x / cluster;  // which 64 or 32
    const int mine = threadIdx.x / S::kGroupThreads;
    for (int i = threadIdx.x; i < groups * group_sums; i += kThreads) sums[i] = 0.0f;
    load_routing(routing, reinterpret_cast<int*>(values), p);
    DownWork<groups, kColumnTiles> work{p, routing, sums + mine * group_sums, rows, rank * groups + mine, cluster * groups};
    run_passes<kFormat, groups == 1 ? 2 : 1, groups, kColumnTiles, kStages>(work, p.down, routing, values, rings, halves);
    __syncthreads();
    if (cluster > 1) cluster_sync_all();
    // Every CTA of the cluster finishes its share of the elements: the partial sums in the order of ranks and groups.
    const unsigned sums_at = smem_u32(sums);
    const int count = p.tokens * S::kRows;
    for (int i = rank * kThreads + static_cast<int>(threadIdx.x); i < count; i += cluster * kThreads) {
        const int token = i / S::kRows, c = i - token * S::kRows;
        const unsigned at = sums_at + static_cast<unsigned>(token * S::kPitch + c) * 4u;
        float v = 0.0f;
        for (int z = 0; z < cluster; ++z) {
#pragma unroll
            for (int g = 0; g < groups; ++g) {
                float part;
                if (cluster > 1) {
                    asm volatile("ld.shared::cluster.f32 %0, [%1];"
                                 : "=f"(part)
                                 : "r"(peer_address(at + static_cast<unsigned>(g * group_sums * 4), static_cast<unsigned>(z)))
                                 : "memory");
                } else {
                    part = sums[g * group_sums + token * S::kPitch + c];
                }
                v += part;
            }
        }
        const int r = work.row_in_y(c >> 4, c & 15);
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

template <int kFormat, int kHalves>
int launch_up(MoeParams p, int reached, cudaStream_t s) {
    using S = Shape<kHalves, 1>;
    static SharedMemoryOnce once;
    if (int rc = once.allow(mc_moe_up<kFormat, kHalves>, kUpSmem<kFormat, kHalves>)) return rc;
    p.gate_up.rounds = (p.d + S::kRoundK - 1) / S::kRoundK;
    const long long items = static_cast<long long>(reached) * (p.f_groups / S::kTiles);
    const auto grid = static_cast<unsigned>(std::min<long long>(items, 2LL * sm_count()));
    return launch(mc_moe_up<kFormat, kHalves>, grid, 1, kThreads, kUpSmem<kFormat, kHalves>, s, "mc_moe_up", p);
}

template <int kFormat, int kGroups, int kColumnTiles, int kStages>
int launch_down(MoeParams p, int reached, cudaStream_t s) {
    using S = DownShape<kGroups, kColumnTiles>;
    static_assert(down_smem<kFormat, kGroups, kColumnTiles, kStages>(MCD_MOE_MAX_TOKENS) + 10 * 1024 <= 227 * 1024, "shared memory");
    static SharedMemoryOnce once;
    if (int rc = once.allow(mc_moe_down<kFormat, kGroups, kColumnTiles, kStages>, down_smem<kFormat, kGroups, kColumnTiles, kStages>(MCD_MOE_MAX_TOKENS))) return rc;
    p.down.rounds = (p.f + S::kRoundK - 1) / S::kRoundK;
    int cluster = 8;
    while (cluster > reached) cluster /= 2;
    const auto grid = static_cast<unsigned>((p.d + 127) / 128 * S::kRowGroups * cluster);
    return launch(mc_moe_down<kFormat, kGroups, kColumnTiles, kStages>, grid, static_cast<unsigned>(cluster), kThreads, down_smem<kFormat, kGroups, kColumnTiles, kStages>(p.tokens), s,
                  "mc_moe_down", p, cluster);
}

// Whether two CTAs of the down projection have room on an SM (228 KB, of which a CTA takes one for itself).
template <int kFormat, int kGroups, int kColumnTiles, int kStages>
bool two_fit(int tokens) {
    constexpr int kStatic = sizeof(Routing) + (kGroups == 1 ? kWarps / 2 * 32 : 1) * sizeof(float4) + 128;
    return down_smem<kFormat, kGroups, kColumnTiles, kStages>(tokens) + kStatic + 1024 <= 114 * 1024;
}

// Rings as deep as the sums beside them allow.
template <int kFormat, int kGroups, int kColumnTiles>
int launch_levelled(const MoeParams& p, int reached, cudaStream_t s) {
    return two_fit<kFormat, kGroups, kColumnTiles, 3>(p.tokens) ? launch_down<kFormat, kGroups, kColumnTiles, 3>(p, reached, s)
                                                                 : launch_down<kFormat, kGroups, kColumnTiles, 2>(p, reached, s);
}

template <int kFormat>
int launch_layer(const MoeParams& p, cudaStream_t s) {
    // The router's clusters are declared with the kernel.
    if (int rc = launch(mc_moe_router, static_cast<unsigned>(p.tokens * kRouterCluster), 1, kRouterThreads, 0, s, "mc_moe_router", p)) return rc;
    const int reached = std::min(p.experts, p.tokens * p.top_k);
    const bool many = static_cast<long long>(reached) * (p.f_groups / Shape<2, 1>::kTiles) > 4LL * sm_count();
    if (int rc = many ? launch_up<kFormat, 1>(p, reached, s) : launch_up<kFormat, 2>(p, reached, s)) return rc;
    // Four groups per CTA where their clusters find SMs all at once, two CTAs on each, and there are experts for the groups.
    const bool spread = p.d <= 1024 && reached >= 24 && two_fit<kFormat, 4, 1, 2>(p.tokens);
    // A launch of its own for h pays where many CTAs would each level the same rows of it: 32 row groups for every 2048 of d.
    if (p.tokens * p.top_k <= 32 && !spread) return launch_down<kFormat, 1, 1, 3>(p, reached, s);
    if (int rc = launch(mc_moe_level, static_cast<unsigned>(p.tokens * p.top_k), 1, 128, 0, s, "mc_moe_level", p)) return rc;
    // Two tiles of columns where most experts have more slots than the four of one.
    const bool crowded = p.tokens * p.top_k > 3 * reached;
    if (crowded) return launch_levelled<kFormat, 2, 2>(p, reached, s);
    return spread ? launch_levelled<kFormat, 4, 1>(p, reached, s) : launch_levelled<kFormat, 2, 1>(p, reached, s);
}

constexpr long long kMaxWidth = 1 << 24;  // d and f

size_t rounded(size_t bytes) { return (bytes + 15) / 16 * 16; }

size_t in_eights(long long n) { return static_cast<size_t>((n + 7) / 8 * 8); }
size_t f_groups(long long f) { return static_cast<size_t>((f + 127) / 128 * 16); }

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
    m.rounds = 0;
    return m;
}

}  // namespace

extern "C" size_t mcd_moe_workspace(int tokens, int experts, int top_k, long long d, long long f) {
    if (tokens < 1 || tokens > MCD_MOE_MAX_TOKENS || experts < 1 || experts > MCD_MOE_MAX_EXPERTS || top_k < 1 || top_k > MCD_MOE_MAX_TOP_K ||
        top_k > experts || d < 1 || d > kMaxWidth || f < 1 || f > kMaxWidth) {
        return 0;
    }
    const size_t slots = static_cast<size_t>(tokens) * static_cast<size_t>(top_k);
    return 3 * rounded(slots * 4) + rounded(static_cast<size_t>(tokens) * 4) + slots * in_eights(f) * 4 +
           rounded(static_cast<size_t>(tokens) * in_eights(d) * 2);
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
    if (gu.cols > kMaxWidth || dn.cols > kMaxWidth) return fail("mcd_moe_layer: d and f are at most 2^24");
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
    p.d_pitch = static_cast<int>(in_eights(d));
    p.f_pitch = static_cast<int>(in_eights(f));
    p.f_groups = static_cast<int>(f_groups(f));
    p.router_vec = is_aligned(args->x, 16) && args->ldx % 8 == 0 && is_aligned(args->router, 16) && args->ld_router % 8 == 0;
    p.gate_up = matrix_of(gu);
    p.down = matrix_of(dn);
    p.chosen_out = args->chosen;
    p.weights_out = args->weights;
    const size_t slots = static_cast<size_t>(args->tokens) * static_cast<size_t>(args->top_k);
    auto* at = static_cast<unsigned char*>(args->workspace);
    p.chosen = reinterpret_cast<int*>(at);
    p.weights = reinterpret_cast<float*>(at += rounded(slots * 4));
    p.h_max = reinterpret_cast<int*>(at += rounded(slots * 4));
    p.x_shift = reinterpret_cast<float*>(at += rounded(slots * 4));
    p.h = reinterpret_cast<uint4*>(at += rounded(static_cast<size_t>(args->tokens) * 4));
    p.x16 = reinterpret_cast<unsigned short*>(at += slots * in_eights(f) * 4);
    auto s = static_cast<cudaStream_t>(stream);
    return gu.format == MCD_FP4_E8M0_32 ? launch_layer<MCD_FP4_E8M0_32>(p, s) : launch_layer<MCD_FP4_E4M3_16>(p, s);
}
