#pragma once
// What the host sides of fp4_quantize.cu, fp4_gemm.cu and moe_layer.cu share: checks of arguments, launch bookkeeping.

#include "minicompiler_b200_device.h"

#include "device/driver_api.hpp"
#include "kernels/fp4_format.cuh"

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <initializer_list>
#include <mutex>
#include <string>

namespace mcd {

extern std::atomic<unsigned long long> g_launches;

inline int launched(const char* what) {
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return check_rt(cudaGetLastError(), what);
}

inline int sm_count() {
    static std::atomic<int> cached[64];
    int device = 0;
    cudaGetDevice(&device);
    if (device >= 0 && device < 64 && cached[device].load(std::memory_order_relaxed) > 0) return cached[device].load(std::memory_order_relaxed);
    int sms = 0;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) {
        cudaGetLastError();
        return 148;
    }
    if (device >= 0 && device < 64) cached[device].store(sms, std::memory_order_relaxed);
    return sms;
}

// A kernel's opt-in to more than 48 KB of dynamic shared memory, once per device. Whoever comes while another thread is at
// it waits for that to be done.
class SharedMemoryOnce {
public:
    template <typename Kernel>
    int allow(Kernel kernel, int bytes) {
        int device = 0;
        if (int rc = check_rt(cudaGetDevice(&device), "cudaGetDevice")) return rc;
        std::lock_guard<std::mutex> lock(mutex_);
        const bool kept = device >= 0 && device < 64;
        if (kept && (done_ >> device & 1ull) != 0) return 0;
        if (int rc = check_rt(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                              "cudaFuncSetAttribute(max dynamic shared memory)")) {
            return rc;
        }
        if (kept) done_ |= 1ull << device;
        return 0;
    }

private:
    std::mutex mutex_;
    unsigned long long done_ = 0;
};

// a * b * c <= limit, for non-negative numbers
inline bool fits(long long a, long long b, long long c, long long limit) {
    return static_cast<__int128>(a) * b * c <= limit;
}

inline bool is_aligned(const void* p, std::uintptr_t to) { return (reinterpret_cast<std::uintptr_t>(p) & (to - 1)) == 0; }

inline std::string named(const char* who, const char* what) { return std::string(who) + ": " + what; }

// Shape, format and alignment of a 4-bit operand; looks at no memory.
inline int check_fp4(const char* who, const mcd_fp4_tensor* t) {
    if (t == nullptr) return fail(named(who, "null 4-bit matrix"));
    if (t->format != MCD_FP4_E8M0_32 && t->format != MCD_FP4_E4M3_16) return fail(named(who, "unknown 4-bit format"));
    if (t->batch < 1) return fail(named(who, "no matrices"));
    if (t->rows < 1 || t->cols < 1) return fail(named(who, "empty matrix"));
    if (t->rows > 2147483647LL - 255 || t->cols > (1LL << 30) || !fits(t->batch, t->rows, mcd_fp4_code_pitch(t->cols), 1LL << 46)) {
        return fail(named(who, "matrix too large"));
    }
    if (t->codes == nullptr || t->scales == nullptr) return fail(named(who, "null codes or scales"));
    if (!is_aligned(t->codes, 16) || !is_aligned(t->scales, 16)) return fail(named(who, "codes and scales need 16-byte alignment"));
    if (t->format == MCD_FP4_E8M0_32 && t->tensor_scale != nullptr) return fail(named(who, "e8m0_32 has no tensor scale"));
    if (!is_aligned(t->tensor_scale, 4)) return fail(named(who, "unaligned tensor scale"));
    return 0;
}

// Kernels run on the current device: every pointer has to be memory that this device addresses. Memory the driver does
// not know (pageable host memory) and memory of another device are refused instead of faulting in a kernel.
inline int check_device_pointers(const char* who, std::initializer_list<const void*> pointers) {
    const DriverApi* drv = driver_api();
    if (drv == nullptr) return fail(named(who, "the CUDA driver API is unavailable"));
    int current = 0;
    if (int rc = check_rt(cudaGetDevice(&current), "cudaGetDevice")) return rc;
    for (const void* p : pointers) {
        if (p == nullptr) continue;
        int device = current;
        const CUresult rc = drv->PointerGetAttribute(&device, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, reinterpret_cast<CUdeviceptr>(p));
        if (rc == CUDA_ERROR_INVALID_VALUE) return fail(named(who, "an operand is not device memory"));
        if (rc == CUDA_SUCCESS && device != current) {
            return fail(named(who, "an operand is on device ") + std::to_string(device) + ", the current device is " + std::to_string(current));
        }
    }
    return 0;
}

}  // namespace mcd
