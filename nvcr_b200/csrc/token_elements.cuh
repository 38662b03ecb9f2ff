#pragma once

// Element access and warp sums shared by the token kernels.

#include "launch.cuh"
#include "token_kernels.hpp"

#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace nvcr_sm100::token {

// The first thing every kernel does: a token model's step is a chain of short
// launches, so each starts while the one before it ends, and waits for it here,
// before it touches memory; then the next may start the same way.
__device__ __forceinline__ void join_chain() {
    kernels::grid_dependency_wait();
    kernels::launch_dependents();
}

__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(float v) { return v; }

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }

__device__ __forceinline__ float half_bits(std::uint16_t bits) { return __half2float(__ushort_as_half(bits)); }

// Minimum and maximum that pass a NaN on.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 2^x with results below the normal range flushed to zero: softmax weights.
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) v += __shfl_xor_sync(0xffffffffu, v, offset);
    return v;
}

// n / d for n < 2^31 as (umulhi(n, multiplier) + n) >> shift (Granlund and
// Montgomery's division by an invariant).
struct Divisor {
    unsigned multiplier, shift;
};

__device__ __forceinline__ unsigned divide(unsigned n, Divisor d) { return (__umulhi(n, d.multiplier) + n) >> d.shift; }

inline Divisor divisor(unsigned d) {
    Divisor made{0, 0};
    while ((1u << made.shift) < d) ++made.shift;
    made.multiplier = static_cast<unsigned>((((1ull << made.shift) - d) << 32) / d + 1);
    return made;
}

// A kernel's dynamic shared memory above 48 KB, allowed once on each device.
class SharedAllowance {
public:
    template <typename Kernel>
    cudaError_t allow(Kernel* kernel, int bytes) {
        int device = 0;
        cudaError_t status = cudaGetDevice(&device);
        if (status != cudaSuccess) return status;
        const unsigned long long bit = 1ull << (device & 63);
        if (device < 64 && (devices_.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
        status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (status == cudaSuccess) devices_.fetch_or(bit, std::memory_order_relaxed);
        return status;
    }

private:
    std::atomic<unsigned long long> devices_{0};
};

}  // namespace nvcr_sm100::token
