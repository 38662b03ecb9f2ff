// Routing to experts: s = softmax or sigmoid of a token's scores, b = s + bias; of the groups those with the largest
// sums of their two largest b; of their experts the `count` with the largest b, ties to the lowest index; weights s,
// divided by their sum if asked for, times a scale.
//
// s, b and the sums are FP64: which expert is chosen hangs on differences of b, and FP32 would decide some of them by
// its rounding.
#include "token_elements.cuh"

#include <cmath>

namespace nvcr_sm100::token {
namespace {

constexpr int route_warps = 4;

// The order of doubles that are no NaN as that of unsigned integers. -0 comes as +0 (the caller adds 0).
__device__ __forceinline__ unsigned long long ordered(double v) {
    const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(v));
    return bits >> 63 ? ~bits : bits | 1ull << 63;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) v += __shfl_xor_sync(0xffffffffu, v, offset);
    return v;
}

// The largest key of a warp and the lowest index that has it; -1 where all keys are 0.
struct Best {
    unsigned long long key;
    int index;
};
__device__ __forceinline__ Best warp_best(unsigned long long key, int index) {
    const unsigned high = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(key >> 32));
    const unsigned low = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(key >> 32) == high ? static_cast<unsigned>(key) : 0u);
    const unsigned long long best = static_cast<unsigned long long>(high) << 32 | low;
    const unsigned at = __reduce_min_sync(0xffffffffu, key == best ? static_cast<unsigned>(index) : 0x7fffffffu);
    return {best, best == 0 ? -1 : static_cast<int>(at)};
}

// A warp a token; lane l has experts l, l + 32, ... Key 0 stands for an expert that is left out.
template <typename T, int Each>
__global__ void __launch_bounds__(route_warps * 32) route_kernel(RouteArgs a) {
    extern __shared__ unsigned long long keys_of[];
    join_chain();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const std::int64_t token = blockIdx.x * static_cast<std::int64_t>(route_warps) + warp;
    if (token >= a.tokens) return;
    const T* row = static_cast<const T*>(a.scores) + token * a.stride;
    float score[Each];
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < Each; ++i) {
        const int e = i * 32 + lane;
        score[i] = e < a.experts ? widen(row[e]) : -INFINITY;
        if (!(score[i] > -INFINITY)) score[i] = -INFINITY;  // a NaN is left out
        most = fmaxf(most, score[i]);
    }
    double share[Each];
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            share[i] = score[i] > -INFINITY ? 1.0 / (1.0 + exp(-static_cast<double>(score[i]))) : 0.0;
        }
    } else {
#pragma unroll
        for (int offset = 16; offset > 0; offset /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, offset));
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            // the largest have weight one, infinite ones too
            share[i] = score[i] == -INFINITY ? 0.0
                : score[i] == most           ? 1.0
                                             : exp(static_cast<double>(score[i]) - static_cast<double>(most));
            sum += share[i];
        }
        sum = warp_sum(sum);
#pragma unroll
        for (int i = 0; i < Each; ++i) share[i] = sum > 0.0 ? share[i] / sum : 0.0;
    }
    unsigned long long key[Each];
#pragma unroll
    for (int i = 0; i < Each; ++i) {
        const int e = i * 32 + lane;
        double b = share[i];
        if (a.bias != nullptr && e < a.experts) b += static_cast<double>(a.bias[e]);
        key[i] = score[i] > -INFINITY && b > -HUGE_VAL ? ordered(b + 0.0) : 0;
    }

    if (a.kept_groups < a.groups) {
        unsigned long long* keys = keys_of + warp * a.experts;
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            if (i * 32 + lane < a.experts) keys[i * 32 + lane] = key[i];
        }
        __syncwarp();
        const int size = a.experts / a.groups;
        auto value = [](unsigned long long k) {
            return __longlong_as_double(static_cast<long long>(k >> 63 ? k & ~(1ull << 63) : ~k));
        };
        // lane l has groups l, l + 32, ...; there are at most as many as experts
        unsigned long long group[Each];
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            const int g = i * 32 + lane;
            unsigned long long first = 0, second = 0;
            for (int j = 0; g < a.groups && j < size; ++j) {
                const unsigned long long k = keys[g * size + j];
                if (k > first) {
                    second = first, first = k;
                } else if (k > second) {
                    second = k;
                }
            }
            group[i] = first == 0 ? 0 : ordered(value(first) + (second == 0 ? 0.0 : value(second)) + 0.0);
        }
        unsigned long long kept[Each];  // of this lane's groups
#pragma unroll
        for (int i = 0; i < Each; ++i) kept[i] = 0;
        for (int n = 0; n < a.kept_groups; ++n) {
            unsigned long long best = 0;
            int at = 0;
#pragma unroll
            for (int i = 0; i < Each; ++i) {
                if (group[i] > best) best = group[i], at = i * 32 + lane;
            }
            const Best found = warp_best(best, at);
            if (found.index < 0) break;
#pragma unroll
            for (int i = 0; i < Each; ++i) {
                if (found.index == i * 32 + lane) group[i] = 0, kept[i] = 1;
            }
        }
        __syncwarp();
        // the keys of groups that are not kept become 0, in the shared copy and then here
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            const int g = i * 32 + lane;
            if (g < a.groups && kept[i] == 0) {
                for (int j = 0; j < size; ++j) keys[g * size + j] = 0;
            }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < Each; ++i) key[i] = i * 32 + lane < a.experts ? keys[i * 32 + lane] : 0;
    }

    // the lane n % 32 keeps the n-th choice and its share until their sum is known
    constexpr int most_kept = Each;  // count is at most the number of experts
    int chosen[most_kept];
    double weight[most_kept];
#pragma unroll
    for (int i = 0; i < most_kept; ++i) chosen[i] = -1, weight[i] = 0.0;
    double sum = 0.0;
    for (int n = 0; n < a.count; ++n) {
        unsigned long long best = 0;
        int at = 0;
        double mine = 0.0;
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            if (key[i] > best) best = key[i], at = i * 32 + lane, mine = share[i];
        }
        const Best found = warp_best(best, at);
        if (found.index < 0) break;
        mine = __shfl_sync(0xffffffffu, mine, found.index % 32);
        sum += mine;
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            if (found.index == i * 32 + lane) key[i] = 0;
            if (n == i * 32 + lane) chosen[i] = found.index, weight[i] = mine;
        }
    }
    const double factor = a.renormalise ? (sum > 0.0 ? 1.0 / sum : 0.0) : 1.0;
#pragma unroll
    for (int i = 0; i < most_kept; ++i) {
        const int n = i * 32 + lane;
        if (n >= a.count) continue;
        a.choices[token * a.count + n] = chosen[i];
        a.weights[token * a.count + n] = static_cast<float>(weight[i] * factor * static_cast<double>(a.scale));
    }
}

template <typename T, int Each>
cudaError_t launch(const RouteArgs& a, cudaStream_t stream) {
    const std::int64_t blocks = (a.tokens + route_warps - 1) / route_warps;
    const std::size_t shared = a.kept_groups < a.groups ? static_cast<std::size_t>(route_warps) * a.experts * 8 : 0;
    return kernels::launch_overlapped(route_kernel<T, Each>, dim3(static_cast<unsigned>(blocks)), dim3(route_warps * 32), shared,
                                      stream, a);
}

template <typename T>
cudaError_t by_experts(const RouteArgs& a, cudaStream_t stream) {
    if (a.experts <= 32) return launch<T, 1>(a, stream);
    if (a.experts <= 64) return launch<T, 2>(a, stream);
    if (a.experts <= 128) return launch<T, 4>(a, stream);
    if (a.experts <= 256) return launch<T, 8>(a, stream);
    if (a.experts <= 512) return launch<T, 16>(a, stream);
    return launch<T, 32>(a, stream);
}

}  // namespace

cudaError_t route(const RouteArgs& a, cudaStream_t stream) {
    if (a.tokens == 0) return cudaSuccess;
    switch (a.type) {
    case Type::f16: return by_experts<__half>(a, stream);
    case Type::bf16: return by_experts<__nv_bfloat16>(a, stream);
    default: return by_experts<float>(a, stream);
    }
}

}  // namespace nvcr_sm100::token
