// Routing to experts: s = softmax or sigmoid of a token's scores, b = s + bias; of the groups those with the largest
// sums of their two largest b; of their experts the `count` with the largest b, ties to the lowest index; weights s,
// divided by their sum if asked for, times a scale.
//
// s, b and the sums are FP64 by definition: which expert is chosen hangs on differences of b, and FP32 would decide some of
// them by its rounding. But FP32 says of most tokens that no difference is that small: `route_kernel` chooses in FP32, and
// takes a token whose choices differ by less than that arithmetic's error again in FP64 (`exactly`), unless scores and
// biases are equal. The weights are FP64 in either. 16384 tokens by 8 of 256 experts in groups: 30.9 us, 90 with all
// tokens in FP64; 1130 warp instructions a token keep the schedulers busy for 68% of that, where the scores'
// bytes take 2.7. More than 256 experts, 31 choices or 32 groups go in FP64 throughout: 16384 tokens by 8 of 512 in 118 us, by
// 32 of 256, or by 8 of 256 in 64 groups, in 148.
#include "token_elements.cuh"

#include <climits>
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

// A token by a warp in FP64; lane l has experts l, l + 32, ... Key 0 stands for an expert that is left out. `keys`: room
// for as many as there are experts.
template <typename T, int Each>
__device__ __noinline__ void exactly(const RouteArgs& a, std::int64_t token, unsigned long long* keys) {
    const int lane = threadIdx.x % 32;
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
__global__ void __launch_bounds__(route_warps * 32) exact_kernel(RouteArgs a) {
    extern __shared__ unsigned long long keys_of[];
    join_chain();
    const int warp = threadIdx.x / 32;
    const std::int64_t token = blockIdx.x * static_cast<std::int64_t>(route_warps) + warp;
    if (token < a.tokens) exactly<T, Each>(a, token, keys_of + warp * a.experts);
}

// The order of floats that are no NaN, as that of unsigned integers; 0 for -infinity. -0 lies below +0: it comes as neither a
// share nor a sum of one.
constexpr unsigned least_key = 0x007fffffu;
__device__ __forceinline__ unsigned ordered(float v) {
    const int bits = __float_as_int(v);
    return static_cast<unsigned>(bits ^ (bits >> 31 | INT_MIN)) - least_key;
}
__device__ __forceinline__ float value_of(unsigned key) {
    const unsigned bits = key + least_key;
    return __uint_as_float(bits >> 31 ? bits & 0x7fffffffu : ~bits);
}

__device__ __forceinline__ float reciprocal(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Shared memory of a warp, in words of 8 bytes: 32 candidates with three values each, or a key an expert.
__host__ __device__ __forceinline__ int room_of(const RouteArgs& a) { return a.experts > 96 ? (a.experts + 1) / 2 * 2 : 96; }

// Up to 256 experts, of which up to 31 are chosen.
template <typename T, int Each>
__global__ void __launch_bounds__(route_warps * 32, 8) route_kernel(RouteArgs a) {
    extern __shared__ __align__(16) unsigned long long keys_of[];
    join_chain();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const std::int64_t token = blockIdx.x * static_cast<std::int64_t>(route_warps) + warp;
    if (token >= a.tokens) return;
    const T* row = static_cast<const T*>(a.scores) + token * a.stride;
    float score[Each], bias[Each];
#pragma unroll
    for (int i = 0; i < Each; ++i) {
        const int e = i * 32 + lane;
        score[i] = e < a.experts ? widen(row[e]) : -INFINITY;
        bias[i] = a.bias != nullptr && e < a.experts ? a.bias[e] : 0.0f;
    }
    constexpr float log2e = 1.44269504f;
    float most = -INFINITY, largest_share = 1.0f;
    float share[Each];
    bool certain = true;
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < Each; ++i) share[i] = reciprocal(1.0f + exp2_fast(score[i] * -log2e));
    } else {
#pragma unroll
        for (int i = 0; i < Each; ++i) most = fmaxf(most, score[i]);
#pragma unroll
        for (int offset = 16; offset > 0; offset /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, offset));
        certain = most < INFINITY;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            share[i] = score[i] > -INFINITY ? exp2_fast((score[i] - most) * log2e) : 0.0f;
            sum += share[i];
        }
        largest_share = reciprocal(token::warp_sum(sum));
#pragma unroll
        for (int i = 0; i < Each; ++i) share[i] *= largest_share;
    }
    // How far a share s and its sum b with the bias may be off: of exponents up to 128, rounded twice or three times to 2^-24
    // of themselves, a factor of 1e-5 or 1.6e-5, which a sigmoid has times 1 - s; ex2, rcp and sums 4e-7, a softmax's sum
    // 2e-6; b 2^-24 of itself, and as much again with its error added; and what is flushed to zero.
    auto error = [&](float s, float b) {
        return s * (a.sigmoid ? 4e-7f + (1.0f - s) * 1e-5f : 2e-5f) + 1.8e-7f * fabsf(b) + 1e-37f;
    };
    unsigned key[Each];
#pragma unroll
    for (int i = 0; i < Each; ++i) {
        const float b = score[i] > -INFINITY ? share[i] + bias[i] : -INFINITY;
        key[i] = ordered(fmaxf(b, -INFINITY));  // a NaN is left out
    }
    constexpr float most_exact = 1e30f;  // larger sums with biases could pass FP32's range
    auto* keys = reinterpret_cast<unsigned*>(keys_of + warp * room_of(a));
    if (a.kept_groups < a.groups) {
        const int size = a.experts / a.groups;
        // lane g has group g's value: a group is one register's lanes, or is read from shared memory
        unsigned first = 0, second = 0;
        if (size == 32) {
#pragma unroll
            for (int i = 0; i < Each; ++i) {
                const unsigned top = __reduce_max_sync(0xffffffffu, key[i]);
                const unsigned winners = __ballot_sync(0xffffffffu, key[i] == top);
                const unsigned next = __reduce_max_sync(0xffffffffu, lane == __ffs(winners) - 1 ? 0u : key[i]);
                if (lane == i) first = top, second = next;
            }
        } else {
            certain = certain && a.groups <= 32;
#pragma unroll
            for (int i = 0; i < Each; ++i) {
                if (i * 32 + lane < a.experts) keys[i * 32 + lane] = key[i];
            }
            __syncwarp();
            for (int j = 0; lane < a.groups && j < size; ++j) {
                const unsigned k = keys[lane * size + j];
                second = max(second, min(first, k));
                first = max(first, k);
            }
            __syncwarp();
        }
        const bool some = lane < a.groups && first != 0;
        const float value = some ? value_of(first) + (second == 0 ? 0.0f : value_of(second)) : -INFINITY;
        // two shares' errors, at most: a softmax's sum to one, a sigmoid's have s (1 - s) <= 1/4
        const float off = (a.sigmoid ? 7e-6f : 2.2e-5f) +
            3.6e-7f * (some ? fabsf(value_of(first)) + (second == 0 ? 0.0f : fabsf(value_of(second))) : 0.0f);
        int place = 0;
        for (int g = 0; g < min(a.groups, 32); ++g) {
            const float other = __shfl_sync(0xffffffffu, value, g);
            place += other > value || (other == value && g < lane);
        }
        certain = certain && (!some || fabsf(value) <= most_exact);
        const bool stays = lane < a.groups && place < a.kept_groups;
        const unsigned kept = __ballot_sync(0xffffffffu, stays);
        // the least that a group that stays may have, and the most of the others (groups without an expert are of no matter)
        const unsigned least = __reduce_min_sync(0xffffffffu, stays && some ? ordered(value - off) : 0xffffffffu);
        const unsigned most_out = __reduce_max_sync(0xffffffffu, !stays && some ? ordered(value + off) : 0u);
        certain = certain && least > most_out;
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            const int g = size == 32 ? i : (i * 32 + lane) / size;
            if (g >= 32 || !(kept >> g & 1u)) key[i] = 0;
        }
    }

    // Of the lanes' largest keys the (count + 1)-th bounds the (count + 1)-th of all; those above it, few more, are put in
    // order, a lane each.
    unsigned bound = 0;
#pragma unroll
    for (int i = 0; i < Each; ++i) bound = max(bound, key[i]);
    if (a.count < 16) {  // by taking the largest off
        unsigned largest = 0;
#pragma unroll 1
        for (int k = 0; k <= a.count; ++k) {
            largest = __reduce_max_sync(0xffffffffu, bound);
            if (bound == largest) bound = 0;
        }
        bound = max(1u, largest);
    } else {
#pragma unroll
        for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
            for (int apart = size / 2; apart > 0; apart /= 2) {
                const unsigned other = __shfl_xor_sync(0xffffffffu, bound, apart);
                bound = ((lane & apart) == 0) == ((lane & size) == 0) ? max(bound, other) : min(bound, other);
            }
        }
        bound = max(1u, __shfl_sync(0xffffffffu, bound, min(a.count, 31)));
    }
    auto* entries = reinterpret_cast<unsigned long long*>(keys);
    int candidates = 0;
#pragma unroll
    for (int i = 0; i < Each; ++i) {
        const unsigned holders = __ballot_sync(0xffffffffu, key[i] >= bound);
        if (holders == 0) continue;
        const int at = candidates + __popc(holders & ((1u << lane) - 1));
        if (key[i] >= bound && at < 32) {
            entries[at] = static_cast<unsigned long long>(key[i]) << 32 | ~static_cast<unsigned>(i * 32 + lane);
            auto* values = reinterpret_cast<float*>(entries + 32) + at * 4;
            values[0] = share[i], values[1] = score[i], values[2] = bias[i];
        }
        candidates += __popc(holders);
    }
    __syncwarp();
    // The most that an expert behind the candidates may have: below the bound, and with a bias of its own any share.
    const float edge = value_of(bound);
    const float reach = bound == 1 ? -INFINITY
        : a.bias == nullptr        ? edge + error(edge, edge)
                                   : edge + ((a.sigmoid ? 2.8e-6f : 2e-5f * largest_share) + 1.8e-7f * fabsf(edge) + 1e-37f);
    certain = certain && candidates <= 32;
    const int n = min(candidates, 32);
    const unsigned long long entry = lane < n ? entries[lane] : 0;
    int place = 0;
    for (int k = 0; k < n; ++k) place += entries[k] > entry;
    if (lane >= n) place = lane;
    const float4 mine_here = reinterpret_cast<const float4*>(entries + 32)[min(lane, max(n, 1) - 1)];
    __syncwarp();
    // lane l takes the candidate whose place is l
    auto* slots = reinterpret_cast<int*>(entries);
    slots[place] = lane;
    __syncwarp();
    const int from = slots[lane];
    const int chosen = static_cast<int>(~static_cast<unsigned>(__shfl_sync(0xffffffffu, entry, from)));
    const float v = value_of(static_cast<unsigned>(__shfl_sync(0xffffffffu, entry, from) >> 32));
    const float s = __shfl_sync(0xffffffffu, mine_here.x, from), mine = __shfl_sync(0xffffffffu, mine_here.y, from),
                b = __shfl_sync(0xffffffffu, mine_here.z, from);
    {
        // Each choice has to lie above all that come after it by both errors, but for those right after it that have the
        // same score and bias. Equal ones at the last choice stand for it: the last of them is looked at too.
        const float off = lane < n ? error(s, v) : 0.0f;
        float after = lane < n ? v + off : -INFINITY;  // the most of this and of later ones
        after = fmaxf(after, lane == 31 ? reach : -INFINITY);
#pragma unroll
        for (int apart = 1; apart < 32; apart *= 2) {
            const float other = __shfl_down_sync(0xffffffffu, after, apart);
            if (lane + apart < 32) after = fmaxf(after, other);
        }
        after = __shfl_down_sync(0xffffffffu, after, 1);
        if (lane == 31) after = reach;
        const float next_l = __shfl_down_sync(0xffffffffu, mine, 1), next_b = __shfl_down_sync(0xffffffffu, b, 1);
        const bool tied = lane + 1 < n && mine == next_l && b == next_b;
        const unsigned runs = __ballot_sync(0xffffffffu, tied) >> (a.count - 1);
        const int last = a.count - 1 + __ffs(static_cast<int>(~runs)) - 1;
        if (lane <= last && lane < n && !tied && !(v - off > after && fabsf(v) <= most_exact)) certain = false;
    }
    certain = __all_sync(0xffffffffu, certain);
    if (!certain) {
        exactly<T, Each>(a, token, keys_of + warp * room_of(a));
        return;
    }
    const bool there = lane < min(a.count, n);
    double weight = 0.0;
    if (a.sigmoid) {
        if (there) weight = 1.0 / (1.0 + exp(-static_cast<double>(mine)));
    } else {
        if (there) weight = exp(static_cast<double>(mine) - static_cast<double>(most));
        if (!a.renormalise) {
            double sum = 0.0;
#pragma unroll
            for (int i = 0; i < Each; ++i) {
                if (score[i] > -INFINITY) sum += exp(static_cast<double>(score[i]) - static_cast<double>(most));
            }
            weight /= warp_sum(sum);
        }
    }
    if (a.renormalise) {
        const double sum = warp_sum(weight);
        weight = sum > 0.0 ? weight / sum : 0.0;
    }
    if (lane < a.count) {
        a.choices[token * a.count + lane] = there ? chosen : -1;
        a.weights[token * a.count + lane] = there ? static_cast<float>(weight * static_cast<double>(a.scale)) : 0.0f;
    }
}

template <typename T, int Each>
cudaError_t launch(const RouteArgs& a, cudaStream_t stream) {
    const std::int64_t blocks = (a.tokens + route_warps - 1) / route_warps;
    std::size_t shared = a.kept_groups < a.groups ? static_cast<std::size_t>(route_warps) * a.experts * 8 : 0;
    auto kernel = exact_kernel<T, Each>;
    if constexpr (Each <= 8) {
        if (a.count < 32) kernel = route_kernel<T, Each>, shared = static_cast<std::size_t>(route_warps) * room_of(a) * 8;
    }
    return kernels::launch_overlapped(kernel, dim3(static_cast<unsigned>(blocks)), dim3(route_warps * 32), shared, stream, a);
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
