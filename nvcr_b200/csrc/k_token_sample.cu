// The choice of a symbol from a row of logits l and a uniform number u. With w = exp((l - max l) / temperature) and the
// symbols in the order of falling logits, equal ones by index: the first top_k of them, of these the shortest prefix
// with at least top_p of their weight, of these the ones with w >= min_p are kept; chosen is the first of the kept, in
// the order of their indexes, whose running sum of weights is above u times the whole.
//
// Every filter keeps a prefix of that order, so what is kept is told by a threshold: all logits above one, and the
// first few equal to it. Weights are FP64 and summed as whole multiples of 2^-43 of the largest, so that no order of
// sums changes a choice.
#include "token_elements.cuh"

#include <cmath>

namespace nvcr_sm100::token {
namespace {

constexpr int sample_threads = 1024;
constexpr int bins = 2048;

// The order of logits as that of unsigned integers; 0: left out (-infinity, NaN). -0 and +0 are equal.
template <typename T>
__device__ __forceinline__ unsigned key_of(T logit) {
    const float v = widen(logit) + 0.0f;
    if (!(v > -INFINITY)) return 0;
    const unsigned bits = __float_as_uint(v);
    return bits >> 31 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float logit_of(unsigned key) {
    return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

struct Row {
    unsigned top;        // the largest key
    double temperature;  // 0: the largest alone
};

__device__ __forceinline__ double share_of(unsigned key, const Row& row) {
    if (key == 0) return 0.0;
    if (key == row.top) return 1.0;  // infinite ones too
    if (row.temperature == 0.0) return 0.0;
    return exp((static_cast<double>(logit_of(key)) - static_cast<double>(logit_of(row.top))) / row.temperature);
}
using Weight = unsigned long long;
__device__ __forceinline__ Weight weight_of(double share) { return static_cast<Weight>(__double2ull_rn(share * 8796093022208.0)); }

struct Sums {
    unsigned counts[bins];
    unsigned low[bins], high[bins];  // halves of the weights' sums
    Weight warp_weight[32];
    unsigned warp_count[32];
    Weight found_weight;
    unsigned found_count;
    int found;
};

// The sums of a block's threads before each of them, and of all.
__device__ __forceinline__ Weight before(Weight mine, Weight* scratch, Weight& all) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    Weight sum = mine;
    for (int o = 1; o < 32; o *= 2) {
        const Weight v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
    }
    __syncthreads();
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    Weight earlier = 0;
    all = 0;
    for (int w = 0; w < sample_threads / 32; ++w) {
        if (w < warp) earlier += scratch[w];
        all += scratch[w];
    }
    return earlier + sum - mine;
}

// What is kept: keys above `key`, and the first `ties` equal to it.
struct Threshold {
    unsigned key;
    unsigned ties;
};

// The threshold of the shortest prefix that holds `wanted` of the counts (by_weight: of the weights), among what `kept`
// keeps: the key's bits from the top down, each level a histogram of the keys that agree with those found.
template <typename T>
__device__ Threshold find(const T* logits, int symbols, const Row& row, bool by_weight, Weight wanted, Threshold kept,
                          Sums& sums) {
    unsigned prefix = 0;
    int shift = 32;
    Weight above = 0;  // of keys above the prefix's
    for (const int width : {11, 11, 10}) {
        const int next = shift - width;
        __syncthreads();
        for (int i = threadIdx.x; i < bins; i += sample_threads) sums.counts[i] = sums.low[i] = sums.high[i] = 0;
        if (threadIdx.x == 0) sums.found = -1;
        __syncthreads();
        for (int i = threadIdx.x; i < symbols; i += sample_threads) {
            const unsigned key = key_of(logits[i]);
            if (key < kept.key || key == 0 || (shift < 32 && key >> shift != prefix)) continue;
            const unsigned bin = key >> next & ((1u << width) - 1);
            if (!by_weight) {
                atomicAdd(&sums.counts[bin], 1u);
                continue;
            }
            if (key == kept.key) continue;  // counted below
            const Weight w = weight_of(share_of(key, row));
            if (w == 0) continue;
            const unsigned low = static_cast<unsigned>(w), old = atomicAdd(&sums.low[bin], low);
            atomicAdd(&sums.high[bin], static_cast<unsigned>(w >> 32) + (old + low < old ? 1u : 0u));
        }
        __syncthreads();
        if (by_weight && threadIdx.x == 0 && kept.key != 0 && (shift == 32 || kept.key >> shift == prefix)) {
            const unsigned bin = kept.key >> next & ((1u << width) - 1);
            const Weight w = (static_cast<Weight>(sums.high[bin]) << 32 | sums.low[bin]) +
                kept.ties * weight_of(share_of(kept.key, row));
            sums.low[bin] = static_cast<unsigned>(w), sums.high[bin] = static_cast<unsigned>(w >> 32);
        }
        __syncthreads();
        // from the top bin down: thread t has bins - 1 - 2 t and the one below it
        const int first = bins - 1 - 2 * static_cast<int>(threadIdx.x);
        auto of = [&](int bin) {
            return by_weight ? static_cast<Weight>(sums.high[bin]) << 32 | sums.low[bin] : static_cast<Weight>(sums.counts[bin]);
        };
        Weight all;
        const Weight one = of(first), two = of(first - 1);
        const Weight earlier = above + before(one + two, sums.warp_weight, all);
        if (earlier < wanted && earlier + one + two >= wanted) {
            const bool upper = earlier + one >= wanted;
            sums.found = upper ? first : first - 1;
            sums.found_weight = upper ? earlier : earlier + one;
        }
        __syncthreads();
        if (sums.found < 0) return kept;  // there is less than wanted: all of it
        prefix = prefix << width | static_cast<unsigned>(sums.found);
        above = sums.found_weight;
        shift = next;
    }
    __syncthreads();
    const Weight each = by_weight ? weight_of(share_of(prefix, row)) : 1;
    const Weight ties = (wanted - above + each - 1) / each;
    return {prefix, static_cast<unsigned>(ties)};
}

__device__ __forceinline__ Threshold stricter(Threshold a, Threshold b) {
    return a.key > b.key || (a.key == b.key && a.ties < b.ties) ? a : b;
}

template <typename T>
__global__ void __launch_bounds__(sample_threads) sample_kernel(SampleArgs a) {
    __shared__ Sums sums;
    join_chain();
    const std::int64_t r = blockIdx.x;
    const T* logits = static_cast<const T*>(a.logits) + r * a.stride;
    const int symbols = a.symbols, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const float temperature = a.temperatures == nullptr ? a.temperature : a.temperatures[r];
    const float top_p = a.top_ps == nullptr ? a.top_p : a.top_ps[r];
    const float min_p = a.min_ps == nullptr ? a.min_p : a.min_ps[r];
    const int top_k = a.top_ks == nullptr ? a.top_k : a.top_ks[r];
    const float uniform = a.uniforms[r];

    unsigned top = 0;
    for (int i = threadIdx.x; i < symbols; i += sample_threads) top = max(top, key_of(logits[i]));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) sums.warp_count[warp] = top;
    __syncthreads();
    for (int w = 0; w < sample_threads / 32; ++w) top = max(top, sums.warp_count[w]);
    if (top == 0) {  // nothing to choose
        if (threadIdx.x == 0) a.chosen[r] = -1, a.probabilities[r] = 0.0f;
        return;
    }
    const Row row{top, temperature > 0.0f ? static_cast<double>(temperature) : 0.0};
    Threshold kept{0, 0};
    if (row.temperature == 0.0) {
        kept = {top, 1};
    } else {
        if (top_k > 0 && top_k < symbols) kept = find(logits, symbols, row, false, top_k, kept, sums);
        if (top_p < 1.0f) {
            Weight mine = 0, all;
            for (int i = threadIdx.x; i < symbols; i += sample_threads) {
                const unsigned key = key_of(logits[i]);
                if (key > kept.key) mine += weight_of(share_of(key, row));
            }
            before(mine, sums.warp_weight, all);
            if (kept.key != 0) all += kept.ties * weight_of(share_of(kept.key, row));
            const double part = ceil(static_cast<double>(fmaxf(top_p, 0.0f)) * static_cast<double>(all));
            const Weight wanted = max(static_cast<Weight>(1), static_cast<Weight>(part));
            kept = stricter(kept, find(logits, symbols, row, true, wanted, kept, sums));
        }
    }
    const double least = min_p > 0.0f ? static_cast<double>(fminf(min_p, 1.0f)) : 0.0;

    // a thread a run of symbols, in the order of their indexes
    const int each = (symbols + sample_threads - 1) / sample_threads;
    const int from = min(symbols, static_cast<int>(threadIdx.x) * each), to = min(symbols, from + each);
    Weight ties = 0, all_ties;
    for (int i = from; i < to; ++i) ties += key_of(logits[i]) == kept.key;
    const Weight earlier_ties = before(ties, sums.warp_weight, all_ties);
    auto walk = [&](auto&& visit) {
        Weight nth = earlier_ties;
        for (int i = from; i < to; ++i) {
            const unsigned key = key_of(logits[i]);
            if (key == 0 || key < kept.key || (key == kept.key && nth++ >= kept.ties)) continue;
            const double share = share_of(key, row);
            if (share >= least && !visit(i, share)) return;
        }
    };
    Weight mine = 0, all;
    walk([&](int, double share) {
        mine += weight_of(share);
        return true;
    });
    Weight sum = before(mine, sums.warp_weight, all);
    // u in units of 2^-64; 0 for a NaN and below, the last symbol from 1 on
    const unsigned long long u = !(uniform > 0.0f) ? 0ull
        : uniform >= 1.0f                          ? ~0ull
                                                   : static_cast<unsigned long long>(static_cast<double>(uniform) * 18446744073709551616.0);
    const Weight wanted = __umul64hi(u, all);  // below `all`
    if (wanted >= sum && wanted < sum + mine) {
        walk([&](int i, double share) {
            sum += weight_of(share);
            if (sum <= wanted) return true;
            a.chosen[r] = i;
            a.probabilities[r] = static_cast<float>(share * 8796093022208.0 / static_cast<double>(all));
            return false;
        });
    }
}

template <typename T>
cudaError_t launch(const SampleArgs& a, cudaStream_t stream) {
    return kernels::launch_overlapped(sample_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(sample_threads), 0, stream, a);
}

}  // namespace

cudaError_t sample(const SampleArgs& a, cudaStream_t stream) {
    if (a.rows == 0) return cudaSuccess;
    switch (a.type) {
    case Type::f16: return launch<__half>(a, stream);
    case Type::bf16: return launch<__nv_bfloat16>(a, stream);
    default: return launch<float>(a, stream);
    }
}

}  // namespace nvcr_sm100::token
