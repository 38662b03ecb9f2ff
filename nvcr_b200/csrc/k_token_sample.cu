// The choice of a symbol from a row of logits l and a uniform number u. With w = exp((l - max l) / temperature) and the
// symbols in the order of falling logits, equal ones by index: the first top_k of them, of these the shortest prefix
// with at least top_p of their weight, of these the ones with w >= min_p are kept; chosen is the first of the kept, in
// the order of their indexes, whose running sum of weights is above u times the whole.
//
// Every filter keeps a prefix of that order, so what is kept is told by a threshold: all logits above one, and the
// first few equal to it. Weights are FP64 and summed as whole multiples of 2^-43 of the largest, so that no order of
// sums changes a choice, and which symbol is chosen does not hang on a rounding to FP32.
//
// A few rows are a cluster's each, of up to eight blocks, which has the row in its registers, read once (`cluster_kernel`):
// * Where the symbols that can be kept are few (`candidates`: by min_p, top_k or ten octaves below the largest), they go
//   to the first block, which sorts them and ends the row (`finish`). The rest is summed in FP32 for top_p's whole; a
//   choice that hangs on that sum's error is made again exactly.
// * Where they are many, a histogram of weights or counts over the cluster says between which logits the threshold lies,
//   and these are sorted (`find`); the choice is found by sums of each warp's runs (`locate`).
// Many rows go through three launches whose blocks wait for no other: parts of rows, whose candidates and sums go to memory
// (`part_kernel`); a block a row, which ends it (`end_kernel`); the rows that were not ended, a cluster each
// (`rest_kernel`). 256 rows of 131072 took 58 us by clusters, whose blocks were idle while they waited for one another.
//
// Longer rows (past 2^18 FP32 symbols, 2^19 in 16 bits), infinite logits and, of a few rows, choices that hang on the FP32
// sum's error take `row_by_block`, which finds the threshold's bits from memory with one block in up to eight passes: one
// row of 32768 FP32 logits 47 us (by an infinity 125), of 131072 166, of 2^18 + 1 940, of 2^20 4.2 ms.
//
// One row of 32768 FP32 logits (top_k 50, top_p 0.95) 11 us: launch, four exchanges of a cluster, one warp's end of the
// row. 256 rows of 131072 BF16 logits (top_p 0.9, min_p 0.01) 37 us, of which 10 are the logits at HBM's rate: parts take
// 25, by an exponential a logit; ends 13, by the latency of sums and FP64 weights, some of it side by side.
#include "token_elements.cuh"

#include <algorithm>
#include <climits>
#include <cmath>

namespace nvcr_sm100::token {
namespace {

constexpr int threads = 512;
constexpr int warps = threads / 32;
constexpr int bins = 2048;
constexpr int most_blocks = 8;
constexpr int most_candidates = 2048;
constexpr int most_vectors = 16;  // a thread
constexpr int most_counted = 128; // symbols whose places are counted, not sorted
constexpr int cut_bins = 256;     // of `cut`, so many an octave:
constexpr float cut_steps = 5.5f;

// The order of logits as that of unsigned integers; 0: left out (-infinity, NaN). -0 and +0 are equal.
__device__ __forceinline__ unsigned key_of(float logit) {
    const float v = logit + 0.0f;
    if (!(v > -INFINITY)) return 0;
    const unsigned bits = __float_as_uint(v);
    return bits >> 31 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float logit_of(unsigned key) {
    return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

using Weight = unsigned long long;
constexpr double unit = 8796093022208.0;  // 2^43: 2^20 weights stay below 2^63
constexpr int table_size = 64;

struct Row {
    float largest;
    double temperature;   // 0: the largest alone
    double least;         // of a kept share
    double factor;        // steps of 2^(1/64) a logit
    const double* table;  // unit * 2^(i / 64)
};

// A logit's share of the largest one's weight, in units. With y = 64 log2(e) (l - max) / temperature = n + f, |f| <= 1/2:
// 2^(n / 64) from the table and its exponent, e^(f ln(2) / 64) by Taylor's polynomial, whose fifth term is below 4e-14.
__device__ __forceinline__ double share_of(float logit, const Row& row) {
    const double y = (static_cast<double>(logit) - static_cast<double>(row.largest)) * row.factor;
    const double whole = y + 6755399441055744.0;  // 1.5 * 2^52: rounds to a whole number, in the low word
    const int n = __double2loint(whole);
    const double f = y - (whole - 6755399441055744.0);
    constexpr double c = 0.69314718055994530942 / table_size;
    const double p = fma(f, fma(f, fma(f, fma(f, c * c * c * c / 24.0, c * c * c / 6.0), c * c / 2.0), c), 1.0);
    const double w = row.table[n & (table_size - 1)] * p;
    const double found = __hiloint2double(__double2hiint(w) + (n >> 6) * (1 << 20), __double2loint(w));
    // Infinite largest ones share; below 2^-46, less than half a unit, there is none, and none for a NaN (y is one), an
    // infinity, or all but the largest at temperature 0, whose factor is infinite.
    return logit == row.largest ? unit : y > -46.0 * table_size ? found : 0.0;
}
// One copy of it for code that runs once a row.
__device__ __noinline__ double share_once(float logit, const Row& row) { return share_of(logit, row); }
// Rounded to whole units: below 2^52 the sum's low bits.
__device__ __forceinline__ Weight weight_of(double share) {
    return static_cast<Weight>(__double_as_longlong(share + 4503599627370496.0)) & 0xfffffffffffffull;
}
__device__ __forceinline__ float probability_of(double share, Weight all) {
    return static_cast<float>(share / static_cast<double>(all));
}

// What is kept: keys above `key`, and the first `ties` equal to it.
struct Threshold {
    unsigned key;
    unsigned ties;
};
__device__ __forceinline__ Threshold stricter(Threshold a, Threshold b) {
    return a.key > b.key || (a.key == b.key && a.ties < b.ties) ? a : b;
}

// The least weight that holds top_p of all.
__device__ __forceinline__ Weight part_of(float top_p, Weight all) {
    const double part = ceil(static_cast<double>(fmaxf(top_p, 0.0f)) * static_cast<double>(all));
    return max(static_cast<Weight>(1), static_cast<Weight>(part));
}

// u times the whole, rounded down: below the whole. u is 0 for a NaN and below, the last symbol from 1 on.
__device__ __forceinline__ Weight part_of_uniform(float uniform, Weight all) {
    const unsigned long long u = !(uniform > 0.0f) ? 0ull
        : uniform >= 1.0f                          ? ~0ull
                                                   : static_cast<unsigned long long>(static_cast<double>(uniform) * 18446744073709551616.0);
    return __umul64hi(u, all);
}

struct Settings {
    float temperature, top_p, min_p, uniform;
    int top_k;
};
__device__ __forceinline__ Settings settings_of(const SampleArgs& a, std::int64_t r) {
    return {a.temperatures == nullptr ? a.temperature : a.temperatures[r], a.top_ps == nullptr ? a.top_p : a.top_ps[r],
            a.min_ps == nullptr ? a.min_p : a.min_ps[r], a.uniforms[r], a.top_ks == nullptr ? a.top_k : a.top_ks[r]};
}
__device__ __forceinline__ Row row_of(unsigned top, const Settings& s, const double* table) {
    const double temperature = s.temperature > 0.0f ? static_cast<double>(s.temperature) : 0.0;
    return {logit_of(top), temperature, s.min_p > 0.0f ? static_cast<double>(fminf(s.min_p, 1.0f)) * unit : 0.0,
            table_size * 1.4426950408889634074 / temperature, table};
}
// By the block's first threads; the caller synchronises.
__device__ __forceinline__ void make_table(double* table) {
    if (threadIdx.x < table_size) table[threadIdx.x] = unit * exp2(threadIdx.x / static_cast<double>(table_size));
}

struct Sums {
    alignas(16) unsigned low[bins];  // counts, or halves of the weights' sums
    alignas(16) unsigned high[bins];
    Weight scratch[warps];
    Weight found_weight;
    int found;
};

// The sum of the block's threads before this one, and of all.
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
#pragma unroll 4
    for (int w = 0; w < warps; ++w) {
        if (w < warp) earlier += scratch[w];
        all += scratch[w];
    }
    return earlier + sum - mine;
}

__device__ __forceinline__ void add(Sums& sums, unsigned bin, Weight w) {
    const unsigned low = static_cast<unsigned>(w), old = atomicAdd(&sums.low[bin], low);
    atomicAdd(&sums.high[bin], static_cast<unsigned>(w >> 32) + (old + low < old ? 1u : 0u));
}

// The bin, from the top down, at which the sums pass `wanted`, and what lies above it. found stays -1 where they do not.
template <typename Of>
__device__ __forceinline__ void pass(Sums& sums, Weight above, Weight wanted, Of&& of) {
    constexpr int each = bins / threads;
    const int first = bins - 1 - each * static_cast<int>(threadIdx.x);
    Weight mine[each], sum = 0, all;
#pragma unroll
    for (int i = 0; i < each; ++i) sum += mine[i] = of(first - i);
    Weight earlier = above + before(sum, sums.scratch, all);
#pragma unroll
    for (int i = 0; i < each; ++i) {
        if (earlier < wanted && earlier + mine[i] >= wanted) sums.found = first - i, sums.found_weight = earlier;
        earlier += mine[i];
    }
}

// ---- a block a row, from memory: any row, exactly ----

template <typename T>
__device__ Threshold find_by_block(const T* logits, int symbols, const Row& row, bool by_weight, Weight wanted, Threshold kept,
                                   Sums& sums) {
    unsigned prefix = 0;
    int shift = 32;
    Weight above = 0;  // of keys above the prefix's
    for (const int width : {11, 11, 10}) {
        const int next = shift - width;
        __syncthreads();
        for (int i = threadIdx.x; i < bins; i += threads) sums.low[i] = sums.high[i] = 0;
        if (threadIdx.x == 0) sums.found = -1;
        __syncthreads();
        for (int i = threadIdx.x; i < symbols; i += threads) {
            const unsigned key = key_of(widen(logits[i]));
            if (key < kept.key || key == 0 || (shift < 32 && key >> shift != prefix)) continue;
            const unsigned bin = key >> next & ((1u << width) - 1);
            if (!by_weight) {
                atomicAdd(&sums.low[bin], 1u);
            } else if (key != kept.key) {  // those are added below
                const Weight w = weight_of(share_once(logit_of(key), row));
                if (w != 0) add(sums, bin, w);
            }
        }
        __syncthreads();
        if (by_weight && threadIdx.x == 0 && kept.key != 0 && (shift == 32 || kept.key >> shift == prefix)) {
            add(sums, kept.key >> next & ((1u << width) - 1), kept.ties * weight_of(share_once(logit_of(kept.key), row)));
        }
        __syncthreads();
        pass(sums, above, wanted, [&](int bin) { return static_cast<Weight>(sums.high[bin]) << 32 | sums.low[bin]; });
        __syncthreads();
        if (sums.found < 0) return kept;  // there is less than wanted: all of it
        prefix = prefix << width | static_cast<unsigned>(sums.found);
        above = sums.found_weight;
        shift = next;
    }
    __syncthreads();
    const Weight each = by_weight ? weight_of(share_once(logit_of(prefix), row)) : 1;
    return {prefix, static_cast<unsigned>((wanted - above + each - 1) / each)};
}

template <typename T>
__device__ __noinline__ void row_by_block(const SampleArgs& a, std::int64_t r, Sums& sums, const double* table) {
    const T* logits = static_cast<const T*>(a.logits) + r * a.stride;
    const int symbols = a.symbols, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const Settings s = settings_of(a, r);
    unsigned top = 0;
    for (int i = threadIdx.x; i < symbols; i += threads) top = max(top, key_of(widen(logits[i])));
    top = __reduce_max_sync(0xffffffffu, top);
    __syncthreads();
    if (lane == 0) sums.scratch[warp] = top;
    __syncthreads();
    for (int w = 0; w < warps; ++w) top = max(top, static_cast<unsigned>(sums.scratch[w]));
    if (top == 0) {  // nothing to choose
        if (threadIdx.x == 0) a.chosen[r] = -1, a.probabilities[r] = 0.0f;
        return;
    }
    const Row row = row_of(top, s, table);
    Threshold kept{0, 0};
    if (row.temperature == 0.0) {
        kept = {top, 1};
    } else {
        if (s.top_k > 0 && s.top_k < symbols) kept = find_by_block(logits, symbols, row, false, s.top_k, kept, sums);
        if (s.top_p < 1.0f) {
            Weight mine = 0, all;
            for (int i = threadIdx.x; i < symbols; i += threads) {
                const unsigned key = key_of(widen(logits[i]));
                if (key > kept.key) mine += weight_of(share_once(logit_of(key), row));
            }
            before(mine, sums.scratch, all);
            if (kept.key != 0) all += kept.ties * weight_of(share_once(logit_of(kept.key), row));
            kept = stricter(kept, find_by_block(logits, symbols, row, true, part_of(s.top_p, all), kept, sums));
        }
    }
    // a thread a run of symbols, in the order of their indexes
    const int each = (symbols + threads - 1) / threads;
    const int from = min(symbols, static_cast<int>(threadIdx.x) * each), to = min(symbols, from + each);
    Weight ties = 0, all_ties;
    for (int i = from; i < to; ++i) ties += key_of(widen(logits[i])) == kept.key;
    const Weight earlier_ties = before(ties, sums.scratch, all_ties);
    auto walk = [&](auto&& visit) {
        Weight nth = earlier_ties;
        for (int i = from; i < to; ++i) {
            const unsigned key = key_of(widen(logits[i]));
            if (key == 0 || key < kept.key || (key == kept.key && nth++ >= kept.ties)) continue;
            const double share = share_once(logit_of(key), row);
            if (share >= row.least && !visit(i, share)) return;
        }
    };
    Weight mine = 0, all;
    walk([&](int, double share) {
        mine += weight_of(share);
        return true;
    });
    Weight sum = before(mine, sums.scratch, all);
    const Weight wanted = part_of_uniform(s.uniform, all);
    if (wanted >= sum && wanted < sum + mine) {
        walk([&](int i, double share) {
            sum += weight_of(share);
            if (sum <= wanted) return true;
            a.chosen[r] = i;
            a.probabilities[r] = probability_of(share, all);
            return false;
        });
    }
}

template <typename T>
__global__ void __launch_bounds__(threads) block_kernel(SampleArgs a) {
    __shared__ Sums sums;
    __shared__ double table[table_size];
    make_table(table);
    join_chain();
    __syncthreads();
    row_by_block<T>(a, blockIdx.x, sums, table);
}

// ---- a cluster a row, from registers ----

__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ std::uint32_t at_block(const void* here, int rank) {
    std::uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                 : "=r"(there)
                 : "r"(static_cast<std::uint32_t>(__cvta_generic_to_shared(here))), "r"(rank));
    return there;
}
__device__ __forceinline__ void put(const void* here, int rank, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at_block(here, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned get(const unsigned* here, int rank) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at_block(here, rank)));
    return v;
}
__device__ __forceinline__ uint4 get_four(const unsigned* here, int rank) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at_block(here, rank)));
    return v;
}

struct Shared {
    Sums sums;
    unsigned long long gathered[most_candidates];  // the first block's: a part for each block
    alignas(16) unsigned long long sorted[most_candidates];
    Weight weights[most_candidates];  // running sums
    Weight cells[most_vectors * warps];
    double table[table_size];
    unsigned long long maxima[most_blocks], totals[most_blocks], counts[2][most_blocks], sums_of[2][most_blocks];
    unsigned long long told[2];  // the first block to all
    float parts[2][warps];
    unsigned count, queued, wide;
    unsigned kept, low, high;
    int cut;
};

template <typename T>
struct Elements {
    static constexpr int each = 16 / sizeof(T);
    static __device__ __forceinline__ float get(const uint4& v, int i) {
        const unsigned words[4] = {v.x, v.y, v.z, v.w};
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(words[i]);
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            return __uint_as_float(i % 2 == 0 ? words[i / 2] << 16 : words[i / 2] & 0xffff0000u);
        } else {
            return half_bits(static_cast<std::uint16_t>(words[i / 2] >> (i % 2 * 16)));
        }
    }
    static __device__ __forceinline__ float pick(const uint4& v, int i) {  // i known at run time only
        const int at = i / (each / 4);
        const unsigned word = at == 0 ? v.x : at == 1 ? v.y : at == 2 ? v.z : v.w;
        const uint4 found{word, word, word, word};
        return sizeof(T) == 4 || i % 2 == 0 ? get(found, 0) : get(found, 1);
    }
    static __device__ __forceinline__ float largest(const uint4& v) {  // no NaN, unless all are
        if constexpr (sizeof(T) == 4) {
            return fmaxf(fmaxf(get(v, 0), get(v, 1)), fmaxf(get(v, 2), get(v, 3)));
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            const auto pair = [](const unsigned& w) { return reinterpret_cast<const __nv_bfloat162&>(w); };
            const __nv_bfloat162 most = __hmax2(__hmax2(pair(v.x), pair(v.y)), __hmax2(pair(v.z), pair(v.w)));
            return fmaxf(__low2float(most), __high2float(most));
        } else {
            const auto pair = [](const unsigned& w) { return reinterpret_cast<const __half2&>(w); };
            const __half2 most = __hmax2(__hmax2(pair(v.x), pair(v.y)), __hmax2(pair(v.z), pair(v.w)));
            return fmaxf(__low2float(most), __high2float(most));
        }
    }
    // -infinity in every place
    static __device__ __forceinline__ uint4 none() {
        const unsigned w = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __nv_bfloat16> ? 0xff80ff80u : 0xfc00fc00u;
        return {w, w, w, w};
    }
};

// Logits at .. of a row, with -infinity outside it.
template <typename T>
__device__ __forceinline__ uint4 load_vector(const T* logits, int symbols, int at) {
    using Of = Elements<T>;
    constexpr int each = Of::each;
    uint4 v = Of::none();
    if (at >= 0 && at + each <= symbols) {
        v = *reinterpret_cast<const uint4*>(logits + at);
    } else if (at + each > 0 && at < symbols) {
        unsigned words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < each; ++i) {
            if (at + i < 0 || at + i >= symbols) continue;
            if constexpr (sizeof(T) == 4) {
                words[i] = __float_as_uint(logits[at + i]);
            } else {
                const unsigned bits = reinterpret_cast<const std::uint16_t*>(logits)[at + i];
                words[i / 2] = i % 2 == 0 ? (words[i / 2] & 0xffff0000u) | bits : (words[i / 2] & 0xffffu) | bits << 16;
            }
        }
        v = {words[0], words[1], words[2], words[3]};
    }
    return v;
}

// What a cluster keeps: logits above `value`, and those equal to it up to index `last`. A NaN is not among them.
struct Kept {
    float value;
    int last;
    __device__ __forceinline__ bool holds(float l, int index) const { return l > value || (l == value && index <= last); }
};

// 2048 in falling order, by 512 threads: four neighbours a thread, so that only exchanges over 128 places and more pass
// through shared memory.
__device__ __noinline__ void sort(unsigned long long* shared) {
    static_assert(most_candidates == 4 * threads);
    unsigned long long v[4];
    const int base = 4 * static_cast<int>(threadIdx.x);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = shared[base + i];
    auto order = [](unsigned long long& a, unsigned long long& b, bool falling) {
        if ((a < b) == falling) {
            const unsigned long long t = a;
            a = b, b = t;
        }
    };
#pragma unroll 1
    for (int size = 2; size <= most_candidates; size *= 2) {
        int apart = size / 2;
        if (apart >= 128) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) shared[base + i] = v[i];
#pragma unroll 1
            for (; apart >= 128; apart /= 2) {
                __syncthreads();
#pragma unroll
                for (int k = 0; k < most_candidates / 2 / threads; ++k) {
                    const int p = static_cast<int>(threadIdx.x) + k * threads, at = 2 * p - (p & (apart - 1));
                    unsigned long long a = shared[at], b = shared[at + apart];
                    order(a, b, (at & size) == 0);
                    shared[at] = a, shared[at + apart] = b;
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = shared[base + i];
        }
#pragma unroll 1
        for (; apart >= 4; apart /= 2) {
            const bool lower = (base & apart) == 0, falling = ((base & size) == 0) == lower;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, v[i], apart / 4);
                v[i] = falling ? max(v[i], other) : min(v[i], other);
            }
        }
        if (size >= 4) {
            const bool falling = (base & size) == 0;
            order(v[0], v[2], falling), order(v[1], v[3], falling);
            order(v[0], v[1], falling), order(v[2], v[3], falling);
        } else {
            order(v[0], v[1], true), order(v[2], v[3], false);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) shared[base + i] = v[i];
    __syncthreads();
}

constexpr int most_crowded = 256;  // entries of a bin that are compared with one another

// n entries in falling order, n up to 2048: to bins by equal steps of their logits (shift < 0), or by their indexes'
// leading bits, and within a bin by comparing them all. 1300 take 3 us where `sort` takes 12; it is left for those that
// crowd in few bins.
__device__ __noinline__ void arrange(unsigned long long* list, int n, int shift, Sums& sums) {
    constexpr int most = most_candidates / threads, each = bins / threads;
    static_assert(each == 4);
    const int thread = static_cast<int>(threadIdx.x);
    __syncthreads();
    reinterpret_cast<uint4*>(sums.low)[thread] = {0, 0, 0, 0};
    unsigned long long entry[most];
    unsigned top = 0, least = 0xffffffffu;
#pragma unroll
    for (int k = 0; k < most; ++k) {
        const int i = k * threads + thread;
        entry[k] = i < n ? list[i] : 0;
        if (entry[k] != 0) top = max(top, static_cast<unsigned>(entry[k] >> 32)), least = min(least, static_cast<unsigned>(entry[k] >> 32));
    }
    float largest = 0.0f, scale = 0.0f;
    if (shift < 0) {
        top = __reduce_max_sync(0xffffffffu, top), least = __reduce_min_sync(0xffffffffu, least);
        if (thread % 32 == 0) sums.scratch[thread / 32] = static_cast<Weight>(top) << 32 | least;
        __syncthreads();
#pragma unroll 4
        for (int w = 0; w < warps; ++w) {
            const Weight both = sums.scratch[w];
            top = max(top, static_cast<unsigned>(both >> 32)), least = min(least, static_cast<unsigned>(both));
        }
        largest = logit_of(top);
        scale = (bins - 1) / (largest - logit_of(least));
    }
    __syncthreads();
    int bin[most];
    unsigned place[most];
#pragma unroll
    for (int k = 0; k < most; ++k) {
        if (entry[k] == 0) continue;
        const auto high = static_cast<unsigned>(entry[k] >> 32);
        // falling in the logit, whatever is rounded; a NaN, of an infinite scale, is the largest's
        bin[k] = shift < 0 ? min(bins - 1, static_cast<int>((largest - logit_of(high)) * scale)) : static_cast<int>(~high >> shift);
        place[k] = atomicAdd(&sums.low[bin[k]], 1u);
    }
    __syncthreads();
    const uint4 count = reinterpret_cast<const uint4*>(sums.low)[thread];
    Weight all;
    const auto first = static_cast<unsigned>(before(count.x + count.y + count.z + count.w, sums.scratch, all));
    reinterpret_cast<uint4*>(sums.high)[thread] = {first, first + count.x, first + count.x + count.y, first + count.x + count.y + count.z};
    if (__syncthreads_or(max(max(count.x, count.y), max(count.z, count.w)) > most_crowded)) {
        for (int i = n + thread; i < most_candidates; i += threads) list[i] = 0;
        sort(list);
        return;
    }
#pragma unroll
    for (int k = 0; k < most; ++k) {
        if (entry[k] != 0) list[sums.high[bin[k]] + place[k]] = entry[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < most; ++k) {
        if (entry[k] == 0) continue;
        const unsigned start = sums.high[bin[k]], end = start + sums.low[bin[k]];
        place[k] = start;
        for (unsigned i = start; i < end; ++i) place[k] += list[i] > entry[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < most; ++k) {
        if (entry[k] != 0) list[place[k]] = entry[k];
    }
    __syncthreads();
}

// FP32 sums of weights that are not candidates may be off by this share of them: exponents of up to 46 by 2.2 * 2^-24 of
// themselves (the factor's rounding and their own) and by 2^-24 of largest * factor, times ln 2; ex2.approx 2^-22, and up to
// 181 additions one after another.
__device__ __forceinline__ double bulk_error(float largest, float factor) {
    return 1.6e-5 + 5e-8 * fabs(static_cast<double>(largest) * static_cast<double>(factor));
}

template <typename T>
struct ClusterRow {
    using Of = Elements<T>;
    static constexpr int each = Of::each;
    const SampleArgs& a;
    Shared& shared;
    std::int64_t r;
    int rank, blocks;
    int vectors;  // of this thread
    int first;    // index of this thread's first element: of its n-th vector first + n * threads * each

    __device__ __forceinline__ uint4 load(int n) const {
        return load_vector(static_cast<const T*>(a.logits) + r * a.stride, a.symbols, first + n * threads * each);
    }

    // body(n, vector) for each, four loads at a time under way.
    template <typename Body>
    __device__ __forceinline__ void for_vectors(Body&& body) const {
        for (int n = 0; n < vectors; n += 4) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = n + i < vectors ? load(n + i) : Of::none();
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                if (n + i >= vectors) break;
                const uint4 one = i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3];
                body(n + i, one);
            }
        }
    }

    // body(first, elements 0 .. each / 2 - 1 of it) for both halves of a vector: as many FP64 values at once as there are
    // registers for.
    template <typename Body>
    static __device__ __forceinline__ void for_halves(const uint4& v, Body&& body) {
#pragma unroll 1
        for (int h = 0; h < 2; ++h) body(h * (each / 2), h == 0 ? uint4{v.x, v.y, 0, 0} : uint4{v.z, v.w, 0, 0});
    }

    // Where the running sum of amounts, in the order of indexes, first exceeds wanted(their whole): visit(index, logit, whole)
    // there, by one thread of the cluster.
    template <typename Amount, typename Wanted, typename Visit>
    __device__ __forceinline__ void locate(Amount&& amount, Wanted&& wanted_of, Visit&& visit) {
        __syncthreads();
        const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
        for_vectors([&](int n, const uint4& v) {
            Weight sum = 0;
            for_halves(v, [&](int from, const uint4& half) {
#pragma unroll
                for (int i = 0; i < each / 2; ++i) sum += amount(first + n * threads * each + from + i, Of::get(half, i));
            });
#pragma unroll
            for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) shared.cells[n * warps + warp] = sum;
        });
        __syncthreads();
        Weight block_sum = 0;
        if (warp == 0) {
            for (int c = lane; c < vectors * warps; c += 32) block_sum += shared.cells[c];
#pragma unroll
            for (int o = 16; o > 0; o /= 2) block_sum += __shfl_xor_sync(0xffffffffu, block_sum, o);
            if (lane < blocks) put(&shared.totals[rank], lane, block_sum);
        }
        cluster_sync();
        Weight earlier = 0, all = 0;
        for (int b = 0; b < blocks; ++b) {
            if (b < rank) earlier += shared.totals[b];
            all += shared.totals[b];
        }
        const Weight wanted = wanted_of(all);
        if (earlier > wanted || earlier + shared.totals[rank] <= wanted) return;
        int cell = 0;
        while (earlier + shared.cells[cell] <= wanted) earlier += shared.cells[cell++];
        if (cell % warps != warp) return;
        const int n = cell / warps;
        const uint4 v = load(n);
        Weight sum = 0;
#pragma unroll
        for (int i = 0; i < each; ++i) sum += amount(first + n * threads * each + i, Of::get(v, i));
        Weight to = sum;
        for (int o = 1; o < 32; o *= 2) {
            const Weight u = __shfl_up_sync(0xffffffffu, to, o);
            if (lane >= o) to += u;
        }
        Weight from = earlier + to - sum;
        if (wanted < from || wanted >= earlier + to) return;
#pragma unroll
        for (int i = 0; i < each; ++i) {
            const int index = first + n * threads * each + i;
            const float l = Of::get(v, i);
            const Weight w = amount(index, l);
            if (wanted >= from && wanted < from + w) visit(index, l, all);
            from += w;
        }
    }

    // The gathered symbols of all blocks, sorted; how many there are. Of up to 128 each one's place is counted, by a group of
    // threads.
    __device__ __forceinline__ int collect(const unsigned long long* counts, int part) {
        unsigned long long* from = shared.gathered;
        int n = 0;
        for (int b = 0; b < blocks; ++b) n += static_cast<int>(counts[b] & 0xffffffffu);
        unsigned long long* to = n <= most_counted ? shared.weights : shared.sorted;
        n = 0;
        for (int b = 0; b < blocks; ++b) {
            const int count = static_cast<int>(counts[b] & 0xffffffffu);
            for (int i = threadIdx.x; i < count; i += threads) to[n + i] = from[b * part + i];
            n += count;
        }
        if (n <= most_counted) {
            __syncthreads();
            const int group = group_of(n), i = static_cast<int>(threadIdx.x) / group;
            const unsigned long long mine = i < n ? to[i] : 0;
            int place = 0;
            for (int k = static_cast<int>(threadIdx.x) % group; k < n; k += group) place += to[k] > mine;
            for (int o = group / 2; o > 0; o /= 2) place += __shfl_xor_sync(0xffffffffu, place, o);
            if (i < n && threadIdx.x % group == 0) shared.sorted[place] = mine;
            __syncthreads();
            return n;
        }
        arrange(shared.sorted, n, -1, shared.sums);
        return n;
    }
    // Threads for each of n, a power of two.
    static __device__ __forceinline__ int group_of(int n) {
        int group = 32;
        while (group > 1 && group * n > threads) group /= 2;
        return group;
    }

    __device__ __forceinline__ void gather(unsigned key, int index, int part) {
        const unsigned nth = atomicAdd(&shared.count, 1u);
        if (nth < static_cast<unsigned>(part)) {
            put(&shared.gathered[rank * part + nth], 0, static_cast<unsigned long long>(key) << 32 | ~static_cast<unsigned>(index));
        }
    }

    // A histogram of the symbols that bin_of(logit) puts in a bin, the largest logits in the first, by counts or
    // weights: the bin in which wanted_of(whole) is reached, or -1, and what of it is wanted there.
    template <typename BinOf, typename WantedOf>
    __device__ __forceinline__ int reach(const Row& row, bool by_weight, const Kept& kept, BinOf&& bin_of, WantedOf&& wanted_of,
                                         Weight& wanted) {
        Sums& sums = shared.sums;
        __syncthreads();
        for (int i = threadIdx.x; i < bins; i += threads) sums.low[i] = sums.high[i] = 0;
        if (threadIdx.x == 0) sums.found = -1;
        __syncthreads();
        for_vectors([&](int n, const uint4& v) {
            for_halves(v, [&](int from, const uint4& half) {
                int bin[each / 2];
                Weight w[each / 2];
#pragma unroll
                for (int i = 0; i < each / 2; ++i) {
                    const float l = Of::get(half, i);
                    bin[i] = bin_of(l);
                    if (!kept.holds(l, first + n * threads * each + from + i)) bin[i] = -1;
                    if (by_weight) w[i] = weight_of(share_of(l, row));
                }
#pragma unroll
                for (int i = 0; i < each / 2; ++i) {
                    if (bin[i] < 0) continue;
                    if (!by_weight) {
                        atomicAdd(&sums.low[bin[i]], 1u);
                    } else if (w[i] != 0) {
                        add(sums, static_cast<unsigned>(bin[i]), w[i]);
                    }
                }
            });
        });
        cluster_sync();
        if (rank == 0) {
            constexpr int run = bins / threads;
            static_assert(run == 4);
            Weight mine[run] = {0, 0, 0, 0}, all = 0, sum = 0;
            const int first_bin = run * static_cast<int>(threadIdx.x);
#pragma unroll 1
            for (int from = 0; from < blocks; from += 4) {  // four blocks' loads under way: each takes some 700 cycles
                uint4 low[4], high[4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int of = min(from + b, blocks - 1);
                    low[b] = get_four(&sums.low[first_bin], of), high[b] = get_four(&sums.high[first_bin], of);
                }
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    if (from + b >= blocks) break;
                    mine[0] += static_cast<Weight>(high[b].x) << 32 | low[b].x, mine[1] += static_cast<Weight>(high[b].y) << 32 | low[b].y;
                    mine[2] += static_cast<Weight>(high[b].z) << 32 | low[b].z, mine[3] += static_cast<Weight>(high[b].w) << 32 | low[b].w;
                }
            }
#pragma unroll
            for (int i = 0; i < run; ++i) sum += mine[i];
            Weight earlier = before(sum, sums.scratch, all);
            const Weight want = wanted_of(all);
#pragma unroll
            for (int i = 0; i < run; ++i) {
                if (earlier < want && earlier + mine[i] >= want) {
                    sums.found = run * static_cast<int>(threadIdx.x) + i, sums.found_weight = want - earlier;
                }
                earlier += mine[i];
            }
            __syncthreads();
            if (threadIdx.x < static_cast<unsigned>(blocks)) {
                put(&shared.told[0], static_cast<int>(threadIdx.x), static_cast<unsigned long long>(sums.found));
                put(&shared.told[1], static_cast<int>(threadIdx.x), sums.found_weight);
            }
        }
        cluster_sync();
        wanted = shared.told[1];
        return static_cast<int>(shared.told[0]);
    }

    // What the shortest prefix of the symbols kept so far that holds top_k of them (by_weight: top_p of their weight) ends
    // with: a histogram over 46 octaves, of which bins hold equal steps, then the symbols of the bin that it ends in, in
    // order. A bin with too many of them is divided by keys, down to one key, whose symbols go by their indexes.
    __device__ __noinline__ Kept find(const Row& row, const Settings& s, bool by_weight, float largest, float factor, Kept kept) {
        const int part = most_candidates / blocks;
        const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
        auto octave_of = [&](float l) { return __fmul_rn(__fsub_rn(l, largest), -44.0f * factor); };
        auto octave_bin = [&](float l) {
            const float x = octave_of(l);
            return x < static_cast<float>(bins) ? static_cast<int>(x) : -1;  // a NaN is in none
        };
        Weight wanted;
        const int octave = reach(
            row, by_weight, kept, octave_bin,
            [&](Weight all) { return by_weight ? part_of(s.top_p, all) : static_cast<Weight>(s.top_k); }, wanted);
        if (octave < 0) return kept;  // there is less than wanted: all of it
        unsigned low = 0, high = 0;   // the keys looked at, once they are known
        for (int turn = 0;; ++turn) {
            if (threadIdx.x == 0) shared.count = 0;
            __syncthreads();
            unsigned least = 0xffffffffu, most = 0;
            const float from_logit = turn == 0 ? 0.0f : logit_of(low), to_logit = turn == 0 ? 0.0f : logit_of(high);
            for_vectors([&](int n, const uint4& v) {
                unsigned in = 0;  // the elements looked at
#pragma unroll
                for (int i = 0; i < each; ++i) {
                    const float l = Of::get(v, i);
                    bool here;
                    if (turn == 0) {
                        const float x = octave_of(l);
                        here = x >= static_cast<float>(octave) && x < static_cast<float>(octave + 1);
                    } else {
                        here = l >= from_logit && l <= to_logit;
                    }
                    in |= here ? 1u << i : 0u;
                }
                while (in != 0) {
                    const int i = __ffs(static_cast<int>(in)) - 1;
                    in &= in - 1;
                    const float l = Of::pick(v, i);
                    const int index = first + n * threads * each + i;
                    if (!kept.holds(l, index)) continue;
                    const unsigned key = key_of(l);
                    least = min(least, key), most = max(most, key);
                    gather(key, index, part);
                }
            });
            least = __reduce_min_sync(0xffffffffu, least), most = __reduce_max_sync(0xffffffffu, most);
            if (lane == 0) shared.sums.scratch[warp] = static_cast<Weight>(least) << 32 | most;
            __syncthreads();
            for (int w = 0; w < warps; ++w) {
                least = min(least, static_cast<unsigned>(shared.sums.scratch[w] >> 32));
                most = max(most, static_cast<unsigned>(shared.sums.scratch[w]));
            }
            if (threadIdx.x < static_cast<unsigned>(blocks)) {
                put(&shared.counts[0][rank], static_cast<int>(threadIdx.x), shared.count);
                put(&shared.sums_of[0][rank], static_cast<int>(threadIdx.x), static_cast<unsigned long long>(least) << 32 | most);
            }
            cluster_sync();
            bool fits = true;
            low = 0xffffffffu, high = 0;
            for (int b = 0; b < blocks; ++b) {
                fits = fits && shared.counts[0][b] <= static_cast<unsigned>(part);
                low = min(low, static_cast<unsigned>(shared.sums_of[0][b] >> 32));
                high = max(high, static_cast<unsigned>(shared.sums_of[0][b]));
            }
            if (fits) {
                if (rank == 0) {
                    const int n = collect(shared.counts[0], part);
                    constexpr int most_each = most_candidates / threads;
                    const int run = (n + threads - 1) / threads, from = static_cast<int>(threadIdx.x) * run;
                    Weight mine[most_each], sum = 0, all;
#pragma unroll
                    for (int i = 0; i < most_each; ++i) {
                        mine[i] = i >= run || from + i >= n ? 0
                            : by_weight ? weight_of(share_of(logit_of(static_cast<unsigned>(shared.sorted[from + i] >> 32)), row)) : 1;
                        sum += mine[i];
                    }
                    Weight earlier = before(sum, shared.sums.scratch, all);
#pragma unroll
                    for (int i = 0; i < most_each; ++i) {
                        if (mine[i] != 0 && earlier < wanted && earlier + mine[i] >= wanted) {
                            for (int b = 0; b < blocks; ++b) put(&shared.told[0], b, shared.sorted[from + i]);
                        }
                        earlier += mine[i];
                    }
                }
                break;
            }
            if (low == high) {
                const Weight one = by_weight ? weight_of(share_of(logit_of(low), row)) : 1;
                locate(
                    [&](int index, float l) { return static_cast<Weight>(key_of(l) == low && kept.holds(l, index)); },
                    [&](Weight) { return (wanted + one - 1) / one - 1; },
                    [&](int index, float l, Weight) {
                        for (int b = 0; b < blocks; ++b) {
                            put(&shared.told[0], b, static_cast<unsigned long long>(key_of(l)) << 32 | ~static_cast<unsigned>(index));
                        }
                    });
                break;
            }
            const int shift = max(0, 32 - __clz(high - low) - 11);
            const Weight still = wanted;
            const unsigned from = low, to = high;
            const int found = reach(
                row, by_weight, kept,
                [&](float l) {
                    const unsigned key = key_of(l);
                    return key >= from && key <= to ? static_cast<int>((to - key) >> shift) : -1;
                },
                [&](Weight) { return still; }, wanted);
            high = to - (static_cast<unsigned>(found) << shift);
            low = high - min(high - from, (1u << shift) - 1);
        }
        cluster_sync();
        const unsigned long long end = shared.told[0];
        __syncthreads();
        return {logit_of(static_cast<unsigned>(end >> 32)), static_cast<int>(~static_cast<unsigned>(end))};
    }

    // Any row of finite logits, exactly.
    __device__ __forceinline__ void whole(const Row& row, const Settings& s, float largest, float factor) {
        Kept kept{-INFINITY, INT_MAX};
        if (row.temperature == 0.0) {
            kept = {row.largest, INT_MAX};
        } else {
            if (s.top_k > 0 && s.top_k < a.symbols) kept = find(row, s, false, largest, factor, kept);
            if (s.top_p < 1.0f) kept = find(row, s, true, largest, factor, kept);
        }
        // with a temperature of 0, u is taken as 0: the first of the largest
        locate(
            [&](int index, float l) -> Weight {
                const double share = share_of(l, row);
                return kept.holds(l, index) && share >= row.least ? weight_of(share) : 0;
            },
            [&](Weight all) { return row.temperature == 0.0 ? 0 : part_of_uniform(s.uniform, all); },
            [&](int index, float l, Weight all) {
                a.chosen[r] = index;
                a.probabilities[r] = row.temperature == 0.0 ? 1.0f : probability_of(share_of(l, row), all);
            });
    }

    // As `finish`, for at most 64 symbols, by one warp: a fraction of the latency of a block's barriers.
    __device__ __forceinline__ bool finish_few(const Row& row, const Settings& s, const unsigned long long* counts, int part, int all_count,
                                               double bulk, double slack) {
        const int lane = threadIdx.x % 32;
        int filled = 0;
        for (int b = 0; b < blocks; ++b) {
            const int count = static_cast<int>(counts[b] & 0xffffffffu);
            for (int i = lane; i < count; i += 32) shared.weights[filled + i] = shared.gathered[b * part + i];
            filled += count;
        }
        for (int i = all_count + lane; i < 64; i += 32) shared.weights[i] = 0;
        __syncwarp();
        const unsigned long long one = shared.weights[lane], two = shared.weights[lane + 32];
        int place_one = 0, place_two = 0;
#pragma unroll 2
        for (int k = 0; k < all_count; ++k) {
            const unsigned long long other = shared.weights[k];
            place_one += other > one, place_two += other > two;
        }
        if (lane < all_count) shared.sorted[place_one] = one;
        if (lane + 32 < all_count) shared.sorted[place_two] = two;
        __syncwarp();
        int n = s.top_k > 0 ? min(all_count, s.top_k) : all_count;
        // a lane has two neighbours
        unsigned long long entry[2];
        Weight w[2], to[2], all = 0;
        unsigned kept = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool there = 2 * lane + i < n;
            entry[i] = there ? shared.sorted[2 * lane + i] : 0;
            const double share = there ? share_of(logit_of(static_cast<unsigned>(entry[i] >> 32)), row) : 0.0;
            w[i] = weight_of(share);
            kept += there && share >= row.least;
        }
        Weight sum = w[0] + w[1];
        for (int o = 1; o < 32; o *= 2) {
            const Weight v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        all = __shfl_sync(0xffffffffu, sum, 31);
        to[1] = sum, to[0] = sum - w[1];
        n = min(n, static_cast<int>(__reduce_add_sync(0xffffffffu, kept)));
        if (s.top_p < 1.0f) {
            const double p = static_cast<double>(fmaxf(s.top_p, 0.0f));
            const double least_part = p * (static_cast<double>(all) + bulk - slack), most_part = p * (static_cast<double>(all) + bulk + slack);
            unsigned low = 0, high = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                low += 2 * lane + i < n && static_cast<double>(to[i]) < least_part;
                high += 2 * lane + i < n && static_cast<double>(to[i]) < most_part;
            }
            low = __reduce_add_sync(0xffffffffu, low), high = __reduce_add_sync(0xffffffffu, high);
            if (min(n, 1 + static_cast<int>(low)) != min(n, 1 + static_cast<int>(high))) return false;
            n = min(n, 1 + static_cast<int>(low));
        }
        const Weight last = __shfl_sync(0xffffffffu, (n - 1) % 2 == 0 ? to[0] : to[1], (n - 1) / 2);
        const Weight wanted = part_of_uniform(s.uniform, last);
        shared.weights[2 * lane] = w[0], shared.weights[2 * lane + 1] = w[1];
        __syncwarp();
        Weight lower[2] = {0, 0};  // of those with lower indexes, whose complements are larger
#pragma unroll 2
        for (int k = 0; k < n; ++k) {
            const unsigned other = static_cast<unsigned>(shared.sorted[k]);
            const Weight weight = shared.weights[k];
#pragma unroll
            for (int i = 0; i < 2; ++i) lower[i] += other > static_cast<unsigned>(entry[i]) ? weight : 0;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (2 * lane + i < n && wanted >= lower[i] && wanted < lower[i] + w[i]) {
                a.chosen[r] = static_cast<std::int64_t>(~static_cast<unsigned>(entry[i]));
                a.probabilities[r] = probability_of(share_of(logit_of(static_cast<unsigned>(entry[i] >> 32)), row), last);
            }
        }
        return true;
    }

    // The first block: the symbols in `gathered` are all that can be kept. False where the choice hangs on the error of
    // `bulk`, the weight of the others.
    __device__ __forceinline__ bool finish(const Row& row, const Settings& s, const unsigned long long* counts, int part, double bulk,
                                           double slack) {
        if (threadIdx.x == 0) shared.kept = shared.low = shared.high = 0;
        int n = collect(counts, part);
        if (s.top_k > 0) n = min(n, s.top_k);
        const int run = (n + threads - 1) / threads, from = static_cast<int>(threadIdx.x) * run;
        const int until = min(n, from + run);
        Weight sum = 0, all;
        unsigned kept = 0;
#pragma unroll 1
        for (int i = from; i < until; ++i) {
            const double share = share_once(logit_of(static_cast<unsigned>(shared.sorted[i] >> 32)), row);
            const Weight w = weight_of(share);
            shared.weights[i] = w;
            kept += share >= row.least;
            sum += w;
        }
        Weight to = before(sum, shared.sums.scratch, all);
        double least_part = 0.0, most_part = 0.0;
        if (s.top_p < 1.0f) {
            const double p = static_cast<double>(fmaxf(s.top_p, 0.0f));
            least_part = p * (static_cast<double>(all) + bulk - slack), most_part = p * (static_cast<double>(all) + bulk + slack);
        }
        unsigned low = 0, high = 0;
#pragma unroll 1
        for (int i = from; i < until; ++i) {
            to += shared.weights[i];
            shared.weights[i] = to;
            low += static_cast<double>(to) < least_part;
            high += static_cast<double>(to) < most_part;
        }
        kept = __reduce_add_sync(0xffffffffu, kept);
        low = __reduce_add_sync(0xffffffffu, low), high = __reduce_add_sync(0xffffffffu, high);
        if (threadIdx.x % 32 == 0) {
            atomicAdd(&shared.kept, kept);
            atomicAdd(&shared.low, low);
            atomicAdd(&shared.high, high);
        }
        __syncthreads();
        n = min(n, static_cast<int>(shared.kept));
        if (s.top_p < 1.0f) {
            if (min(n, 1 + static_cast<int>(shared.low)) != min(n, 1 + static_cast<int>(shared.high))) return false;
            n = min(n, 1 + static_cast<int>(shared.low));
        }
        const Weight whole_kept = shared.weights[n - 1];
        const Weight wanted = part_of_uniform(s.uniform, whole_kept);
        auto choose = [&](unsigned long long entry) {
            a.chosen[r] = static_cast<std::int64_t>(~static_cast<unsigned>(entry));
            a.probabilities[r] = probability_of(share_once(logit_of(static_cast<unsigned>(entry >> 32)), row), whole_kept);
        };
        auto weight_at = [&](int i) { return shared.weights[i] - (i == 0 ? 0 : shared.weights[i - 1]); };
        if (n <= most_counted) {  // the weight of those with lower indexes, for each
            const int group = group_of(n), i = static_cast<int>(threadIdx.x) / group;
            const unsigned index = i < n ? static_cast<unsigned>(shared.sorted[i]) : 0;  // its complement
            Weight lower = 0;
            for (int k = static_cast<int>(threadIdx.x) % group; k < n; k += group) {
                lower += static_cast<unsigned>(shared.sorted[k]) > index ? weight_at(k) : 0;
            }
            for (int o = group / 2; o > 0; o /= 2) lower += __shfl_xor_sync(0xffffffffu, lower, o);
            if (i < n && threadIdx.x % group == 0 && wanted >= lower && wanted < lower + weight_at(i)) choose(shared.sorted[i]);
            return true;
        }
        // in the order of indexes: the largest complement first
        for (int i = threadIdx.x; i < n; i += threads) {
            shared.gathered[i] = (shared.sorted[i] & 0xffffffffull) << 32 | static_cast<unsigned>(i);
        }
        arrange(shared.gathered, n, max(0, 21 - __clz(max(a.symbols - 1, 1))), shared.sums);
        const int start = static_cast<int>(threadIdx.x) * run, stop = min(n, start + run);
        sum = 0;
#pragma unroll 1
        for (int i = start; i < stop; ++i) sum += weight_at(static_cast<int>(shared.gathered[i] & 0xffffffffull));
        to = before(sum, shared.sums.scratch, all);
#pragma unroll 1
        for (int i = start; i < stop; ++i) {
            const int at = static_cast<int>(shared.gathered[i] & 0xffffffffull);
            const Weight w = weight_at(at);
            if (wanted >= to && wanted < to + w) choose(shared.sorted[at]);
            to += w;
        }
        return true;
    }
};

template <typename T, int Vectors>
__global__ void __launch_bounds__(threads, Vectors == 8 ? 2 : 1) cluster_kernel(SampleArgs a, int blocks) {
    extern __shared__ unsigned char memory[];
    using Of = Elements<T>;
    constexpr int each = Of::each;
    auto& shared = *reinterpret_cast<Shared*>(memory);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int rank = static_cast<int>(blockIdx.x) % blocks;
    const std::int64_t r = blockIdx.x / blocks;
    cluster_arrive();  // the others' memory is there once all have
    make_table(shared.table);
    join_chain();
    const T* logits = static_cast<const T*>(a.logits) + r * a.stride;
    // Vectors begin on 16-byte boundaries, the first one up to 15 bytes before the row; this block has a run of them.
    const int skew = static_cast<int>(reinterpret_cast<std::uintptr_t>(logits) % 16 / sizeof(T));
    const int all_vectors = (a.symbols + skew + each - 1) / each;
    const int share = (all_vectors + blocks * threads - 1) / (blocks * threads);  // vectors a thread
    const int first = (rank * share * threads + static_cast<int>(threadIdx.x)) * each - skew;
    ClusterRow<T> of_cluster{a, shared, r, rank, blocks, share, first};
    uint4 v[Vectors];
    float most = -INFINITY;
#pragma unroll
    for (int k = 0; k < Vectors; ++k) v[k] = k < share ? of_cluster.load(k) : Of::none();
    const Settings s = settings_of(a, r);
#pragma unroll
    for (int k = 0; k < Vectors; ++k) most = fmaxf(most, Of::largest(v[k]));
    unsigned top = __reduce_max_sync(0xffffffffu, key_of(most));
    if (threadIdx.x == 0) shared.count = shared.queued = shared.wide = 0;
    if (lane == 0) shared.sums.scratch[warp] = top;
    __syncthreads();
    for (int w = 0; w < warps; ++w) top = max(top, static_cast<unsigned>(shared.sums.scratch[w]));
    cluster_wait();
    if (threadIdx.x < static_cast<unsigned>(blocks)) put(&shared.maxima[rank], static_cast<int>(threadIdx.x), top);
    cluster_sync();
    for (int b = 0; b < blocks; ++b) top = max(top, static_cast<unsigned>(shared.maxima[b]));
    if (top == 0) {  // nothing to choose
        if (rank == 0 && threadIdx.x == 0) a.chosen[r] = -1, a.probabilities[r] = 0.0f;
        return;
    }
    const Row row = row_of(top, s, shared.table);
    const bool by_count = s.top_k > 0 && s.top_k < a.symbols;
    const bool by_part = s.top_p < 1.0f;
    const float largest = logit_of(top);
    const float factor = 1.44269504f / s.temperature;  // octaves a logit
    const bool greedy = row.temperature == 0.0;
    if (!greedy && !(largest < INFINITY && factor < 1e30f && factor > 1e-30f)) {  // FP32 exponents
        if (rank == 0) row_by_block<T>(a, r, shared.sums, shared.table);
        return;
    }
    if (!greedy && (by_count || by_part || row.least > 0.0) && (!by_count || s.top_k <= most_candidates / 2) &&
        fabsf(largest * factor) < 1e4f) {
        // candidates: octaves from `cut` up; below -46 a weight rounds to none
        const int part = most_candidates / blocks;
        const bool sum_rest = by_part && !by_count;
        const float base = -largest * factor;
        auto exponent = [&](float l) { return fmaf(l, factor, base); };
        const double error = bulk_error(largest, factor);
        auto* queue = reinterpret_cast<uint4*>(shared.sorted);  // vectors with a candidate, in sorted and weights
        auto* places = reinterpret_cast<int*>(shared.sums.high);
        constexpr float wide_cut = -14.5f;
        float cut = -10.0f;
        const bool by_least = row.least > 0.0 && !(by_count && by_part);  // top_p's whole is that of the first top_k
        const float least_cut = by_least ? fmaxf(log2f(fminf(s.min_p, 1.0f)) - 0.01f, -46.0f) : -INFINITY;
        if (!by_count && by_least) {
            cut = least_cut;
        } else if (by_count) {
            // at which top_k vectors have their largest logits above: so many candidates at least, and seldom many more
            for (int i = threadIdx.x; i < cut_bins; i += threads) shared.sums.low[i] = 0;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < Vectors; ++k) {
                const float x = exponent(Of::largest(v[k])) * -cut_steps;
                if (x < static_cast<float>(cut_bins)) atomicAdd(&shared.sums.low[static_cast<int>(x)], 1u);
            }
            if (threadIdx.x == 0) shared.cut = cut_bins;
            cluster_sync();
            Weight mine = 0, all;
            if (threadIdx.x < cut_bins) {
                unsigned some[most_blocks];
#pragma unroll
                for (int b = 0; b < most_blocks; ++b) some[b] = get(&shared.sums.low[threadIdx.x], min(b, blocks - 1));
#pragma unroll
                for (int b = 0; b < most_blocks; ++b) mine += b < blocks ? some[b] : 0;
            }
            const Weight earlier = before(mine, shared.sums.scratch, all), wanted = static_cast<Weight>(s.top_k);
            if (earlier < wanted && earlier + mine >= wanted) shared.cut = static_cast<int>(threadIdx.x) + 1;
            __syncthreads();
            cut = fmaxf(static_cast<float>(shared.cut) * (-1.0f / cut_steps) - 0.001f, least_cut);
        }
        for (int turn = 0;; ++turn) {
            float held = 0.0f, rest = 0.0f;  // weights of candidates and of the others
            unsigned wide = 0;               // vectors with a candidate of the wider cut
#pragma unroll
            for (int k = 0; k < Vectors; ++k) {
                const float x = exponent(Of::largest(v[k]));
                wide += x >= wide_cut;
                if (x >= cut) {  // looked at below, by all threads
                    const unsigned nth = atomicAdd(&shared.queued, 1u);
                    if (nth < static_cast<unsigned>(part)) queue[nth] = v[k], places[nth] = first + k * threads * each;
                } else if (sum_rest) {
#pragma unroll
                    for (int i = 0; i < each; ++i) rest += exp2_fast(exponent(Of::get(v[k], i)));
                }
            }
            __syncthreads();
            const int queued = static_cast<int>(shared.queued);
            for (int e = threadIdx.x; e < min(queued, part) * each; e += threads) {
                const float l = Of::pick(queue[e / each], e % each), x = exponent(l);
                if (x >= cut) {
                    of_cluster.gather(key_of(l), places[e / each] + e % each, part);
                    held += exp2_fast(x);
                } else if (l == l) {
                    rest += exp2_fast(x);
                }
            }
            held = warp_sum(held), rest = warp_sum(rest);
            wide = __reduce_add_sync(0xffffffffu, wide);
            if (lane == 0) shared.parts[0][warp] = held, shared.parts[1][warp] = rest, atomicAdd(&shared.wide, wide);
            __syncthreads();
            held = rest = 0.0f;
            for (int w = 0; w < warps; ++w) held += shared.parts[0][w], rest += shared.parts[1][w];
            const int parity = turn & 1;
            if (threadIdx.x < static_cast<unsigned>(blocks)) {
                put(&shared.counts[parity][rank], static_cast<int>(threadIdx.x),
                    static_cast<unsigned long long>(shared.wide) << 32 | max(shared.count, shared.queued));
                put(&shared.sums_of[parity][rank], static_cast<int>(threadIdx.x),
                    static_cast<unsigned long long>(__float_as_uint(held)) << 32 | __float_as_uint(rest));
            }
            __syncthreads();
            if (threadIdx.x == 0) shared.count = shared.queued = shared.wide = 0;
            cluster_sync();
            int count = 0;
            bool fits = true, wide_fits = true;
            double all_held = 0.0, bulk = 0.0;
            for (int b = 0; b < blocks; ++b) {
                const int some = static_cast<int>(shared.counts[parity][b] & 0xffffffffu);
                fits = fits && some <= part;
                wide_fits = wide_fits && shared.counts[parity][b] >> 32 <= static_cast<unsigned long long>(part);
                count += some;
                const unsigned long long both = shared.sums_of[parity][b];
                all_held += __uint_as_float(static_cast<unsigned>(both >> 32)), bulk += __uint_as_float(static_cast<unsigned>(both));
            }
            if (!fits || !(bulk <= 1e30)) break;  // a NaN among the sums too
            const bool complete = cut <= -46.0f;  // what is left out has no weight
            const bool enough = complete || cut == least_cut ||
                (by_count ? count >= s.top_k
                          : all_held * (1.0 - error) >= static_cast<double>(fmaxf(s.top_p, 0.0f)) *
                                 ((all_held + bulk) * (1.0 + error) + a.symbols / unit));
            if (enough) {
                if (rank != 0) return;
                const double others = sum_rest ? bulk * unit : 0.0, slack = sum_rest ? others * error + a.symbols : 0.0;
                bool done;
                if (count <= 64) {
                    if (warp == 0) {
                        done = of_cluster.finish_few(row, s, shared.counts[parity], part, count, others, slack);
                        if (lane == 0) shared.queued = done;
                    }
                    __syncthreads();
                    done = shared.queued != 0;
                } else {
                    done = of_cluster.finish(row, s, shared.counts[parity], part, others, slack);
                    __syncthreads();
                }
                if (!done) row_by_block<T>(a, r, shared.sums, shared.table);
                return;
            }
            if (cut < -14.0f || !wide_fits) break;
            cut = wide_cut;
        }
    }
    of_cluster.whole(row, s, largest, factor);
    cluster_sync();  // no block ends while another one reads its memory
}

// ---- many rows ----

// Two FP32 values in one instruction.
struct Two {
    unsigned long long bits;
    __device__ __forceinline__ Two(float one, float two) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(one), "f"(two)); }
    __device__ __forceinline__ void add(const Two& v) { asm("add.rn.f32x2 %0, %0, %1;" : "+l"(bits) : "l"(v.bits)); }
    __device__ __forceinline__ Two by(const Two& factor, const Two& more) const {
        Two made(*this);
        asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(made.bits) : "l"(bits), "l"(factor.bits), "l"(more.bits));
        return made;
    }
    __device__ __forceinline__ float2 values() const {
        float2 v;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(bits));
        return v;
    }
};

constexpr int part_threads = 256;
constexpr int part_vectors = 8;    // a thread
constexpr int part_candidates = 2048;

// What `part_kernel` tells of a part of a row.
struct Part {
    unsigned top;    // the largest key
    float cut;       // the least logit of its candidates
    unsigned count;  // of them; past part_candidates some are missing
    float rest;      // the others' weights, the part's largest one's as one
};

struct ManyArgs {
    int parts;  // a row
    Part* told;
    unsigned long long* candidates;  // [row][part][part_candidates]: a key and the complement of an index
    unsigned* left;                  // how many rows `end_kernel` has left, and which
};

// What a row's settings ask for, the largest logit known.
struct Wishes {
    bool greedy, by_count, by_part;
    bool by_least;  // min_p tells the candidates; not where top_p's whole is that of the first top_k
    int top_k;
    float factor;  // octaves a logit
    bool ordinary; // FP32 exponents will do
    bool few;      // candidates can be told
    __device__ __forceinline__ float least_octaves(const Settings& s) const {
        return fmaxf(log2f(fminf(s.min_p, 1.0f)) - 0.01f, -46.0f);
    }
};
__device__ __forceinline__ Wishes wishes_of(const SampleArgs& a, const Settings& s, float largest) {
    Wishes w;
    w.greedy = !(s.temperature > 0.0f);
    w.top_k = w.greedy ? 1 : s.top_k;
    w.by_count = w.greedy || (s.top_k > 0 && s.top_k < a.symbols);
    w.by_part = !w.greedy && s.top_p < 1.0f;
    w.by_least = !w.greedy && s.min_p > 0.0f && !(w.by_count && w.by_part);
    w.factor = w.greedy ? 1.0f : 1.44269504f / s.temperature;
    w.ordinary = largest < INFINITY && w.factor < 1e30f && w.factor > 1e-30f;
    w.few = w.ordinary && (w.by_count || w.by_part || s.min_p > 0.0f) && (!w.by_count || w.top_k <= part_candidates / 2) &&
        fabsf(largest * w.factor) < 1e4f;
    return w;
}

// A part of a row: its largest logit, its candidates (a cut below its own largest, so those below the row's largest are
// among them) and the sum of the others' weights.
template <typename T>
__global__ void __launch_bounds__(part_threads, 4) part_kernel(SampleArgs a, ManyArgs m) {
    using Of = Elements<T>;
    constexpr int each = Of::each, warps_here = part_threads / 32;
    __shared__ uint4 queue[part_candidates];
    __shared__ int places[part_candidates];
    __shared__ unsigned bins_here[cut_bins], scratch[warps_here];
    __shared__ float sums_here[warps_here];
    __shared__ unsigned count, queued;
    __shared__ int cut_bin;
    join_chain();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const std::int64_t r = blockIdx.x / m.parts;
    const int part = static_cast<int>(blockIdx.x - r * m.parts);
    if (blockIdx.x == 0 && threadIdx.x == 0) *m.left = 0;
    const T* logits = static_cast<const T*>(a.logits) + r * a.stride;
    const int skew = static_cast<int>(reinterpret_cast<std::uintptr_t>(logits) % 16 / sizeof(T));
    const int first = (part * part_vectors * part_threads + static_cast<int>(threadIdx.x)) * each - skew;
    uint4 v[part_vectors];
    const int block_first = part * part_vectors * part_threads * each - skew;
    if (block_first >= 0 && block_first + part_vectors * part_threads * each <= a.symbols) {
        const auto* from = reinterpret_cast<const uint4*>(logits + first);
#pragma unroll
        for (int k = 0; k < part_vectors; ++k) v[k] = from[k * part_threads];
    } else {
#pragma unroll
        for (int k = 0; k < part_vectors; ++k) v[k] = load_vector(logits, a.symbols, first + k * part_threads * each);
    }
    const Settings s = settings_of(a, r);
    float of_vector[part_vectors], most = -INFINITY;
#pragma unroll
    for (int k = 0; k < part_vectors; ++k) of_vector[k] = Of::largest(v[k]), most = fmaxf(most, of_vector[k]);
    unsigned top = __reduce_max_sync(0xffffffffu, key_of(most));
    if (threadIdx.x == 0) count = queued = 0, cut_bin = cut_bins;
    if (lane == 0) scratch[warp] = top;
    if (threadIdx.x < cut_bins) bins_here[threadIdx.x] = 0;
    static_assert(cut_bins <= part_threads);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < warps_here; ++w) top = max(top, scratch[w]);
    const float largest = top == 0 ? -INFINITY : logit_of(top);
    const Wishes wishes = wishes_of(a, s, largest);
    Part told{top, INFINITY, 0, 0.0f};
    if (top != 0 && wishes.few) {
        const float base = -largest * wishes.factor;
        auto exponent = [&](float l) { return fmaf(l, wishes.factor, base); };
        float octaves = wishes.by_least ? wishes.least_octaves(s) : -10.0f;
        if (wishes.by_count && !wishes.greedy) {
            // at which top_k vectors have their largest logits above: so many candidates at least, and seldom many more
#pragma unroll
            for (int k = 0; k < part_vectors; ++k) {
                const float x = exponent(of_vector[k]) * -cut_steps;
                if (x < static_cast<float>(cut_bins)) atomicAdd(&bins_here[static_cast<int>(x)], 1u);
            }
            __syncthreads();
            if (warp == 0) {  // a lane eight bins
                unsigned mine[cut_bins / 32], sum = 0;
#pragma unroll
                for (int i = 0; i < cut_bins / 32; ++i) sum += mine[i] = bins_here[lane * (cut_bins / 32) + i];
                unsigned to = sum;
                for (int o = 1; o < 32; o *= 2) {
                    const unsigned u = __shfl_up_sync(0xffffffffu, to, o);
                    if (lane >= o) to += u;
                }
                unsigned earlier = to - sum;
                // a part's share of the row's, and half as many again: where that is too few, the row is left
                const auto wanted = static_cast<unsigned>(min(wishes.top_k, 3 * wishes.top_k / (2 * m.parts) + 32));
#pragma unroll
                for (int i = 0; i < cut_bins / 32; ++i) {
                    if (earlier < wanted && earlier + mine[i] >= wanted) cut_bin = lane * (cut_bins / 32) + i + 1;
                    earlier += mine[i];
                }
            }
            __syncthreads();
            const float by_count = static_cast<float>(cut_bin) * (-1.0f / cut_steps) - 0.01f;
            octaves = wishes.by_least ? fmaxf(octaves, by_count) : by_count;
        }
        told.cut = wishes.greedy ? largest : largest + octaves / wishes.factor;
        const bool sum_rest = wishes.by_part && !wishes.by_count;
        const Two factors(wishes.factor, wishes.factor), bases(base, base);
        Two sums(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < part_vectors; ++k) {
            if (of_vector[k] >= told.cut) {  // looked at below, by all threads
                const unsigned nth = atomicAdd(&queued, 1u);
                if (nth < part_candidates) queue[nth] = v[k], places[nth] = first + k * part_threads * each;
            } else if (sum_rest) {
#pragma unroll
                for (int i = 0; i < each; i += 2) {
                    const float2 x = Two(Of::get(v[k], i), Of::get(v[k], i + 1)).by(factors, bases).values();
                    sums.add(Two(exp2_fast(x.x), exp2_fast(x.y)));
                }
            }
        }
        float rest = sums.values().x + sums.values().y;
        __syncthreads();
        unsigned long long* list = m.candidates + (r * m.parts + part) * part_candidates;
        const int all = static_cast<int>(min(queued, static_cast<unsigned>(part_candidates))) * each;
        for (int e = threadIdx.x; e < all; e += part_threads) {
            const float l = Of::pick(queue[e / each], e % each);
            if (l >= told.cut) {
                const unsigned nth = atomicAdd(&count, 1u);
                if (nth < part_candidates) {
                    list[nth] = static_cast<unsigned long long>(key_of(l)) << 32 | ~static_cast<unsigned>(places[e / each] + e % each);
                }
            } else if (l == l) {
                rest += exp2_fast(exponent(l));
            }
        }
        rest = warp_sum(rest);
        if (lane == 0) sums_here[warp] = rest;
        __syncthreads();
        for (int w = 0; w < warps_here; ++w) told.rest += sums_here[w];
        told.count = queued > part_candidates ? queued : count;
    }
    if (threadIdx.x == 0) m.told[r * m.parts + part] = told;
}

// A block a row: its candidates of all parts, those above the highest cut, in which nothing is missing.
template <typename T>
__global__ void __launch_bounds__(threads, 2) end_kernel(SampleArgs a, ManyArgs m) {
    extern __shared__ unsigned char memory[];
    auto& shared = *reinterpret_cast<Shared*>(memory);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    make_table(shared.table);
    if (threadIdx.x == 0) shared.count = 0;
    join_chain();
    const std::int64_t r = blockIdx.x;
    const Part* told = m.told + r * m.parts;
    const Settings s = settings_of(a, r);
    unsigned top = 0;
    float cut = -INFINITY;
    bool whole = true;
    for (int p = lane; p < m.parts; p += 32) {
        const Part part = told[p];
        top = max(top, part.top);
        if (part.top != 0) cut = fmaxf(cut, part.cut);
        whole = whole && part.count <= part_candidates;
    }
    top = __reduce_max_sync(0xffffffffu, top);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) cut = fmaxf(cut, __shfl_xor_sync(0xffffffffu, cut, o));
    whole = __all_sync(0xffffffffu, whole);
    if (top == 0) {  // nothing to choose
        if (threadIdx.x == 0) a.chosen[r] = -1, a.probabilities[r] = 0.0f;
        return;
    }
    const float largest = logit_of(top);
    const Wishes wishes = wishes_of(a, s, largest);
    const Row row = row_of(top, s, shared.table);
    bool done = false;
    if (whole && wishes.few && cut < INFINITY) {  // a part whose largest is not ordinary has an infinite cut
        const float base = -largest * wishes.factor;
        auto exponent = [&](float l) { return fmaf(l, wishes.factor, base); };
        double bulk = 0.0;
        for (int p = lane; p < m.parts; p += 32) {
            const Part part = told[p];
            if (part.top != 0) bulk += static_cast<double>(part.rest) * exp2_fast(exponent(logit_of(part.top)));
        }
#pragma unroll
        for (int o = 16; o > 0; o /= 2) bulk += __shfl_xor_sync(0xffffffffu, bulk, o);
        __syncthreads();
        // a part by one warp, or by as many as there are for each
        double held_here = 0.0, rest_here = 0.0;
        const int sharing = max(1, warps / m.parts);
        for (int p = warp / sharing; p < m.parts; p += warps / sharing) {
            const int count = static_cast<int>(told[p].count);
            const unsigned long long* list = m.candidates + (r * m.parts + p) * part_candidates;
            float held = 0.0f, rest = 0.0f;
            for (int from = warp % sharing * 128; from < count; from += sharing * 128) {
                unsigned long long entry[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = from + k * 32 + lane;
                    entry[k] = i < count ? list[i] : 0;
                }
#pragma unroll 1
                for (int k = 0; k < 4; ++k) {
                    const unsigned long long one = k == 0 ? entry[0] : k == 1 ? entry[1] : k == 2 ? entry[2] : entry[3];
                    if (one == 0) break;
                    const float l = logit_of(static_cast<unsigned>(one >> 32));
                    if (l >= cut) {
                        const unsigned nth = atomicAdd(&shared.count, 1u);
                        if (nth < most_candidates) shared.gathered[nth] = one;
                        held += exp2_fast(exponent(l));
                    } else {
                        rest += exp2_fast(exponent(l));
                    }
                }
            }
            held_here += held, rest_here += rest;
        }
        const float held = warp_sum(static_cast<float>(held_here)), rest = warp_sum(static_cast<float>(rest_here));
        if (lane == 0) shared.parts[0][warp] = held, shared.parts[1][warp] = rest;
        __syncthreads();
        double all_held = 0.0;
        for (int w = 0; w < warps; ++w) all_held += shared.parts[0][w], bulk += shared.parts[1][w];
        const int count = static_cast<int>(shared.count);
        const bool sum_rest = wishes.by_part && !wishes.by_count;
        // exponents in two steps, each with a rounding of its own largest logit's
        const double error = 2.0 * bulk_error(largest, wishes.factor);
        const bool enough = count <= most_candidates && bulk <= 1e30 &&
            ((wishes.by_least && cut == largest + wishes.least_octaves(s) / wishes.factor) ||
             (wishes.by_count ? count >= wishes.top_k
                              : all_held * (1.0 - error) >= static_cast<double>(fmaxf(s.top_p, 0.0f)) *
                                      ((all_held + bulk) * (1.0 + error) + a.symbols / unit)));
        if (enough) {
            if (threadIdx.x == 0) shared.counts[0][0] = static_cast<unsigned long long>(count);
            __syncthreads();
            Settings set = s;
            if (wishes.greedy) set.top_k = 1, set.top_p = 1.0f, set.min_p = 0.0f;
            const double others = sum_rest ? bulk * unit : 0.0, slack = sum_rest ? others * error + a.symbols : 0.0;
            ClusterRow<T> one{a, shared, r, 0, 1, 0, 0};
            if (count <= 64) {
                if (warp == 0) {
                    done = one.finish_few(row, set, shared.counts[0], most_candidates, count, others, slack);
                    if (lane == 0) shared.queued = done;
                }
                __syncthreads();
                done = shared.queued != 0;
            } else {
                done = one.finish(row, set, shared.counts[0], most_candidates, others, slack);
            }
        }
    }
    if (!done && threadIdx.x == 0) m.left[1 + atomicAdd(m.left, 1u)] = static_cast<unsigned>(r);
}

// The rows that are left, a cluster each.
template <typename T>
__global__ void __launch_bounds__(threads, 2) rest_kernel(SampleArgs a, ManyArgs m, int blocks) {
    extern __shared__ unsigned char memory[];
    constexpr int each = Elements<T>::each;
    auto& shared = *reinterpret_cast<Shared*>(memory);
    const int lane = threadIdx.x % 32;
    const int rank = static_cast<int>(blockIdx.x) % blocks;
    join_chain();
    const unsigned count = *m.left;
    if (count == 0) return;
    cluster_arrive();  // the others' memory is there once all have
    make_table(shared.table);
    cluster_wait();
    __syncthreads();
    for (unsigned nth = blockIdx.x / blocks; nth < count; nth += gridDim.x / blocks) {
        const std::int64_t r = m.left[1 + nth];
        const T* logits = static_cast<const T*>(a.logits) + r * a.stride;
        const int skew = static_cast<int>(reinterpret_cast<std::uintptr_t>(logits) % 16 / sizeof(T));
        const int all_vectors = (a.symbols + skew + each - 1) / each;
        const int share = (all_vectors + blocks * threads - 1) / (blocks * threads);
        ClusterRow<T> of_cluster{a, shared, r, rank, blocks, share, (rank * share * threads + static_cast<int>(threadIdx.x)) * each - skew};
        const Settings s = settings_of(a, r);
        unsigned top = 0;
        for (int p = lane; p < m.parts; p += 32) top = max(top, m.told[r * m.parts + p].top);
        top = __reduce_max_sync(0xffffffffu, top);
        const Row row = row_of(top, s, shared.table);
        const float largest = logit_of(top), factor = 1.44269504f / s.temperature;
        if (row.temperature != 0.0 && !(largest < INFINITY && factor < 1e30f && factor > 1e-30f)) {
            if (rank == 0) row_by_block<T>(a, r, shared.sums, shared.table);
        } else {
            of_cluster.whole(row, s, largest, factor);
        }
        cluster_sync();  // before the next row, or the end, while another block reads this one's memory
    }
}

template <typename T, int Vectors>
cudaError_t launch_cluster(const SampleArgs& a, int blocks, cudaStream_t stream) {
    static SharedAllowance allowance;
    const cudaError_t status = allowance.allow(cluster_kernel<T, Vectors>, sizeof(Shared));
    if (status != cudaSuccess) return status;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(a.rows * blocks));
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = sizeof(Shared);
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = static_cast<unsigned>(blocks);
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, cluster_kernel<T, Vectors>, a, blocks);
}

int parts_of(Type type, int symbols) {
    const int part = part_threads * part_vectors * (type == Type::f32 ? 4 : 8);
    return (symbols + 7 + part - 1) / part;  // a row may begin within a vector
}
int parts_of(const SampleArgs& a) {
    const int each = a.type == Type::f32 ? 4 : 8, part = part_threads * part_vectors * each;
    const bool whole = reinterpret_cast<std::uintptr_t>(a.logits) % 16 == 0 && a.stride % each == 0;
    return whole ? (a.symbols + part - 1) / part : parts_of(a.type, a.symbols);
}
std::size_t rounded(std::size_t bytes) { return (bytes + 255) / 256 * 256; }
// Blocks of a cluster that has a row in its registers.
int blocks_of(Type type, int symbols) {
    const int held = threads * 8 * (type == Type::f32 ? 4 : 8);
    int blocks = 1;
    while (blocks < most_blocks && blocks * held < symbols) blocks *= 2;
    return blocks;
}
bool many_rows(Type type, std::int64_t rows, int symbols) {
    return blocks_of(type, symbols) > 1 && rows * blocks_of(type, symbols) > 2 * sm_count() &&
        symbols + 7 <= most_vectors * 4 * threads * most_blocks &&  // what a cluster's threads have
        rows <= INT_MAX / parts_of(type, symbols);
}

template <typename T>
cudaError_t launch_many(const SampleArgs& a, cudaStream_t stream) {
    static SharedAllowance end_allowance, rest_allowance;
    cudaError_t status = end_allowance.allow(end_kernel<T>, sizeof(Shared));
    if (status == cudaSuccess) status = rest_allowance.allow(rest_kernel<T>, sizeof(Shared));
    if (status != cudaSuccess) return status;
    ManyArgs m{};
    m.parts = parts_of(a);
    const std::size_t parts = static_cast<std::size_t>(a.rows) * m.parts;
    auto* memory = static_cast<unsigned char*>(a.workspace);
    m.told = reinterpret_cast<Part*>(memory);
    m.candidates = reinterpret_cast<unsigned long long*>(memory + rounded(parts * sizeof(Part)));
    m.left = reinterpret_cast<unsigned*>(memory + rounded(parts * sizeof(Part)) + parts * part_candidates * 8);
    status = kernels::launch_overlapped(part_kernel<T>, dim3(static_cast<unsigned>(parts)), dim3(part_threads), 0, stream, a, m);
    if (status != cudaSuccess) return status;
    status = kernels::launch_overlapped(end_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(threads), sizeof(Shared), stream, a, m);
    if (status != cudaSuccess) return status;
    const int blocks = blocks_of(a.type, a.symbols);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(std::min<std::int64_t>(a.rows, 2 * sm_count() / blocks) * blocks));
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = sizeof(Shared);
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = static_cast<unsigned>(blocks);
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, rest_kernel<T>, a, m, blocks);
}

template <typename T>
cudaError_t launch(const SampleArgs& a, cudaStream_t stream) {
    if (many_rows(a.type, a.rows, a.symbols)) return launch_many<T>(a, stream);
    constexpr int each = 16 / sizeof(T);
    const bool aligned = reinterpret_cast<std::uintptr_t>(a.logits) % 16 == 0 && (a.rows == 1 || a.stride % each == 0);
    const int vectors = (a.symbols + each - 1) / each + (aligned ? 0 : 1);  // a row may begin within one
    auto fits = [&](int blocks, int held) { return vectors <= blocks * threads * held; };
    int blocks = 1;
    while (blocks < most_blocks && !fits(blocks, 8)) blocks *= 2;
    // few rows: while all blocks run at once and each has two vectors a thread
    while (blocks < most_blocks && a.rows * blocks * 2 <= sm_count() && vectors > blocks * threads * 2) blocks *= 2;

    if (a.rows > INT_MAX / most_blocks) blocks = 0;  // more blocks than a grid holds
    if (fits(blocks, 8)) return launch_cluster<T, 8>(a, blocks, stream);
    if (fits(blocks, 16)) return launch_cluster<T, 16>(a, blocks, stream);
    return kernels::launch_overlapped(block_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(threads), 0, stream, a);
}

}  // namespace

std::size_t sample_workspace(Type type, std::int64_t rows, int symbols) {
    if (!many_rows(type, rows, symbols)) return 0;
    const std::size_t parts = static_cast<std::size_t>(rows) * parts_of(type, symbols);
    return rounded(parts * sizeof(Part)) + parts * part_candidates * 8 + rounded((static_cast<std::size_t>(rows) + 1) * sizeof(unsigned));
}

cudaError_t sample(const SampleArgs& a, cudaStream_t stream) {
    if (a.rows == 0) return cudaSuccess;
    switch (a.type) {
    case Type::f16: return launch<__half>(a, stream);
    case Type::bf16: return launch<__nv_bfloat16>(a, stream);
    default: return launch<float>(a, stream);
    }
}

}  // namespace nvcr_sm100::token
