// Attention of new tokens over the paged 4-bit cache. Token i of a sequence's
// count new ones is at position length - count + i and sees the keys up to its
// own position; one that sees none gives zeros. Grouped heads: query head h
// reads cache head h / (heads / kv_heads).
//
// The codes are never expanded to values. With s, m a group's scale and minimum,
//   score = sum_g s_g (q_g . c_g) + m_g sum(q_g),
//   out_d = sum_t (p_t s_tg) (c_td - 7.5) + sum_t p_t (m_tg + 7.5 s_tg),
// so both products run on the codes themselves: a nibble masked out of its
// place in a 16-bit half is the FP16 number c 2^-24 or, four bits up, c 2^-20
// (subnormal, exact in the tensor cores), and the powers of two are taken out
// with the scales. Five integer instructions give eight codes of an operand.
// Keys and transposed values are the 16-row operand of mma.m16n8k16, the query
// rows that share a cache head (grouped heads times new tokens) its 8 columns:
// a step's work is a cache read of 4.5 bits a value against one or two such
// columns, so what bounds it is HBM and the conversion, not the tensor pipe,
// and the warp-level instruction leaves codes, scores and weights in registers.
// Queries are scaled by a power of two per row into FP16's range (exact but for
// channels 2^-35 of the row's largest); weights p s are rounded to FP16
// after scaling to the group's largest scale so far, as a 16-bit operand must.
// Their rounding then weighs on c - 7.5, not on c: the 7.5 is taken out with a
// product of the same rounded weights with ones, and put back in FP32 with the
// minimums. Scores, softmax statistics and sums are FP32.
//
// One block takes one cache head, 8 or 16 query rows and a range of the
// length; each warp streams its own tiles of 16 or 32 keys through a ring in
// shared memory (cp.async, three stages, chunks XOR-swizzled so that the
// fragment reads touch every bank once) and keeps its own running maximum and
// sum. The warps' results are joined in shared memory; ranges of one sequence
// in the context's workspace by the last block to finish, in the ranges' order.
#include "token_elements.cuh"

#include <algorithm>
#include <cfloat>

namespace nvcr_sm100::token {
namespace {

constexpr int warps = 8;
constexpr int stages = 3;
constexpr float log2_e = 1.4426950408889634f;
// A running maximum is raised only when a score passes it by this much (in
// powers of two): weights stay below 2^8, and few tiles rescale their sums.
constexpr float top_slack = 8.0f;

__device__ __forceinline__ void note(const Cache& cache, unsigned bit) {
    if (cache.status != nullptr) atomicOr(cache.status, bit);
}

__device__ __forceinline__ void copy_async(unsigned shared, const void* global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
}

__device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ unsigned pack_half(float low, float high) {
    const __half2 v = __floats2half2_rn(low, high);
    return reinterpret_cast<const unsigned&>(v);
}

__device__ __forceinline__ float2 pair_at(const std::uint8_t* scales, int byte) {
    return __half22float2(*reinterpret_cast<const __half2*>(scales + byte));
}

// n / d for n < 2^31 as (umulhi(n, multiplier) + n) >> shift (Granlund and
// Montgomery's division by an invariant).
struct Divisor {
    unsigned multiplier, shift;
};

struct Work {
    Cache cache;
    AttendArgs a;
    Divisor tiles_per_page;  // of the index of a run of 16 places
    int ratio;               // query heads of a cache head
    int row_blocks;
    int range;               // places a block covers
    int ranges;
    float* partials;         // [block of rows][range][rows][D + 2]
    unsigned* tickets;       // [block of rows], zero between calls
    bool aligned;            // queries can be read 16 bytes at a time
};

// Fragment row r of a run of 8 keys holds key row_key(r): with it the four keys
// that a value fragment reads at once lie in different rows of banks.
__device__ __forceinline__ int row_key(int r) { return (r & 4) | (r & 1) << 1 | (r & 2) >> 1; }

// XOR of the 16-byte chunk index of key t's row of D / 2 bytes.
template <int D>
__device__ __forceinline__ int swizzle(int t) {
    if (D == 64) return t >> 2 & 1;
    if (D == 128) return ((t >> 1 ^ t >> 2) & 1) << 1 | (t >> 2 & 1);
    return (t & 1) << 1 | ((t >> 1 ^ t >> 2) & 1) << 2;
}

template <int D>
constexpr int tile_keys = D == 256 ? 16 : 32;

template <int D, int G>
constexpr int stage_bytes = tile_keys<D> * (D + 8 * (D / G));

template <int D, int G, int NT>
constexpr int shared_bytes = std::max(warps * stages * stage_bytes<D, G>, warps * 8 * NT * (D + 4) * 4);

template <typename T, int D, int G, int NT>
__global__ void __launch_bounds__(32 * warps) attend_kernel(const Work work) {
    constexpr int groups = D / G, rows = 8 * NT, keys = tile_keys<D>, runs = keys / 16;
    constexpr int row_bytes = D / 2, chunks = row_bytes / 16;
    constexpr int words = G / 32;  // 32-bit words of codes a lane holds of a group of one key
    constexpr int tiles = G / 16;  // 16-channel tiles of a group
    extern __shared__ __align__(128) std::uint8_t shared[];
    __shared__ float joint_top[warps][rows], joint_sum[warps][rows];
    __shared__ bool joint_last;
    const Cache& cache = work.cache;
    const AttendArgs& a = work.a;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = lane / 4, j = lane % 4;
    const int range = blockIdx.x, row_block = blockIdx.y % work.row_blocks, kv_head = blockIdx.y / work.row_blocks;
    const int sequence = blockIdx.z;

    // ---- what this block has to do ----
    std::int64_t first = sequence, last = sequence + 1;
    if (a.query_offsets != nullptr) first = a.query_offsets[sequence], last = a.query_offsets[sequence + 1];
    int length = a.lengths[sequence];
    const std::int64_t count64 = last - first;
    if (first < 0 || last > a.tokens || count64 < 0 || count64 > a.max_queries) {
        if (threadIdx.x == 0) note(cache, status_length);
        return;
    }
    const int count = static_cast<int>(count64);
    const int first_row = row_block * rows, total_rows = count * work.ratio;
    if (first_row >= total_rows) return;
    if (length < 0 || length > a.max_length) {
        if (threadIdx.x == 0) note(cache, status_length);
        length = length < 0 ? 0 : a.max_length;
    }
    const int used_rows = min(rows, total_rows - first_row);
    const int visible_first = max(0, length - count + first_row / work.ratio + 1);  // of the block's first row
    const int visible_last = max(0, length - count + (first_row + used_rows - 1) / work.ratio + 1);
    const int begin = range * work.range;
    const int active = max(1, (visible_last + work.range - 1) / work.range);  // ranges that hold anything
    if (range >= active) return;
    const int end = min(visible_last, begin + work.range);

    // ---- the ring ----
    const unsigned ring = static_cast<unsigned>(__cvta_generic_to_shared(shared)) + warp * stages * stage_bytes<D, G>;
    const std::uint8_t* const ring_bytes = shared + warp * stages * stage_bytes<D, G>;
    const std::int32_t* const table = a.page_table + sequence * a.table_stride;
    auto page_of = [&](int place) {  // of a run of 16 places; 0 past the end
        if (place >= end) return 0;
        const unsigned index = static_cast<unsigned>(place) / 16;
        return table[(__umulhi(index, work.tiles_per_page.multiplier) + index) >> work.tiles_per_page.shift];
    };
    int page[runs];
    unsigned bad = 0;  // bit stage * runs + run: a run of places without a page
    auto fetch_pages = [&](int tile) {
#pragma unroll
        for (int u = 0; u < runs; ++u) page[u] = page_of(begin + tile * keys + 16 * u);
    };
    const int tile_count = (end - begin + keys - 1) / keys;
    // Copies a tile whose pages are fetched; lays codes out as [key][chunk ^ swizzle] and scales as [key][group].
    auto issue = [&](int tile, int stage) {
#pragma unroll
        for (int u = 0; u < runs; ++u) {
            const int place = begin + tile * keys + 16 * u;
            const bool good = page[u] >= 0 && page[u] < cache.pages;
            if (!good && lane == 0) note(cache, status_page);
            const unsigned bit = 1u << (stage * runs + u);
            bad = good ? bad & ~bit : bad | bit;
            if (place >= end || !good) continue;
            const unsigned index = static_cast<unsigned>(place) / 16;
            const unsigned whole = (__umulhi(index, work.tiles_per_page.multiplier) + index) >> work.tiles_per_page.shift;
            const int within = place - static_cast<int>(whole) * cache.page_size;
            const std::int64_t at =
                (static_cast<std::int64_t>(page[u]) * cache.kv_heads + kv_head) * cache.page_size + within;
            const unsigned to = ring + stage * stage_bytes<D, G>;
            const std::uint8_t* key_codes = cache.key_codes + at * row_bytes;
            const std::uint8_t* value_codes = cache.value_codes + at * row_bytes;
#pragma unroll
            for (int i = 0; i < 16 * chunks / 32; ++i) {
                const int chunk = lane + 32 * i, key = chunk / chunks;
                const unsigned place_in = (16 * u + key) * row_bytes + ((chunk % chunks) ^ swizzle<D>(key & 7)) * 16;
                copy_async(to + place_in, key_codes + chunk * 16);
                copy_async(to + keys * row_bytes + place_in, value_codes + chunk * 16);
            }
            if (lane < 8 * groups) {  // 4 * groups chunks of scales for keys, as many for values
                const bool value = lane >= 4 * groups;
                const int chunk = value ? lane - 4 * groups : lane;
                const std::uint8_t* scales = reinterpret_cast<const std::uint8_t*>(value ? cache.value_scales : cache.key_scales);
                copy_async(to + keys * D + (value ? keys * 4 * groups : 0) + u * 64 * groups + chunk * 16,
                           scales + at * (4 * groups) + chunk * 16);
            }
        }
    };
    int next = warp;  // the next tile to copy
    fetch_pages(next);
#pragma unroll
    for (int s = 0; s < stages - 1; ++s) {
        if (next < tile_count) {
            issue(next, s);
            next += warps;
            fetch_pages(next);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // ---- the queries, as fragments: lane (r, j) holds row r, channels j * G / 4 .. of each group ----
    unsigned query[groups][words][2][2][NT];
    float query_sum[groups][NT][2], factor[NT][2];
    int visible[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int row = first_row + 8 * n + r;
        const bool used = row < total_rows;
        float q[groups][8 * words];
        const T* source = static_cast<const T*>(a.queries) +
            (first + (used ? row / work.ratio : 0)) * a.query_stride +
            (kv_head * work.ratio + (used ? row % work.ratio : 0)) * a.query_head_stride;
        float largest = 0.0f;
#pragma unroll
        for (int g = 0; g < groups; ++g) {
            const T* part = source + g * G + j * (G / 4);
#pragma unroll
            for (int w = 0; w < words; ++w) {
                if (work.aligned) {
                    const uint4 raw = *reinterpret_cast<const uint4*>(part + 8 * w);
                    const T* values = reinterpret_cast<const T*>(&raw);
#pragma unroll
                    for (int i = 0; i < 8; ++i) q[g][8 * w + i] = used ? widen(values[i]) : 0.0f;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) q[g][8 * w + i] = used ? widen(part[8 * w + i]) : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) largest = max_nan(largest, fabsf(q[g][8 * w + i]));
            }
        }
        largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // below 2^13 after the scaling; a row below 2^-114 keeps the factor of that size
        const int exponent = max(13, static_cast<int>(__float_as_uint(largest) >> 23 & 255u));
        const float up = __uint_as_float(static_cast<unsigned>(266 - exponent) << 23);
        const float down = __uint_as_float(static_cast<unsigned>(exponent - 12) << 23);  // 1 / up
#pragma unroll
        for (int g = 0; g < groups; ++g) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < words; ++w) {
                float* v = &q[g][8 * w];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= up, sum += v[i];
                // the even places of a word hold c 2^-24, the odd ones c 2^-20
                query[g][w][0][0][n] = pack_half(v[0], v[4]);
                query[g][w][0][1][n] = pack_half(v[2], v[6]);
                query[g][w][1][0][n] = pack_half(v[1] * 0.0625f, v[5] * 0.0625f);
                query[g][w][1][1][n] = pack_half(v[3] * 0.0625f, v[7] * 0.0625f);
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            // to the columns 2 j and 2 j + 1 that a score fragment holds, times 2^-24 as the codes
            query_sum[g][n][0] = __shfl_sync(0xffffffffu, sum, 8 * j) * 0x1p-24f;
            query_sum[g][n][1] = __shfl_sync(0xffffffffu, sum, 8 * j + 4) * 0x1p-24f;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            factor[n][i] = __shfl_sync(0xffffffffu, down, 8 * j + 4 * i) * 0x1p24f * (a.scale * log2_e);
            const int column = first_row + 8 * n + 2 * j + i;
            visible[n][i] = column < total_rows ? length - count + column / work.ratio + 1 : visible_last;
        }
    }

    // ---- one pass over the keys ----
    float top[NT][2], sum[NT][2], low[groups][NT][2], acc[groups][tiles][NT][4];
    float rounded[groups][NT][4];  // sums of the rounded weights, in elements 0 and 1
    constexpr unsigned ones[4] = {0x3c003c00u, 0u, 0x3c003c00u, 0u};
    float value_top[groups], value_factor[groups];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) top[n][i] = -FLT_MAX, sum[n][i] = 0.0f;
    }
#pragma unroll
    for (int g = 0; g < groups; ++g) {
        value_top[g] = 0.0f, value_factor[g] = 1.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            low[g][n][0] = low[g][n][1] = 0.0f;
            rounded[g][n][0] = rounded[g][n][1] = rounded[g][n][2] = rounded[g][n][3] = 0.0f;
#pragma unroll
            for (int t = 0; t < tiles; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[g][t][n][i] = 0.0f;
            }
        }
    }
    const int my_key = row_key(r);                  // score rows my_key and my_key + 8 of a run
    const int pair_key = (j & 1) | (j & 2) << 1;    // value keys pair_key and pair_key + 2, and 8 on
    int key_offset[groups], value_offset[groups][2];
#pragma unroll
    for (int g = 0; g < groups; ++g) {
        const int kb = g * (G / 2) + j * (G / 8), vb = g * (G / 2) + r * (G / 16);
        key_offset[g] = my_key * row_bytes + (((kb / 16) ^ swizzle<D>(my_key)) * 16 + kb % 16);
        value_offset[g][0] = pair_key * row_bytes + (((vb / 16) ^ swizzle<D>(pair_key)) * 16 + vb % 16);
        value_offset[g][1] = (pair_key + 2) * row_bytes + (((vb / 16) ^ swizzle<D>(pair_key + 2)) * 16 + vb % 16);
    }

    // A run of 16 keys. `masked`: some of them are hidden from some rows, or hold nothing.
    auto process = [&](auto masked_tag, const std::uint8_t* codes, const std::uint8_t* key_scales,
                       const std::uint8_t* value_scales, int place, bool absent) {
        constexpr bool masked = decltype(masked_tag)::value;
        float x[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
#pragma unroll
        for (int g = 0; g < groups; ++g) {
            unsigned near[words], far[words];
            const std::uint8_t* at = codes + key_offset[g];
            if constexpr (words == 4) {
                *reinterpret_cast<uint4*>(near) = *reinterpret_cast<const uint4*>(at);
                *reinterpret_cast<uint4*>(far) = *reinterpret_cast<const uint4*>(at + 8 * row_bytes);
            } else if constexpr (words == 2) {
                *reinterpret_cast<uint2*>(near) = *reinterpret_cast<const uint2*>(at);
                *reinterpret_cast<uint2*>(far) = *reinterpret_cast<const uint2*>(at + 8 * row_bytes);
            } else {
                near[0] = *reinterpret_cast<const unsigned*>(at);
                far[0] = *reinterpret_cast<const unsigned*>(at + 8 * row_bytes);
            }
            float dot[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) dot[n][0] = dot[n][1] = dot[n][2] = dot[n][3] = 0.0f;
#pragma unroll
            for (int w = 0; w < words; ++w) {
                const unsigned near8 = near[w] >> 8, far8 = far[w] >> 8;
                const unsigned even[4] = {near[w] & 0x000f000fu, far[w] & 0x000f000fu, near8 & 0x000f000fu,
                                          far8 & 0x000f000fu};
                const unsigned odd[4] = {near[w] & 0x00f000f0u, far[w] & 0x00f000f0u, near8 & 0x00f000f0u,
                                         far8 & 0x00f000f0u};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma(dot[n], even, query[g][w][0][0][n], query[g][w][0][1][n]);
                    mma(dot[n], odd, query[g][w][1][0][n], query[g][w][1][1][n]);
                }
            }
            const float2 pair_near = pair_at(key_scales, (my_key * groups + g) * 4);
            const float2 pair_far = pair_at(key_scales, ((my_key + 8) * groups + g) * 4);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    x[n][i] = fmaf(pair_near.x, dot[n][i], fmaf(pair_near.y, query_sum[g][n][i], x[n][i]));
                    x[n][i + 2] = fmaf(pair_far.x, dot[n][i + 2], fmaf(pair_far.y, query_sum[g][n][i], x[n][i + 2]));
                }
            }
        }
        float2 value_near[groups], value_far[groups];
        bool raise = false;
#pragma unroll
        for (int g = 0; g < groups; ++g) {
            value_near[g] = pair_at(value_scales, (my_key * groups + g) * 4);
            value_far[g] = pair_at(value_scales, ((my_key + 8) * groups + g) * 4);
            if (masked) {  // what lies past the block's last visible key is no one's
                if (absent || place + my_key >= end) value_near[g] = {0.0f, 0.0f};
                if (absent || place + my_key + 8 >= end) value_far[g] = {0.0f, 0.0f};
            }
            raise |= (value_near[g].x > value_top[g] && value_near[g].x < INFINITY) ||
                (value_far[g].x > value_top[g] && value_far[g].x < INFINITY);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[n][i] *= factor[n][i & 1];
                if (masked && (absent || place + my_key + (i & 2) * 4 >= visible[n][i & 1])) x[n][i] = -INFINITY;
                raise |= x[n][i] > top[n][i & 1] + top_slack;
            }
        }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float most = fmaxf(x[n][i], x[n][i + 2]);
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
                    most = fmaxf(most, top[n][i]);
                    const float shrink = exp2_fast(top[n][i] - most);
                    top[n][i] = most;
                    sum[n][i] *= shrink;
#pragma unroll
                    for (int g = 0; g < groups; ++g) {
                        low[g][n][i] *= shrink, rounded[g][n][i] *= shrink;
#pragma unroll
                        for (int t = 0; t < tiles; ++t) acc[g][t][n][i] *= shrink, acc[g][t][n][i + 2] *= shrink;
                    }
                }
            }
#pragma unroll
            for (int g = 0; g < groups; ++g) {
                float most = fmaxf(value_near[g].x < INFINITY ? value_near[g].x : 0.0f,
                                   value_far[g].x < INFINITY ? value_far[g].x : 0.0f);
                most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(most, 0.0f))));
                if (most > value_top[g]) {  // the power of two above it becomes 2^6
                    const unsigned exponent = (__float_as_uint(most) >> 23) + 1;
                    value_top[g] = __uint_as_float(exponent << 23);
                    const float scaled = __uint_as_float((260u - exponent) << 23);
                    const float change = scaled / value_factor[g];
                    value_factor[g] = scaled;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        rounded[g][n][0] *= change, rounded[g][n][1] *= change;
#pragma unroll
                        for (int t = 0; t < tiles; ++t) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[g][t][n][i] *= change;
                        }
                    }
                }
            }
        }
        float p[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[n][i] = exp2_fast(x[n][i] - top[n][i & 1]);
            sum[n][0] += p[n][0] + p[n][2];
            sum[n][1] += p[n][1] + p[n][3];
        }
        const std::uint8_t* values = codes + keys * row_bytes;
#pragma unroll
        for (int g = 0; g < groups; ++g) {
            unsigned b[NT][2];
            const float near_scale = value_near[g].x * value_factor[g], far_scale = value_far[g].x * value_factor[g];
            const float near_middle = fmaf(7.5f, value_near[g].x, value_near[g].y);
            const float far_middle = fmaf(7.5f, value_far[g].x, value_far[g].y);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[4], m[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = p[n][i] * (i < 2 ? near_scale : far_scale);
                    m[i] = p[n][i] * (i < 2 ? near_middle : far_middle);
                    // a hidden key's weight is 0 even against a scale that is no number
                    if (masked && x[n][i] == -INFINITY) w[i] = m[i] = 0.0f;
                }
                low[g][n][0] += m[0] + m[2];
                low[g][n][1] += m[1] + m[3];
                b[n][0] = transpose8x8(pack_half(w[0], w[1]));
                b[n][1] = transpose8x8(pack_half(w[2], w[3]));
                mma(rounded[g][n], ones, b[n][0], b[n][1]);
            }
            // the lane's channels of four keys: 4 codes of each (halves), 8 (a word) or 16 (two words)
            constexpr int value_words = G == 128 ? 2 : 1;
            unsigned code[4][value_words];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const std::uint8_t* at = values + value_offset[g][k & 1] + (k & 2) * 4 * row_bytes;
                if constexpr (G == 128) {
                    *reinterpret_cast<uint2*>(code[k]) = *reinterpret_cast<const uint2*>(at);
                } else if constexpr (G == 64) {
                    code[k][0] = *reinterpret_cast<const unsigned*>(at);
                } else {
                    code[k][0] = *reinterpret_cast<const std::uint16_t*>(at);
                }
            }
#pragma unroll
            for (int t = 0; t < tiles; t += 2) {
                const int w = t / 4;
                const unsigned select = t % 4 == 0 ? 0x5410u : 0x7632u;
                const unsigned one = __byte_perm(code[0][w], code[1][w], select);
                const unsigned two = __byte_perm(code[2][w], code[3][w], select);
                const unsigned front[4] = {one & 0x000f000fu, one & 0x00f000f0u, two & 0x000f000fu, two & 0x00f000f0u};
                const unsigned one8 = one >> 8, two8 = two >> 8;
                const unsigned back[4] = {one8 & 0x000f000fu, one8 & 0x00f000f0u, two8 & 0x000f000fu,
                                          two8 & 0x00f000f0u};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma(acc[g][t][n], front, b[n][0], b[n][1]);
                    mma(acc[g][t + 1][n], back, b[n][0], b[n][1]);
                }
            }
        }
    };

    for (int tile = warp, stage = 0; tile < tile_count; tile += warps, stage = stage + 1 == stages ? 0 : stage + 1) {
        asm volatile("cp.async.wait_group %0;" ::"n"(stages - 2) : "memory");
        __syncwarp();
        const std::uint8_t* base = ring_bytes + stage * stage_bytes<D, G>;
#pragma unroll 1
        for (int u = 0; u < runs; ++u) {
            const int place = begin + tile * keys + 16 * u;
            if (place >= end) break;
            const std::uint8_t* codes = base + 16 * u * row_bytes;
            const std::uint8_t* key_scales = base + keys * D + u * 64 * groups;
            const std::uint8_t* value_scales = key_scales + keys * 4 * groups;
            const bool absent = bad >> (stage * runs + u) & 1u;
            if (absent || place + 16 > visible_first || place + 16 > end) {
                process(std::true_type{}, codes, key_scales, value_scales, place, absent);
            } else {
                process(std::false_type{}, codes, key_scales, value_scales, place, false);
            }
        }
        __syncwarp();
        if (next < tile_count) {
            issue(next, stage == 0 ? stages - 1 : stage - 1);
            next += warps;
            fetch_pages(next);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- join the warps ----
    constexpr int pitch = D + 4;
    float* const outs = reinterpret_cast<float*>(shared);  // [warp][row][pitch]
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int offset = 4; offset < 32; offset *= 2) sum[n][i] += __shfl_xor_sync(0xffffffffu, sum[n][i], offset);
            if (r == 0) {
                joint_top[warp][8 * n + 2 * j + i] = top[n][i];
                joint_sum[warp][8 * n + 2 * j + i] = sum[n][i];
            }
        }
    }
    __syncthreads();  // every warp is done with its ring
#pragma unroll
    for (int g = 0; g < groups; ++g) {
        const float unscale = 0x1p24f / value_factor[g];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float m = low[g][n][i];
#pragma unroll
                for (int offset = 4; offset < 32; offset *= 2) m += __shfl_xor_sync(0xffffffffu, m, offset);
                const float middle = -7.5f * 0x1p-24f * rounded[g][n][i];
                float* row = outs + (warp * rows + 8 * n + 2 * j + i) * pitch + g * G + r * (G / 8);
#pragma unroll
                for (int t = 0; t < tiles; ++t) {
                    float2 o;
                    o.x = fmaf(acc[g][t][n][i] + middle, unscale, m);
                    o.y = fmaf(fmaf(acc[g][t][n][i + 2], 0.0625f, middle), unscale, m);
                    *reinterpret_cast<float2*>(row + 2 * t) = o;
                }
            }
        }
    }
    __syncthreads();
    const int block_index = (sequence * cache.kv_heads + kv_head) * work.row_blocks + row_block;
    float* const part = work.partials == nullptr || active == 1
        ? nullptr
        : work.partials + (static_cast<std::int64_t>(block_index) * work.ranges + range) * (rows * (D + 2));
    auto store = [&](int row, int d, float value, float total) {
        const int at = first_row + row;
        static_cast<T*>(a.output)[((first + at / work.ratio) * a.heads + kv_head * work.ratio + at % work.ratio) * D + d] =
            narrow<T>(total == 0.0f ? 0.0f : value / total);
    };
    for (int i = threadIdx.x; i < used_rows * D; i += 32 * warps) {
        const int row = i / D, d = i % D;
        float most = -FLT_MAX, total = 0.0f, value = 0.0f;
#pragma unroll
        for (int w = 0; w < warps; ++w) most = fmaxf(most, joint_top[w][row]);
#pragma unroll
        for (int w = 0; w < warps; ++w) {
            const float weight = exp2_fast(joint_top[w][row] - most);
            total = fmaf(joint_sum[w][row], weight, total);
            value = fmaf(outs[(w * rows + row) * pitch + d], weight, value);
        }
        if (part == nullptr) {
            store(row, d, value, total);
        } else {
            part[row * D + d] = value;
            if (d == 0) part[rows * D + row] = most, part[rows * D + rows + row] = total;
        }
    }
    if (part == nullptr) return;

    // ---- join the ranges: the last block of them to get here ----
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned ticket = atomicAdd(&work.tickets[block_index], 1u);
        joint_last = ticket + 1 == static_cast<unsigned>(active);
        if (joint_last) work.tickets[block_index] = 0;
    }
    __syncthreads();
    if (!joint_last) return;
    __threadfence();
    const float* const parts = work.partials + static_cast<std::int64_t>(block_index) * work.ranges * (rows * (D + 2));
    for (int i = threadIdx.x; i < used_rows * D; i += 32 * warps) {
        const int row = i / D, d = i % D;
        float most = -FLT_MAX, total = 0.0f, value = 0.0f;
        for (int s = 0; s < active; ++s) most = fmaxf(most, __ldcg(parts + s * (rows * (D + 2)) + rows * D + row));
        for (int s = 0; s < active; ++s) {
            const float* one = parts + s * (rows * (D + 2));
            const float weight = exp2_fast(__ldcg(one + rows * D + row) - most);
            total = fmaf(__ldcg(one + rows * D + rows + row), weight, total);
            value = fmaf(__ldcg(one + row * D + d), weight, value);
        }
        store(row, d, value, total);
    }
}

// Blocks that run at once (two an SM) times the rounds of them a call is cut into.
int block_target() { return 2 * 2 * sm_count(); }

template <typename T, int D, int G, int NT>
cudaError_t launch(const Work& work, cudaStream_t stream) {
    constexpr int bytes = shared_bytes<D, G, NT>;
    static SharedAllowance allowance;
    const cudaError_t allowed = allowance.allow(attend_kernel<T, D, G, NT>, bytes);
    if (allowed != cudaSuccess) return allowed;
    const dim3 grid(static_cast<unsigned>(work.ranges), static_cast<unsigned>(work.cache.kv_heads * work.row_blocks),
                    static_cast<unsigned>(work.a.batch));
    attend_kernel<T, D, G, NT><<<grid, 32 * warps, bytes, stream>>>(work);
    return cudaGetLastError();
}

template <typename T, int D, int G>
cudaError_t launch_rows(Work& work, const AttendWorkspace& workspace, cudaStream_t stream) {
    // 16 rows a block read the cache once for twice the rows; one block of 8 has half the registers. With heads of
    // 256 channels 16 rows' sums do not fit the registers.
    const std::int64_t rows = static_cast<std::int64_t>(work.a.max_queries) * work.ratio;
    const bool wide = D < 256 && rows > 8;
    const std::int64_t block_rows = wide ? 16 : 8;
    work.row_blocks = static_cast<int>((rows + block_rows - 1) / block_rows);
    const std::int64_t base = static_cast<std::int64_t>(work.a.batch) * work.cache.kv_heads * work.row_blocks;
    if (static_cast<std::int64_t>(work.cache.kv_heads) * work.row_blocks > 65535) return cudaErrorInvalidValue;
    const int step = warps * tile_keys<D>;  // a tile for every warp
    std::int64_t ranges = std::min<std::int64_t>((block_target() + base - 1) / base, (work.a.max_length + step - 1) / step);
    if (base >= block_target() || ranges < 1) ranges = 1;
    work.range = static_cast<int>((work.a.max_length + ranges * step - 1) / (ranges * step) * step);
    if (work.range == 0) work.range = step;
    work.ranges = std::max(1, (work.a.max_length + work.range - 1) / work.range);
    work.partials = work.ranges > 1 ? workspace.partials : nullptr;
    work.tickets = workspace.tickets;
    if constexpr (D < 256) {
        if (wide) return launch<T, D, G, 2>(work, stream);
    }
    return launch<T, D, G, 1>(work, stream);
}

template <typename T>
cudaError_t launch_shape(Work& work, const AttendWorkspace& workspace, cudaStream_t stream) {
    const int d = work.cache.head_dim, g = work.cache.group;
    if (d == 64) return g == 32 ? launch_rows<T, 64, 32>(work, workspace, stream) : launch_rows<T, 64, 64>(work, workspace, stream);
    if (d == 128) {
        return g == 32 ? launch_rows<T, 128, 32>(work, workspace, stream)
            : g == 64  ? launch_rows<T, 128, 64>(work, workspace, stream)
                       : launch_rows<T, 128, 128>(work, workspace, stream);
    }
    return g == 64 ? launch_rows<T, 256, 64>(work, workspace, stream) : launch_rows<T, 256, 128>(work, workspace, stream);
}

}  // namespace

// A call is cut into ranges only while there are fewer than block_target()
// blocks of rows, and then into fewer than twice that many blocks.
std::size_t attend_partial_bytes() {
    constexpr std::size_t floats = std::max(16 * (128 + 2), 8 * (256 + 2));
    return 2 * static_cast<std::size_t>(block_target()) * floats * sizeof(float);
}

std::size_t attend_ticket_bytes() { return static_cast<std::size_t>(block_target()) * sizeof(unsigned); }

cudaError_t attend(const Cache& cache, const AttendArgs& args, const AttendWorkspace& workspace, cudaStream_t stream) {
    if (args.tokens == 0 || args.batch == 0) return cudaSuccess;
    Work work{};
    work.cache = cache;
    work.a = args;
    work.ratio = args.heads / cache.kv_heads;
    const unsigned divisor = static_cast<unsigned>(cache.page_size / 16);
    while ((1u << work.tiles_per_page.shift) < divisor) ++work.tiles_per_page.shift;
    work.tiles_per_page.multiplier = static_cast<unsigned>(
        (((1ull << work.tiles_per_page.shift) - divisor) << 32) / divisor + 1);
    work.aligned = reinterpret_cast<std::uintptr_t>(args.queries) % 16 == 0 && args.query_stride % 8 == 0 &&
        args.query_head_stride % 8 == 0;
    return args.type == Type::f16 ? launch_shape<__half>(work, workspace, stream)
                                  : launch_shape<__nv_bfloat16>(work, workspace, stream);
}

}  // namespace nvcr_sm100::token
