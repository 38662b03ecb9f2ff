// The paged cache of keys and values in 4 bits: appending tokens, with the
// position rotation of keys and queries applied on the way, and reading stored
// tokens back as values. Per token, head and group of channels:
//   m = fp16(min x), s = fp16((max x - min x) * (1 / 15)), or 2^-24 (the smallest
//   FP16) where that is 0 and the range is not,
//   c = clamp(rint((x - m) / s), 0, 15), 0 where s is 0 or (x - m) / s is NaN.
// The codes are computed against the rounded s and m, so their rounding costs
// nothing but the ends of the range. s and m are FP16, as the cache's readers
// want them in one 32-bit word; groups beyond the FP16 range (or holding a NaN
// or infinity) stand for non-finite values. The rotation is FP32, each product
// rounded by itself, and keys are quantised from the unrounded rotation.
//
// Measured on a B200, 32 query heads, 8 cache heads of 128: 8192 BF16 tokens, 64
// channels rotated, groups of 32, appended and read back (225 MB) 49.5 us, 4.5 TB/s,
// bound by instruction issue and HBM (the append is 24 million warp instructions);
// one FP16 token, all channels rotated, groups of 64, 3.4 us for the two launches.
#include "token_elements.cuh"

#include <algorithm>
#include <type_traits>

namespace nvcr_sm100::token {
namespace {

__device__ __forceinline__ void note(const Cache& cache, unsigned bit) {
    if (cache.status != nullptr) atomicOr(cache.status, bit);
}

// A group's scale and minimum, and the codes of its values.
struct GroupForm {
    __half scale, minimum;
    float s, m, inverse;
    __device__ __forceinline__ GroupForm(float low, float high) {
        minimum = __float2half_rn(low);
        scale = __float2half_rn((high - low) * (1.0f / 15.0f));
        if (high > low && __half2float(scale) == 0.0f) scale = __ushort_as_half(1);
        m = __half2float(minimum), s = __half2float(scale);
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(s));
        if (s == 0.0f) inverse = 0.0f;
    }
    // The codes of N values, packed, on the FP32 and integer pipes alone (conversions run at a quarter of their rate):
    // adding 1.5 * 2^23 rounds to the nearest integer, ties to even, in the low bits. A product with the reciprocal is
    // within 2^-18 of the quotient (which is below 16, or clamped), so only where one is that close to a tie are the
    // values divided.
    template <int N>
    __device__ __forceinline__ unsigned codes(const float (&x)[N]) const {
        unsigned packed = 0, offset = 0;
        bool tie = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float level = clamped((x[i] - m) * inverse), sum = level + 12582912.0f;
            tie |= fabsf(level - (sum - 12582912.0f)) > 0.49999f;
            packed += __float_as_uint(sum) << (4 * i);
            offset += 0x4b400000u << (4 * i);
        }
        if (tie) {
            packed = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float level = s > 0.0f ? clamped(__fdiv_rn(x[i] - m, s)) : 0.0f;
                packed += __float_as_uint(level + 12582912.0f) << (4 * i);
            }
        }
        return packed - offset;
    }
    __device__ __forceinline__ unsigned bits() const {
        return __half_as_ushort(scale) | static_cast<unsigned>(__half_as_ushort(minimum)) << 16;
    }

private:
    static __device__ __forceinline__ float clamped(float v) { return fminf(fmaxf(v, 0.0f), 15.0f); }  // a NaN is 0
};

// Any strides, alignment and rotation: one warp a (token, head) of keys, values
// or queries; lane l holds channels l * D / 32 .., so a group of channels is a
// run of group * 32 / D lanes.
template <typename T, int D>
__global__ void append_kernel(Cache cache, AppendArgs a) {
    constexpr int per_lane = D / 32;
    join_chain();
    const int lane = threadIdx.x % 32;
    const int heads = 2 * cache.kv_heads + (a.queries != nullptr ? a.query_heads : 0);
    const std::int64_t item = (static_cast<std::int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
    const std::int64_t token = item / heads;
    if (token >= a.tokens) return;
    int head = static_cast<int>(item % heads);
    const bool is_key = head < cache.kv_heads;
    const bool is_value = !is_key && head < 2 * cache.kv_heads;
    if (!is_key) head -= is_value ? cache.kv_heads : 2 * cache.kv_heads;
    const T* source = is_key ? static_cast<const T*>(a.keys) + token * a.key_stride + head * a.key_head_stride
        : is_value ? static_cast<const T*>(a.values) + token * a.value_stride + head * a.value_head_stride
                   : static_cast<const T*>(a.queries) + token * a.query_stride + head * a.query_head_stride;
    float x[per_lane];
#pragma unroll
    for (int i = 0; i < per_lane; ++i) x[i] = widen(source[lane * per_lane + i]);
    std::int64_t position = 0;
    if (a.positions != nullptr) position = a.positions[token];
    const bool placed = a.positions == nullptr || (position >= 0 && position < a.table_rows);
    if (!placed && lane == 0) note(cache, status_position);
    if (!is_value && a.positions != nullptr && placed) {
        const int half = a.rotary / 2;
        const float* cosines = a.cosines + position * half;
        const float* sines = a.sines + position * half;
#pragma unroll
        for (int i = 0; i < per_lane; ++i) {
            const int channel = lane * per_lane + i;
            if (channel >= a.rotary) continue;
            const bool second = a.interleaved ? channel % 2 == 1 : channel >= half;
            const int angle = a.interleaved ? channel / 2 : channel - (second ? half : 0);
            const int partner = a.interleaved ? channel ^ 1 : channel + (second ? -half : half);
            const float c = cosines[angle], s = sines[angle], other = widen(source[partner]);
            x[i] = second ? __fadd_rn(__fmul_rn(x[i], c), __fmul_rn(other, s))
                          : __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(other, s));
        }
    }
    if (!is_key && !is_value) {
        T* out = static_cast<T*>(a.rotated) + (token * a.query_heads + head) * D + lane * per_lane;
#pragma unroll
        for (int i = 0; i < per_lane; ++i) out[i] = narrow<T>(placed ? x[i] : NAN);
        return;
    }
    const std::int64_t slot = a.slots[token];
    if (slot < 0 || !placed) return;  // a padding token, or one without a position
    if (slot >= static_cast<std::int64_t>(cache.pages) * cache.page_size) {
        if (lane == 0) note(cache, status_slot);
        return;
    }
    float low = x[0], high = x[0];
#pragma unroll
    for (int i = 1; i < per_lane; ++i) low = min_nan(low, x[i]), high = max_nan(high, x[i]);
    const int lanes = cache.group / per_lane;
    for (int offset = 1; offset < lanes; offset *= 2) {
        low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, offset));
        high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, offset));
    }
    const GroupForm form(low, high);
    const unsigned packed = form.codes(x);
    const std::int64_t page = slot / cache.page_size;
    const std::int64_t place = (page * cache.kv_heads + head) * cache.page_size + slot % cache.page_size;
    std::uint8_t* codes = (is_key ? cache.key_codes : cache.value_codes) + place * (D / 2) + lane * (per_lane / 2);
#pragma unroll
    for (int i = 0; i < per_lane / 2; ++i) codes[i] = static_cast<std::uint8_t>(packed >> (8 * i));
    if (lane % lanes == 0) {
        reinterpret_cast<unsigned*>(is_key ? cache.key_scales : cache.value_scales)[place * (D / cache.group) + lane / lanes] =
            form.bits();
    }
}

// Eight elements of a 16-bit type from one 16-byte access, and eight of any type to memory.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& raw, float (&x)[8]) {
    const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same_v<T, __half>) {
            const float2 pair = __half22float2(reinterpret_cast<const __half2&>(words[i]));
            x[2 * i] = pair.x, x[2 * i + 1] = pair.y;
        } else {
            x[2 * i] = __uint_as_float(words[i] << 16), x[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
        }
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* to, const float (&x)[8]) {
    if constexpr (std::is_same_v<T, float>) {
        reinterpret_cast<float4*>(to)[0] = {x[0], x[1], x[2], x[3]};
        reinterpret_cast<float4*>(to)[1] = {x[4], x[5], x[6], x[7]};
    } else {
        unsigned words[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 pair = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                words[i] = reinterpret_cast<const unsigned&>(pair);
            } else {
                const __nv_bfloat162 pair = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                words[i] = reinterpret_cast<const unsigned&>(pair);
            }
        }
        *reinterpret_cast<uint4*>(to) = {words[0], words[1], words[2], words[3]};
    }
}

// Eight channels a thread, D / 8 threads a (token, run of heads of queries, keys
// or values): a thread reads its angles' cosines and sines once, loads H heads in
// 16-byte accesses before it uses any (that keeps enough bytes in flight), and a
// key's or query's rotation partner, eight channels elsewhere in the head, as a
// second load of a line that is in L1. Takes aligned
// tensors and rotations of whole octets (pairs (i, i + rotary / 2): rotary a
// multiple of 16; (2 i, 2 i + 1): of 8).
template <typename T, int D, int H, bool interleaved>
__global__ void __launch_bounds__(256, 4) append_octets_kernel(Cache cache, AppendArgs a, int run_heads,
                                                               Divisor runs_per_page) {
    constexpr int lanes = D / 8;
    join_chain();
    const int lane = threadIdx.x % lanes, channel = 8 * lane;
    const std::int64_t token = static_cast<std::int64_t>(blockIdx.x) * (256 / lanes) + threadIdx.x / lanes;
    const bool valid = token < a.tokens;  // threads past the end stay for the shuffles
    const int query_runs = a.queries != nullptr ? (a.query_heads + run_heads - 1) / run_heads : 0;
    const int kv_runs = (cache.kv_heads + run_heads - 1) / run_heads;
    const int half = a.rotary / 2;
    const bool second = !interleaved && channel >= half;

    // One body for queries, keys and values (the kind is uniform in a block).
    auto body = [&](auto kind_tag, int run) {
        constexpr int kind = decltype(kind_tag)::value;
        constexpr bool is_query = kind == 0, rotates = kind != 2;
        int first = run * run_heads;
        const int last = min(is_query ? a.query_heads : cache.kv_heads, first + run_heads);
        const std::int64_t head_stride = is_query ? a.query_head_stride : kind == 1 ? a.key_head_stride : a.value_head_stride;
        const T* source = static_cast<const T*>(is_query ? a.queries : kind == 1 ? a.keys : a.values) + channel +
            (valid ? token * (is_query ? a.query_stride : kind == 1 ? a.key_stride : a.value_stride) + first * head_stride : 0);
        const bool turns = rotates && a.positions != nullptr && channel < a.rotary;
        uint4 raw[H], partner[rotates && !interleaved ? H : 1];
        auto load = [&] {
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (first + h < last) {  // a thread past the end reads the first token and stores nothing
                    raw[h] = *reinterpret_cast<const uint4*>(source + h * head_stride);
                    if constexpr (rotates && !interleaved) {
                        if (turns) partner[h] = *reinterpret_cast<const uint4*>(source + h * head_stride + (second ? -half : half));
                    }
                }
            }
        };
        load();
        std::int64_t slot = -1, position = 0;
        if (valid && !is_query) slot = a.slots[token];
        if (valid && a.positions != nullptr) position = a.positions[token];
        const bool placed = a.positions == nullptr || (position >= 0 && position < a.table_rows);
        if (!placed && lane == 0) note(cache, status_position);
        const bool turned = turns && placed;
        // x cos - partner sin for a pair's first element, x cos + partner sin for its second: the sign goes to the sine
        float cosine[8], sine[8];
        if (rotates && turned) {
            const float4* cosines = reinterpret_cast<const float4*>(a.cosines + position * half);
            const float4* sines = reinterpret_cast<const float4*>(a.sines + position * half);
            if constexpr (interleaved) {
                const float4 c = cosines[lane], s = sines[lane];
                cosine[0] = cosine[1] = c.x, cosine[2] = cosine[3] = c.y;
                cosine[4] = cosine[5] = c.z, cosine[6] = cosine[7] = c.w;
                sine[1] = s.x, sine[3] = s.y, sine[5] = s.z, sine[7] = s.w;
                sine[0] = -s.x, sine[2] = -s.y, sine[4] = -s.z, sine[6] = -s.w;
            } else {
                const int at = (second ? channel - half : channel) / 4;
                const float sign = second ? 1.0f : -1.0f;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 c = cosines[at + i], s = sines[at + i];
                    cosine[4 * i] = c.x, cosine[4 * i + 1] = c.y, cosine[4 * i + 2] = c.z, cosine[4 * i + 3] = c.w;
                    sine[4 * i] = sign * s.x, sine[4 * i + 1] = sign * s.y;
                    sine[4 * i + 2] = sign * s.z, sine[4 * i + 3] = sign * s.w;
                }
            }
        }
        const std::int64_t limit = static_cast<std::int64_t>(cache.pages) * cache.page_size;
        const bool stored = !is_query && placed && slot >= 0 && slot < limit;
        if (slot >= limit && lane == 0) note(cache, status_slot);
        std::int64_t place = 0;
        if (stored) {  // slots are below 2^35, their runs of 16 below 2^31
            const std::int64_t page = divide(static_cast<unsigned>(slot >> 4), runs_per_page);
            place = (page * cache.kv_heads + first) * cache.page_size + (slot - page * cache.page_size);
        }
        const int group_lanes = cache.group / 8, group_shift = 31 - __clz(group_lanes);  // 4, 8 or 16
        unsigned* const codes_to = reinterpret_cast<unsigned*>(kind == 1 ? cache.key_codes : cache.value_codes) + lane;
        unsigned* const pairs_to =
            reinterpret_cast<unsigned*>(kind == 1 ? cache.key_scales : cache.value_scales) + (lane >> group_shift);
        T* rotated = static_cast<T*>(a.rotated) + (is_query && valid ? (token * a.query_heads + first) * D + channel : 0);
        for (;;) {
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (first + h >= last) break;
                float x[8];
                unpack8<T>(raw[h], x);
                if (rotates && turned) {
                    float other[8], result[8];
                    if constexpr (interleaved) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) other[i] = x[i ^ 1];
                    } else {
                        unpack8<T>(partner[rotates && !interleaved ? h : 0], other);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) result[i] = __fadd_rn(__fmul_rn(x[i], cosine[i]), __fmul_rn(other[i], sine[i]));
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = result[i];
                }
                if constexpr (is_query) {
                    if (!placed) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = NAN;
                    }
                    if (valid) store8(rotated + h * D, x);
                } else {
                    float low = x[0], high = x[0];
#pragma unroll
                    for (int i = 1; i < 8; ++i) low = min_nan(low, x[i]), high = max_nan(high, x[i]);
#pragma unroll
                    for (int offset = 1; offset < 16; offset *= 2) {
                        if (offset >= group_lanes) break;
                        low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, offset));
                        high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, offset));
                    }
                    if (stored) {
                        const GroupForm form(low, high);
                        const std::int64_t at = place + h * cache.page_size;
                        codes_to[at * lanes] = form.codes(x);
                        if ((lane & (group_lanes - 1)) == 0) pairs_to[at * (lanes >> group_shift)] = form.bits();
                    }
                }
            }
            first += H;
            if (first >= last) return;
            source += H * head_stride, rotated += is_query ? H * D : 0;
            place += static_cast<std::int64_t>(H) * cache.page_size;
            load();
        }
    };
    const int run = blockIdx.y;
    if (run < query_runs) {
        body(std::integral_constant<int, 0>{}, run);
    } else if (run < query_runs + kv_runs) {
        body(std::integral_constant<int, 1>{}, run - query_runs);
    } else {
        body(std::integral_constant<int, 2>{}, run - query_runs - kv_runs);
    }
}

// Eight channels a thread of one stored token's keys and values.
template <typename T, int D>
__global__ void __launch_bounds__(256) read_kernel(Cache cache, const std::int64_t* slots, std::int64_t count, T* keys,
                                                   T* values, Divisor by_heads, Divisor runs_per_page) {
    constexpr int lanes = D / 8;
    join_chain();
    const std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= count * cache.kv_heads * lanes) return;
    const int lane = static_cast<int>(i % lanes);
    const unsigned head_token = static_cast<unsigned>(i / lanes);  // count times heads is below 2^31
    const unsigned token = divide(head_token, by_heads), head = head_token - token * cache.kv_heads;
    const std::int64_t slot = slots[token];
    unsigned codes[2] = {}, pairs[2] = {};
    if (slot >= 0 && slot < static_cast<std::int64_t>(cache.pages) * cache.page_size) {
        const std::int64_t page = divide(static_cast<unsigned>(slot >> 4), runs_per_page);
        const std::int64_t at = (page * cache.kv_heads + head) * cache.page_size + slot - page * cache.page_size;
        const int group_shift = 28 - __clz(cache.group);  // of the lanes of a group: 4, 8 or 16
        const std::int64_t code_at = at * lanes + lane, pair_at = at * (lanes >> group_shift) + (lane >> group_shift);
        codes[0] = reinterpret_cast<const unsigned*>(cache.key_codes)[code_at];
        codes[1] = reinterpret_cast<const unsigned*>(cache.value_codes)[code_at];
        pairs[0] = reinterpret_cast<const unsigned*>(cache.key_scales)[pair_at];
        pairs[1] = reinterpret_cast<const unsigned*>(cache.value_scales)[pair_at];
    } else if (slot >= 0) {
        note(cache, status_slot);
    }
    const bool aligned = (reinterpret_cast<std::uintptr_t>(keys) | reinterpret_cast<std::uintptr_t>(values)) % 16 == 0;
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
        const float2 pair = __half22float2(reinterpret_cast<const __half2&>(pairs[kind]));
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // 2^23 + code, less 2^23: no conversion
            x[e] = fmaf(__uint_as_float((codes[kind] >> (4 * e) & 15u) | 0x4b000000u) - 8388608.0f, pair.x, pair.y);
        }
        T* const out = (kind == 0 ? keys : values) + i * 8;
        if (aligned) {
            store8(out, x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = narrow<T>(x[e]);
        }
    }
}

template <typename T, int D>
cudaError_t append_shape(const Cache& cache, const AppendArgs& a, cudaStream_t stream) {
    const int heads = 2 * cache.kv_heads + (a.queries != nullptr ? a.query_heads : 0);
    const auto aligned = [](const void* p, std::int64_t stride, std::int64_t head_stride) {
        return reinterpret_cast<std::uintptr_t>(p) % 16 == 0 && stride % 8 == 0 && head_stride % 8 == 0;
    };
    const bool octets = aligned(a.keys, a.key_stride, a.key_head_stride) &&
        aligned(a.values, a.value_stride, a.value_head_stride) &&
        aligned(a.queries, a.query_stride, a.query_head_stride) && aligned(a.rotated, 0, 0) &&
        (a.positions == nullptr || (a.rotary % (a.interleaved ? 8 : 16) == 0 && aligned(a.cosines, 0, 0) &&
                                    aligned(a.sines, 0, 0)));
    if (octets) {
        constexpr int tokens_each = 256 / (D / 8);
        const std::int64_t token_blocks = (a.tokens + tokens_each - 1) / tokens_each;
        // Many tokens: eight heads a thread share its angles and addresses, four of them in flight together. A few: one,
        // which makes their threads many. us with one and with eight, 32 query heads and 8 cache heads of 128: 512
        // tokens (192 blocks of eight heads) 6.2, 7.2; 640 (240) 7.6, 7.4; 2048 19.8, 13.7; 8192 84, 41. 16 and 2: 768
        // tokens (192) 4.6, 3.8; 1536 (384) 7.2, 5.6. No queries, 8 cache heads: 1536 (192) 7.0, 7.6. The general kernel
        // takes 2.6 us for one token (2.0 here) and 147 us for 8192.
        const int query_heads = a.queries != nullptr ? a.query_heads : 0;
        const auto runs_of = [&](int n) {
            return static_cast<std::int64_t>((query_heads + n - 1) / n) + 2 * ((cache.kv_heads + n - 1) / n);
        };
        const bool many = 2 * token_blocks * runs_of(8) >= 3 * static_cast<std::int64_t>(sm_count());
        const int run_heads = many ? 8 : 1;
        const std::int64_t runs = runs_of(run_heads);
        if (runs > 65535) return cudaErrorInvalidValue;
        const dim3 grid(static_cast<unsigned>(token_blocks), static_cast<unsigned>(runs));
        const Divisor runs_per_page = divisor(static_cast<unsigned>(cache.page_size / 16));
        const auto kernel = a.interleaved
            ? many ? append_octets_kernel<T, D, 4, true> : append_octets_kernel<T, D, 1, true>
            : many ? append_octets_kernel<T, D, 4, false> : append_octets_kernel<T, D, 1, false>;
        return kernels::launch_overlapped(kernel, grid, dim3(256), 0, stream, cache, a, run_heads, runs_per_page);
    }
    const std::int64_t blocks = (a.tokens * heads + 7) / 8;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    return kernels::launch_overlapped(append_kernel<T, D>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, cache,
                                      a);
}

template <typename T>
cudaError_t append_typed(const Cache& cache, const AppendArgs& args, cudaStream_t stream) {
    switch (cache.head_dim) {
    case 64: return append_shape<T, 64>(cache, args, stream);
    case 128: return append_shape<T, 128>(cache, args, stream);
    default: return append_shape<T, 256>(cache, args, stream);
    }
}

template <typename T>
cudaError_t read_typed(const Cache& cache, const std::int64_t* slots, std::int64_t count, void* keys, void* values,
                       cudaStream_t stream) {
    const std::int64_t heads = count * cache.kv_heads, blocks = (heads * (cache.head_dim / 8) + 255) / 256;
    if (heads > 0x7fffffff || blocks > 0x7fffffff) return cudaErrorInvalidValue;
    const unsigned grid = static_cast<unsigned>(blocks);
    T* const k = static_cast<T*>(keys);
    T* const v = static_cast<T*>(values);
    const Divisor by_heads = divisor(static_cast<unsigned>(cache.kv_heads));
    const Divisor runs = divisor(static_cast<unsigned>(cache.page_size / 16));
    const auto kernel = cache.head_dim == 64 ? read_kernel<T, 64> : cache.head_dim == 128 ? read_kernel<T, 128>
                                                                                        : read_kernel<T, 256>;
    return kernels::launch_overlapped(kernel, dim3(grid), dim3(256), 0, stream, cache, slots, count, k, v, by_heads, runs);
}

}  // namespace

cudaError_t append(const Cache& cache, const AppendArgs& args, cudaStream_t stream) {
    if (args.tokens == 0) return cudaSuccess;
    return args.type == Type::f16 ? append_typed<__half>(cache, args, stream)
                                  : append_typed<__nv_bfloat16>(cache, args, stream);
}

cudaError_t read(const Cache& cache, Type type, const std::int64_t* slots, std::int64_t count, void* keys, void* values,
                 cudaStream_t stream) {
    if (count == 0) return cudaSuccess;
    switch (type) {
    case Type::f16: return read_typed<__half>(cache, slots, count, keys, values, stream);
    case Type::bf16: return read_typed<__nv_bfloat16>(cache, slots, count, keys, values, stream);
    case Type::f32: return read_typed<float>(cache, slots, count, keys, values, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace nvcr_sm100::token
