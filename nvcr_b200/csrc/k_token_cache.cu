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
    float s, m;
    __device__ __forceinline__ GroupForm(float low, float high) {
        minimum = __float2half_rn(low);
        scale = __float2half_rn((high - low) * (1.0f / 15.0f));
        if (high > low && __half2float(scale) == 0.0f) scale = __ushort_as_half(1);
        m = __half2float(minimum), s = __half2float(scale);
    }
    __device__ __forceinline__ unsigned code(float x) const {
        const float level = s > 0.0f ? rintf(__fdiv_rn(x - m, s)) : 0.0f;
        return static_cast<unsigned>(fminf(fmaxf(level, 0.0f), 15.0f));  // fmaxf takes a NaN to 0
    }
    __device__ __forceinline__ unsigned bits() const {
        return __half_as_ushort(scale) | static_cast<unsigned>(__half_as_ushort(minimum)) << 16;
    }
};

// Any strides, alignment and rotation: one warp a (token, head) of keys, values
// or queries; lane l holds channels l * D / 32 .., so a group of channels is a
// run of group * 32 / D lanes.
template <typename T, int D>
__global__ void append_kernel(Cache cache, AppendArgs a) {
    constexpr int per_lane = D / 32;
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
    const std::int64_t page = slot / cache.page_size;
    const std::int64_t place = (page * cache.kv_heads + head) * cache.page_size + slot % cache.page_size;
    std::uint8_t* codes = (is_key ? cache.key_codes : cache.value_codes) + place * (D / 2) + lane * (per_lane / 2);
#pragma unroll
    for (int i = 0; i < per_lane / 2; ++i) codes[i] = static_cast<std::uint8_t>(form.code(x[2 * i]) | form.code(x[2 * i + 1]) << 4);
    if (lane % lanes == 0) {
        reinterpret_cast<unsigned*>(is_key ? cache.key_scales : cache.value_scales)[place * (D / cache.group) + lane / lanes] =
            form.bits();
    }
}

// Eight elements of a 16-bit type in one access.
template <typename T>
__device__ __forceinline__ void load8(const T* from, float (&x)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(from);
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

// Eight channels a thread, D / 8 threads a (token, run of `heads_each` heads): a
// thread reads its angles' cosines and sines once and its heads in 16-byte
// accesses; a key's or query's rotation partner, eight channels elsewhere in the
// head, is a second load of a line that is in L1. Takes aligned tensors and
// rotations of whole octets (pairs (i, i + rotary / 2): rotary a multiple of 16;
// (2 i, 2 i + 1): of 8).
template <typename T, int D>
__global__ void __launch_bounds__(256) append_octets_kernel(Cache cache, AppendArgs a, int heads_each) {
    constexpr int lanes = D / 8;
    const int lane = threadIdx.x % lanes, channel = 8 * lane;
    const std::int64_t token = static_cast<std::int64_t>(blockIdx.x) * (blockDim.x / lanes) + threadIdx.x / lanes;
    const bool valid = token < a.tokens;  // threads past the end stay for the shuffles
    const int query_heads = a.queries != nullptr ? a.query_heads : 0;
    const int all = query_heads + 2 * cache.kv_heads;
    const int first = blockIdx.y * heads_each, last = min(all, first + heads_each);
    const std::int64_t slot = valid ? a.slots[token] : -1;
    bool placed = true;
    float cosine[8], sine[8];
    const int half = a.rotary / 2;
    bool turned = false;
    if (a.positions != nullptr && valid) {
        const std::int64_t position = a.positions[token];
        placed = position >= 0 && position < a.table_rows;
        if (!placed && lane == 0) note(cache, status_position);
        turned = placed && channel < a.rotary;
        if (turned) {
            const float* cosines = a.cosines + position * half;
            const float* sines = a.sines + position * half;
            if (a.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; ++i) cosine[i] = cosines[channel / 2 + i / 2], sine[i] = sines[channel / 2 + i / 2];
            } else {
                const int angle = channel < half ? channel : channel - half;
#pragma unroll
                for (int i = 0; i < 8; ++i) cosine[i] = cosines[angle + i], sine[i] = sines[angle + i];
            }
        }
    }
    const bool second = !a.interleaved && channel >= half;
    const int partner = second ? -half : half;
    const std::int64_t limit = static_cast<std::int64_t>(cache.pages) * cache.page_size;
    const bool stored = valid && placed && slot >= 0 && slot < limit;
    if (valid && slot >= limit && lane == 0) note(cache, status_slot);
    const std::int64_t page = stored ? slot / cache.page_size : 0;
    const std::int64_t place = page * cache.kv_heads * cache.page_size + (stored ? slot - page * cache.page_size : 0);
#pragma unroll 2
    for (int h = first; h < last; ++h) {
        const bool is_query = h < query_heads, is_key = !is_query && h < query_heads + cache.kv_heads;
        const int head = is_query ? h : is_key ? h - query_heads : h - query_heads - cache.kv_heads;
        if (is_query && !valid) continue;
        float x[8] = {}, other[8] = {};
        if (valid) {
            const T* source = is_query ? static_cast<const T*>(a.queries) + token * a.query_stride + head * a.query_head_stride
                : is_key ? static_cast<const T*>(a.keys) + token * a.key_stride + head * a.key_head_stride
                         : static_cast<const T*>(a.values) + token * a.value_stride + head * a.value_head_stride;
            load8(source + channel, x);
            if (turned && (is_query || is_key)) {
                if (a.interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) other[i] = x[i ^ 1];
                } else {
                    load8(source + channel + partner, other);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float one = __fmul_rn(x[i], cosine[i]), two = __fmul_rn(other[i], sine[i]);
                    x[i] = (a.interleaved ? i % 2 == 1 : second) ? __fadd_rn(one, two) : __fsub_rn(one, two);
                }
            }
        }
        if (is_query) {
            if (!placed) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = NAN;
            }
            store8(static_cast<T*>(a.rotated) + (token * a.query_heads + head) * D + channel, x);
            continue;
        }
        float low = x[0], high = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) low = min_nan(low, x[i]), high = max_nan(high, x[i]);
        const int group_lanes = cache.group / 8;
        for (int offset = 1; offset < group_lanes; offset *= 2) {
            low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, offset));
            high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, offset));
        }
        if (!stored) continue;
        const GroupForm form(low, high);
        unsigned codes = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) codes |= form.code(x[i]) << (4 * i);
        const std::int64_t at = place + static_cast<std::int64_t>(head) * cache.page_size;
        reinterpret_cast<unsigned*>(is_key ? cache.key_codes : cache.value_codes)[at * lanes + lane] = codes;
        if (lane % group_lanes == 0) {
            reinterpret_cast<unsigned*>(is_key ? cache.key_scales : cache.value_scales)[at * (lanes / group_lanes) +
                                                                                       lane / group_lanes] = form.bits();
        }
    }
}

// Eight channels a thread of one stored token's keys, then of its values.
template <typename T, int D>
__global__ void __launch_bounds__(256) read_kernel(Cache cache, const std::int64_t* slots, std::int64_t count, T* keys,
                                                   T* values) {
    constexpr int lanes = D / 8;
    const std::int64_t per_kind = count * cache.kv_heads * lanes;
    const std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    const bool is_value = blockIdx.y == 1;
    if (i >= per_kind) return;
    const int lane = static_cast<int>(i % lanes);
    const unsigned head_token = static_cast<unsigned>(i / lanes);  // count times heads is below 2^32
    const unsigned token = head_token / cache.kv_heads, head = head_token - token * cache.kv_heads;
    T* out = (is_value ? values : keys) + i * 8;
    const std::int64_t slot = slots[token];
    float x[8] = {};
    if (slot >= 0 && slot < static_cast<std::int64_t>(cache.pages) * cache.page_size) {
        const std::int64_t page = slot / cache.page_size;
        const std::int64_t at = (page * cache.kv_heads + head) * cache.page_size + slot - page * cache.page_size;
        const unsigned codes = reinterpret_cast<const unsigned*>(is_value ? cache.value_codes : cache.key_codes)[at * lanes + lane];
        const int group_lanes = cache.group / 8;
        const unsigned pair = reinterpret_cast<const unsigned*>(is_value ? cache.value_scales : cache.key_scales)
            [at * (lanes / group_lanes) + lane / group_lanes];
        const float s = half_bits(static_cast<std::uint16_t>(pair)), m = half_bits(static_cast<std::uint16_t>(pair >> 16));
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = fmaf(static_cast<float>(codes >> (4 * e) & 15u), s, m);
    } else if (slot >= 0) {
        note(cache, status_slot);
    }
    if (reinterpret_cast<std::uintptr_t>(out) % 16 == 0) {
        store8(out, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = narrow<T>(x[e]);
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
        (a.positions == nullptr || a.rotary % (a.interleaved ? 8 : 16) == 0);
    if (octets) {
        constexpr int tokens_each = 256 / (D / 8);
        const std::int64_t token_blocks = (a.tokens + tokens_each - 1) / tokens_each;
        // More heads a thread share the angles; fewer keep a few tokens' threads many.
        const std::int64_t room = token_blocks * heads / (16 * static_cast<std::int64_t>(sm_count()));
        const int heads_each = static_cast<int>(std::max<std::int64_t>(1, std::min<std::int64_t>(8, room)));
        const dim3 grid(static_cast<unsigned>(token_blocks), static_cast<unsigned>((heads + heads_each - 1) / heads_each));
        if (grid.y > 65535) return cudaErrorInvalidValue;
        append_octets_kernel<T, D><<<grid, 256, 0, stream>>>(cache, a, heads_each);
    } else {
        const std::int64_t blocks = (a.tokens * heads + 7) / 8;
        if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
        append_kernel<T, D><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(cache, a);
    }
    return cudaGetLastError();
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
    if (heads > 0xffffffffll || blocks > 0x7fffffff) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    T* const k = static_cast<T*>(keys);
    T* const v = static_cast<T*>(values);
    switch (cache.head_dim) {
    case 64: read_kernel<T, 64><<<grid, 256, 0, stream>>>(cache, slots, count, k, v); break;
    case 128: read_kernel<T, 128><<<grid, 256, 0, stream>>>(cache, slots, count, k, v); break;
    default: read_kernel<T, 256><<<grid, 256, 0, stream>>>(cache, slots, count, k, v); break;
    }
    return cudaGetLastError();
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
