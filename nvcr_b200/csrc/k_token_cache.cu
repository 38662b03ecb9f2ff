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

namespace nvcr_sm100::token {
namespace {

__device__ __forceinline__ void note(const Cache& cache, unsigned bit) {
    if (cache.status != nullptr) atomicOr(cache.status, bit);
}

// One warp a (token, head) of keys, values or queries; lane l holds channels
// l * D/32 .. + D/32 - 1, so a group of channels is a run of group * 32 / D lanes.
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
    const __half minimum = __float2half_rn(low);
    __half scale = __float2half_rn((high - low) * (1.0f / 15.0f));
    if (high > low && __half2float(scale) == 0.0f) scale = __ushort_as_half(1);
    const float m = __half2float(minimum), s = __half2float(scale);
    unsigned code[per_lane];
#pragma unroll
    for (int i = 0; i < per_lane; ++i) {
        const float level = s > 0.0f ? rintf(__fdiv_rn(x[i] - m, s)) : 0.0f;
        code[i] = static_cast<unsigned>(fminf(fmaxf(level, 0.0f), 15.0f));  // fmaxf takes a NaN to 0
    }
    const std::int64_t page = slot / cache.page_size;
    const std::int64_t place = (page * cache.kv_heads + head) * cache.page_size + slot % cache.page_size;
    std::uint8_t* codes = (is_key ? cache.key_codes : cache.value_codes) + place * (D / 2) + lane * (per_lane / 2);
#pragma unroll
    for (int i = 0; i < per_lane / 2; ++i) codes[i] = static_cast<std::uint8_t>(code[2 * i] | code[2 * i + 1] << 4);
    if (lane % lanes == 0) {
        std::uint16_t* scales = (is_key ? cache.key_scales : cache.value_scales) +
            (place * (D / cache.group) + lane / lanes) * 2;
        scales[0] = __half_as_ushort(scale);
        scales[1] = __half_as_ushort(minimum);
    }
}

// One thread a code byte of one stored token, keys first, then values.
template <typename T>
__global__ void read_kernel(Cache cache, const std::int64_t* slots, std::int64_t count, T* keys, T* values) {
    const int bytes = cache.head_dim / 2;
    const std::int64_t per_token = static_cast<std::int64_t>(cache.kv_heads) * bytes;
    const std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= 2 * count * per_token) return;
    const bool is_value = i >= count * per_token;
    const std::int64_t at = is_value ? i - count * per_token : i;
    const std::int64_t token = at / per_token;
    const int head = static_cast<int>(at % per_token) / bytes, byte = static_cast<int>(at % per_token) % bytes;
    T* out = (is_value ? values : keys) + 2 * at;
    const std::int64_t slot = slots[token];
    if (slot < 0 || slot >= static_cast<std::int64_t>(cache.pages) * cache.page_size) {
        if (slot >= 0) note(cache, status_slot);
        out[0] = out[1] = narrow<T>(0.0f);
        return;
    }
    const std::int64_t place = (slot / cache.page_size * cache.kv_heads + head) * cache.page_size + slot % cache.page_size;
    const unsigned code = (is_value ? cache.value_codes : cache.key_codes)[place * bytes + byte];
    const std::uint16_t* pair = (is_value ? cache.value_scales : cache.key_scales) +
        (place * (cache.head_dim / cache.group) + 2 * byte / cache.group) * 2;
    const float s = half_bits(pair[0]), m = half_bits(pair[1]);
    out[0] = narrow<T>(fmaf(static_cast<float>(code & 15u), s, m));
    out[1] = narrow<T>(fmaf(static_cast<float>(code >> 4), s, m));
}

template <typename T>
cudaError_t append_typed(const Cache& cache, const AppendArgs& args, cudaStream_t stream) {
    const std::int64_t items = args.tokens * (2 * cache.kv_heads + (args.queries != nullptr ? args.query_heads : 0));
    const unsigned grid = static_cast<unsigned>((items + 7) / 8);
    switch (cache.head_dim) {
    case 64: append_kernel<T, 64><<<grid, 256, 0, stream>>>(cache, args); break;
    case 128: append_kernel<T, 128><<<grid, 256, 0, stream>>>(cache, args); break;
    default: append_kernel<T, 256><<<grid, 256, 0, stream>>>(cache, args); break;
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
    const std::int64_t items = 2 * count * cache.kv_heads * (cache.head_dim / 2);
    const unsigned grid = static_cast<unsigned>((items + 255) / 256);
    if (type == Type::f16) {
        read_kernel<<<grid, 256, 0, stream>>>(cache, slots, count, static_cast<__half*>(keys), static_cast<__half*>(values));
    } else if (type == Type::bf16) {
        read_kernel<<<grid, 256, 0, stream>>>(cache, slots, count, static_cast<__nv_bfloat16*>(keys),
                                              static_cast<__nv_bfloat16*>(values));
    } else {
        read_kernel<<<grid, 256, 0, stream>>>(cache, slots, count, static_cast<float*>(keys), static_cast<float*>(values));
    }
    return cudaGetLastError();
}

}  // namespace nvcr_sm100::token
