// Attention of new tokens over the paged 4-bit cache. Token i of a sequence's
// count new ones is at position length - count + i and sees the keys up to its
// own position; one that sees none gives zeros. Grouped heads: query head h
// reads cache head h / (heads / kv_heads). One pass over the keys with the
// running maximum and sum of the softmax, in FP32.
#include "token_elements.cuh"

namespace nvcr_sm100::token {
namespace {

constexpr int warps = 4;
constexpr float log2_e = 1.4426950408889634f;

__device__ __forceinline__ void note(const Cache& cache, unsigned bit) {
    if (cache.status != nullptr) atomicOr(cache.status, bit);
}

// One block a (head, new token, sequence); a warp takes every fourth key, a
// lane D / 32 consecutive channels of it.
template <typename T, int D>
__global__ void __launch_bounds__(32 * warps) attend_kernel(Cache cache, AttendArgs a) {
    constexpr int per_lane = D / 32;
    __shared__ float part_top[warps], part_sum[warps], part_out[warps][D];
    const int head = blockIdx.x, index = blockIdx.y, sequence = blockIdx.z;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    std::int64_t first = sequence, last = sequence + 1;
    if (a.query_offsets != nullptr) first = a.query_offsets[sequence], last = a.query_offsets[sequence + 1];
    const std::int64_t count = last - first;
    if (first < 0 || last > a.tokens || count < 0 || count > a.max_queries) {
        if (threadIdx.x == 0) note(cache, status_length);
        return;
    }
    if (index >= count) return;
    int length = a.lengths[sequence];
    if (length < 0 || length > a.max_length) {
        if (threadIdx.x == 0) note(cache, status_length);
        length = length < 0 ? 0 : a.max_length;
    }
    const int visible = static_cast<int>(length - count + index + 1);
    const int kv_head = head / (a.heads / cache.kv_heads);
    const T* query = static_cast<const T*>(a.queries) + (first + index) * a.query_stride + head * a.query_head_stride;
    float q[per_lane];
#pragma unroll
    for (int i = 0; i < per_lane; ++i) q[i] = widen(query[lane * per_lane + i]);
    const float factor = a.scale * log2_e;
    float top = -INFINITY, sum = 0.0f, out[per_lane] = {};
    const int part = lane * per_lane / cache.group;
    for (int t = warp; t < visible; t += warps) {
        const int page = a.page_table[sequence * a.table_stride + t / cache.page_size];
        if (page < 0 || page >= cache.pages) {
            if (lane == 0) note(cache, status_page);
            continue;
        }
        const std::int64_t place = (static_cast<std::int64_t>(page) * cache.kv_heads + kv_head) * cache.page_size +
            t % cache.page_size;
        const std::int64_t codes = place * (D / 2) + lane * (per_lane / 2);
        const std::int64_t pair = (place * (D / cache.group) + part) * 2;
        float score = 0.0f;
        const float ks = half_bits(cache.key_scales[pair]), km = half_bits(cache.key_scales[pair + 1]);
#pragma unroll
        for (int i = 0; i < per_lane; ++i) {
            const unsigned code = cache.key_codes[codes + i / 2] >> (i % 2 * 4) & 15u;
            score = fmaf(q[i], fmaf(static_cast<float>(code), ks, km), score);
        }
        score = warp_sum(score) * factor;
        const float next = fmaxf(top, score);
        const float base = next == -INFINITY ? 0.0f : next;  // every score so far is -infinity
        const float shrink = exp2_fast(top - base), weight = exp2_fast(score - base);
        top = next;
        sum = fmaf(sum, shrink, weight);
        const float vs = half_bits(cache.value_scales[pair]), vm = half_bits(cache.value_scales[pair + 1]);
#pragma unroll
        for (int i = 0; i < per_lane; ++i) {
            const unsigned code = cache.value_codes[codes + i / 2] >> (i % 2 * 4) & 15u;
            out[i] = fmaf(out[i], shrink, weight * fmaf(static_cast<float>(code), vs, vm));
        }
    }
    if (lane == 0) part_top[warp] = top, part_sum[warp] = sum;
#pragma unroll
    for (int i = 0; i < per_lane; ++i) part_out[warp][lane * per_lane + i] = out[i];
    __syncthreads();
    top = -INFINITY;
    for (int w = 0; w < warps; ++w) top = fmaxf(top, part_top[w]);
    if (top == -INFINITY) top = 0.0f;
    sum = 0.0f;
    for (int w = 0; w < warps; ++w) sum += part_sum[w] * exp2_fast(part_top[w] - top);
    T* result = static_cast<T*>(a.output) + ((first + index) * a.heads + head) * D;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float value = 0.0f;
        for (int w = 0; w < warps; ++w) value += part_out[w][d] * exp2_fast(part_top[w] - top);
        result[d] = narrow<T>(sum == 0.0f ? 0.0f : value / sum);
    }
}

template <typename T>
cudaError_t attend_typed(const Cache& cache, const AttendArgs& args, cudaStream_t stream) {
    const dim3 grid(static_cast<unsigned>(args.heads), static_cast<unsigned>(args.max_queries),
                    static_cast<unsigned>(args.batch));
    switch (cache.head_dim) {
    case 64: attend_kernel<T, 64><<<grid, 32 * warps, 0, stream>>>(cache, args); break;
    case 128: attend_kernel<T, 128><<<grid, 32 * warps, 0, stream>>>(cache, args); break;
    default: attend_kernel<T, 256><<<grid, 32 * warps, 0, stream>>>(cache, args); break;
    }
    return cudaGetLastError();
}

}  // namespace

cudaError_t attend(const Cache& cache, const AttendArgs& args, cudaStream_t stream) {
    if (args.tokens == 0 || args.batch == 0) return cudaSuccess;
    return args.type == Type::f16 ? attend_typed<__half>(cache, args, stream)
                                  : attend_typed<__nv_bfloat16>(cache, args, stream);
}

}  // namespace nvcr_sm100::token
