// Norms after and before a block, fused with the block's gate and the residual:
//   p = post ? N(block) : block,  hidden = residual_scale * residual + gate * p,
//   normed = N(hidden), with N(v) = v / sqrt(mean(v^2) + epsilon) * (weight +
//   weight_offset) + bias, of v - mean(v) for a layer norm.
// Sums, the residual sum and everything between the inputs and the two outputs
// are FP32; `normed` comes from the unrounded sum. HBM-bound: each input is
// read once and each output written once.
#include "token_elements.cuh"

namespace nvcr_sm100::token {
namespace {

constexpr int threads = 256;

__device__ __forceinline__ float block_sum(float v, float* scratch) {
    v = warp_sum(v);
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
    __syncthreads();
    float total = 0.0f;
    for (int w = 0; w < threads / 32; ++w) total += scratch[w];
    return total;
}

template <typename T>
__device__ __forceinline__ float weight_at(const void* weight, int i, float offset) {
    return weight == nullptr ? 1.0f : widen(static_cast<const T*>(weight)[i]) + offset;
}

template <typename T>
__device__ __forceinline__ float bias_at(const void* bias, int i) {
    return bias == nullptr ? 0.0f : widen(static_cast<const T*>(bias)[i]);
}

// One row a block, re-reading the row for each pass; right for any width and stride.
template <typename T>
__global__ void __launch_bounds__(threads) norm_kernel(NormArgs a) {
    __shared__ float scratch[threads / 32];
    const std::int64_t row = blockIdx.x;
    const T* block = static_cast<const T*>(a.block) + row * a.block_stride;
    const T* residual = a.residual == nullptr ? nullptr : static_cast<const T*>(a.residual) + row * a.residual_stride;
    const T* gate = a.gate == nullptr ? nullptr : static_cast<const T*>(a.gate) + row * a.gate_stride;
    const float inverse = 1.0f / static_cast<float>(a.width);
    float mean = 0.0f, factor = 1.0f;
    if (a.post) {
        if (a.layer) {
            float sum = 0.0f;
            for (int i = threadIdx.x; i < a.width; i += threads) sum += widen(block[i]);
            mean = block_sum(sum, scratch) * inverse;
        }
        float squares = 0.0f;
        for (int i = threadIdx.x; i < a.width; i += threads) {
            const float v = widen(block[i]) - mean;
            squares = fmaf(v, v, squares);
        }
        factor = rsqrtf(block_sum(squares, scratch) * inverse + a.epsilon);
    }
    auto hidden_at = [&](int i) {
        float p = widen(block[i]);
        if (a.post) p = fmaf((p - mean) * factor, weight_at<T>(a.post_weight, i, a.weight_offset), bias_at<T>(a.post_bias, i));
        if (gate != nullptr) p *= widen(gate[i]);
        return residual == nullptr ? p : fmaf(widen(residual[i]), a.residual_scale, p);
    };
    float hidden_mean = 0.0f, hidden_factor = 1.0f;
    if (a.normed != nullptr) {
        if (a.layer) {
            float sum = 0.0f;
            for (int i = threadIdx.x; i < a.width; i += threads) sum += hidden_at(i);
            hidden_mean = block_sum(sum, scratch) * inverse;
        }
        float squares = 0.0f;
        for (int i = threadIdx.x; i < a.width; i += threads) {
            const float v = hidden_at(i) - hidden_mean;
            squares = fmaf(v, v, squares);
        }
        hidden_factor = rsqrtf(block_sum(squares, scratch) * inverse + a.epsilon);
    }
    for (int i = threadIdx.x; i < a.width; i += threads) {
        const float h = hidden_at(i);
        if (a.hidden != nullptr) static_cast<T*>(a.hidden)[row * a.width + i] = narrow<T>(h);
        if (a.normed != nullptr) {
            static_cast<T*>(a.normed)[row * a.width + i] = narrow<T>(fmaf(
                (h - hidden_mean) * hidden_factor, weight_at<T>(a.pre_weight, i, a.weight_offset), bias_at<T>(a.pre_bias, i)));
        }
    }
}

}  // namespace

cudaError_t block_norm(const NormArgs& args, cudaStream_t stream) {
    if (args.rows == 0) return cudaSuccess;
    const unsigned grid = static_cast<unsigned>(args.rows);
    switch (args.type) {
    case Type::f16: norm_kernel<__half><<<grid, threads, 0, stream>>>(args); break;
    case Type::bf16: norm_kernel<__nv_bfloat16><<<grid, threads, 0, stream>>>(args); break;
    case Type::f32: norm_kernel<float><<<grid, threads, 0, stream>>>(args); break;
    }
    return cudaGetLastError();
}

}  // namespace nvcr_sm100::token
